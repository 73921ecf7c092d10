"""Scratch of many-row calls over the 8-bit cache: bounded by the pool, whatever the tables' width."""

from __future__ import annotations

import pytest


def lib():
    from llm_engineering_b200 import _lib

    return _lib.load()


def wide(blocks, bs, hkv, d):
    return 2 * blocks * bs * hkv * d * 2


def test_a_ragged_batch_takes_no_more_than_the_pool():
    """32 prompts of which one has 131,072 tokens (8 heads of 128): 17 GB by the tables' entries."""
    c = lib()
    n, width, bs, hkv, hq, d, rows = 32, 8192, 16, 8, 32, 128, 8192
    blocks = 12000  # what the pool holds
    args = (hq, hkv, d, bs, 512, 0)
    size = c.b2p_paged_prefill_fp8_pool_scratch_size(n, rows, width, blocks * bs, *args)
    # K and V in 16 bits, the checked lengths and offsets, and alignment; no runs at so many rows
    assert wide(blocks, bs, hkv, d) <= size <= wide(blocks, bs, hkv, d) + 4096
    assert size < 1.6e9 < 17e9 < c.b2p_paged_prefill_fp8_scratch_size(n, rows, width, *args)


@pytest.mark.parametrize("n,width,blocks", [(4, 40, 1000), (4, 40, 160), (4, 40, 159), (1, 1, 1), (7, 3000, 20001)])
def test_the_smaller_of_entries_and_blocks(n, width, blocks):
    c = lib()
    hq, hkv, d, bs, rows = 4, 2, 64, 16, 100000
    size = c.b2p_paged_prefill_fp8_pool_scratch_size(n, rows, width, blocks * bs, hq, hkv, d, bs, 200, 1)
    least = wide(min(n * width, blocks), bs, hkv, d)
    assert least <= size <= least + 4 * (n * width + 2 * n + 3) + 2048
    assert size <= c.b2p_paged_prefill_fp8_scratch_size(n, rows, width, hq, hkv, d, bs, 200, 1)


def test_calls_that_need_none():
    c = lib()
    assert c.b2p_paged_prefill_fp8_pool_scratch_size(2, 300, 10, 640, 4, 2, 64, 16, 5, 0) == 0    # few rows
    assert c.b2p_paged_prefill_fp8_pool_scratch_size(2, 300, 10, 640, 4, 2, 64, 16, 200, 2) == 0  # fp32
    assert c.b2p_paged_prefill_fp8_pool_scratch_size(2, 300, 10, 640, 4, 2, 40, 16, 200, 0) == 0  # head_dim
    assert c.b2p_paged_prefill_fp8_pool_scratch_size(2, 300, 10, 0, 4, 2, 64, 16, 200, 0) == 0


def test_refusals_of_a_width():
    from llm_engineering_b200 import _lib

    c = lib()
    fake = 1 << 20

    def prefill(width, stride=4, n=1, rows=200):
        return c.b2p_paged_prefill_fp8_reach(fake, 256, 64, fake, fake, fake, fake, 0, 1, 64, fake, stride, width, fake,
                                             fake, n, rows, 200, 4, 2, 64, 16, 0.1, fake, 256, 64, None, 0, None, 0, 0,
                                             None, None)

    assert prefill(5) == prefill(-1) == _lib.B2P_EINVAL
    assert prefill(4, n=0) == prefill(0, rows=0) == _lib.B2P_OK
    assert prefill(4) == prefill(1) == _lib.B2P_EWORKSPACE
