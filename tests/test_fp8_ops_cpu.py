"""Refusals of the 8-bit cache, verification and page entry points (no GPU needed), and the plain
forms that the GPU tests compare with."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ref

FAKE = 1 << 20  # an aligned non-null address: nothing is dereferenced on these paths


def lib():
    from llm_engineering_b200 import _lib

    return _lib, _lib.load()


def test_write_and_read_refusals():
    L, c = lib()

    def write(rows=4, n=1, layer=0, slots=64, hkv=2, d=64, bs=16, dtype=0, keys=FAKE, max_q=4):
        return c.b2p_kv_write_fp8(keys, 128, 64, FAKE, 128, 64, FAKE, FAKE, FAKE, FAKE, FAKE, 4, FAKE, FAKE, n,
                                  rows, max_q, layer, 1, slots, hkv, d, bs, dtype, None, None)

    assert write(n=0) == write(rows=0) == write(max_q=0) == L.B2P_OK
    assert write(layer=1) == L.B2P_ERANGE
    assert write(keys=None) == write(slots=60) == write(rows=-1) == write(hkv=0) == L.B2P_EINVAL
    assert write(d=60) == write(dtype=7) == L.B2P_EUNSUPPORTED

    def read(rows=4, layer=0, d=64, bs=16, cache=FAKE, dtype=2):
        return c.b2p_kv_read_fp8(cache, FAKE, FAKE, FAKE, FAKE, rows, FAKE, FAKE, layer, 1, 64, 2, d, bs, dtype,
                                 None, None)

    assert read(rows=0) == L.B2P_OK
    assert read(layer=-1) == L.B2P_ERANGE
    assert read(cache=None) == read(cache=FAKE + 4) == read(bs=15) == L.B2P_EINVAL
    assert read(d=12) == read(dtype=3) == L.B2P_EUNSUPPORTED


def test_attention_refusals():
    L, c = lib()

    def decode(n=1, hq=4, hkv=2, d=64, bs=16, layer=0, q=FAKE, dtype=0, slots=64, cache=FAKE, scale=0.1, ws=None):
        return c.b2p_paged_decode_fp8(q, 256, 64, cache, FAKE, FAKE, FAKE, layer, 1, slots, FAKE, 4, FAKE, n, hq,
                                      hkv, d, bs, scale, FAKE, 256, 64, ws, 0, dtype, None, None)

    def prefill(n=1, rows=2, max_q=2, hq=4, hkv=2, d=64, q=FAKE):
        return c.b2p_paged_prefill_fp8(q, 256, 64, FAKE, FAKE, FAKE, FAKE, 0, 1, 64, FAKE, 4, FAKE, FAKE, n, rows,
                                       max_q, hq, hkv, d, 16, 0.1, FAKE, 256, 64, None, 0, None, 0, 0, None, None)

    assert decode(n=0) == prefill(n=0) == prefill(rows=0) == prefill(max_q=0) == L.B2P_OK
    assert decode(layer=3) == L.B2P_ERANGE
    assert decode(hq=5) == decode(slots=60) == decode(q=None) == decode(dtype=9) == L.B2P_EINVAL
    assert decode(scale=-0.1) == decode(scale=float("nan")) == decode(ws=FAKE + 4) == L.B2P_EINVAL
    assert decode(cache=FAKE + 1) == prefill(q=None) == prefill(max_q=-1) == L.B2P_EINVAL
    assert decode(d=60) == decode(d=512) == prefill(d=264) == L.B2P_EUNSUPPORTED
    # rows that fit no pass of the few-row kernel need the scratch, few rows the workspace
    assert prefill(rows=200, max_q=200) == decode() == L.B2P_EWORKSPACE
    assert c.b2p_paged_prefill_fp8_scratch_size(2, 300, 10, 4, 2, 64, 16, 200, 0) >= 2 * 10 * 16 * 2 * 64 * 4
    assert c.b2p_paged_prefill_fp8_scratch_size(2, 300, 10, 4, 2, 64, 16, 5, 0) == 0
    assert c.b2p_paged_prefill_fp8_scratch_size(2, 300, 10, 4, 2, 64, 16, 200, 2) == 0
    assert c.b2p_paged_fp8_workspace_size(0, 4, 2, 64, 1) == 0
    assert c.b2p_paged_fp8_workspace_size(4, 12, 2, 128, 1) > 0


def test_verify_refusals():
    L, c = lib()

    def verify(n=2, total=4, top=3, vocab=100, dtype=2, out_row=4, target=FAKE, tokens=FAKE):
        return c.b2p_verify_drafts(target, 100, FAKE, 100, tokens, FAKE, FAKE, FAKE, n, total, top, vocab, dtype,
                                   FAKE, out_row, FAKE, None, None)

    assert verify(n=0) == L.B2P_OK
    assert verify(out_row=3) == verify(target=None) == verify(tokens=None) == L.B2P_EINVAL
    assert verify(vocab=0) == verify(total=-1) == verify(dtype=4) == L.B2P_EINVAL
    assert verify(vocab=(1 << 30) + 1) == L.B2P_EUNSUPPORTED

    def greedy(n=2, total=4, out_row=4, ids=FAKE):
        return c.b2p_verify_drafts_greedy(ids, FAKE, FAKE, n, total, 3, FAKE, out_row, FAKE, None, None)

    assert greedy(n=0) == L.B2P_OK
    assert greedy(out_row=2) == greedy(ids=None) == greedy(n=-1) == L.B2P_EINVAL


def test_page_refusals():
    L, c = lib()

    def copy(pairs=2, ks=None, vs=None, bs=16, es=2, cache=FAKE):
        return c.b2p_copy_blocks(cache, FAKE, ks, vs, FAKE, FAKE, pairs, 2, 64, 2, 64, es, bs, None, None)

    assert copy(pairs=0) == L.B2P_OK
    assert copy(pairs=-1) == copy(bs=15) == copy(ks=FAKE) == copy(cache=None) == L.B2P_EINVAL
    assert copy(es=3) == L.B2P_EUNSUPPORTED

    def compact(width=4, stride=4, ws=FAKE, size=1 << 16, n=2, tables=FAKE):
        return c.b2p_compact_blocks(FAKE, FAKE, None, None, tables, stride, width, FAKE, n, 2, 64, 2, 64, 2, 16,
                                    FAKE, FAKE, ws, size, None, None)

    assert compact(stride=3) == compact(tables=None) == compact(n=-1) == L.B2P_EINVAL
    assert compact(ws=FAKE + 8) == L.B2P_EINVAL
    assert compact(ws=None) == compact(size=16) == L.B2P_EWORKSPACE
    assert c.b2p_compact_blocks_workspace_size(0) == 0
    assert c.b2p_compact_blocks_workspace_size(1 << 20) >= (1 << 17) + (1 << 22)


def test_python_checks_refuse_cpu_tensors():
    from llm_engineering_b200 import ops

    kc = torch.zeros(1, 32, 2, 64).to(torch.float8_e4m3fn)
    s = torch.ones(1, 2, 2)
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 2, 64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.kv_write_fp8(kc, kc, s, s, 0, i.view(1, 2), i, i, 1, 16, x, x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.paged_decode_fp8(x, kc, kc, s, s, 0, i.view(1, 2), i, 16, 1.0)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.verify_drafts(torch.rand(2, 8), i.long()[:1], i, torch.rand(1), torch.rand(1), 1)
    with pytest.raises(ValueError, match="8-bit pool needs"):
        ops.copy_blocks(kc, kc, i, i, 16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.compact_blocks(x.view(1, 1, 2, 64), x.view(1, 1, 2, 64), i.view(1, 2), i, 1)


def test_plain_encode_matches_the_format():
    """The oracle's rounding against torch's own e4m3 cast (both round to nearest even)."""
    x = np.concatenate([np.linspace(-448, 448, 20001), np.linspace(-0.05, 0.05, 9999), ref.VALUES[:127],
                        (ref.VALUES[:126] + ref.VALUES[1:127]) / 2])
    codes = torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    x32 = x.astype(np.float32).astype(np.float64)
    assert np.array_equal(ref.encode(x32), codes)
    assert ref.block_scale(0.0) == 2.0 ** -110
    assert ref.block_scale(448.0) == 1.0 and ref.block_scale(448.1) == 2.0


def test_plain_compaction_is_a_bijection():
    moves, new, live = ref.compact([[7, 3], [9, 3], [1]], [30, 32, 5], 16, 12)
    assert live == 4 and moves == [(7, 0), (9, 2)]
    assert sorted(x for x in new if x >= 0) == list(range(4))
