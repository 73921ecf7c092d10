"""Values of an 8-bit pool near and past the range of f16, read back as f16. A code is rounded by
2^-4 of its value at most, so the block's largest magnitudes round up past 65,504."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def empty_pool(blocks, bs, hkv, d):
    codes = [torch.zeros(1, blocks * bs, hkv, d, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2)]
    return codes + [torch.zeros(1, blocks, hkv, device="cuda") for _ in range(2)]


def test_largest_f16_rows_read_back_finite(ops):
    """65,504 is stored as 65,536: within half a step of e4m3, so finite in and finite out, and as
    close as f16 can say."""
    hkv, d, bs = 2, 64, 16
    top = torch.finfo(torch.float16).max
    new = torch.tensor([top, 63488.0, 63456.0, 61440.0, 57344.0, -top, -63488.0, 1.0], dtype=torch.float16)
    rows = new.repeat(16 * hkv * d // 8).view(16, hkv, d).cuda()
    dev = empty_pool(1, bs, hkv, d)
    bt = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 16], dtype=torch.int32, device="cuda")
    ctx = torch.tensor([16], dtype=torch.int32, device="cuda")
    ops.kv_write_fp8(*dev, 0, bt, cu, ctx, 16, bs, rows, -rows)
    slots = torch.arange(16, dtype=torch.int32, device="cuda")
    keys, values = ops.kv_read_fp8(*dev, 0, slots, bs, torch.float16)
    for got, want in ((keys, rows), (values, -rows)):
        assert got.isfinite().all()
        assert ((got.double() - want.double()).abs() <= want.double().abs() * 2.0 ** -4).all()
    wide, _ = ops.kv_read_fp8(*dev, 0, slots, bs, torch.float32)  # the stored values themselves
    assert torch.equal(keys, wide.clamp(-top, top).half())
    assert wide.abs().max() == 65536


def test_reads_past_f16_are_its_largest_and_nan_stays(ops):
    hkv, d, bs = 1, 64, 16
    rng = np.random.default_rng(0)
    dev = empty_pool(3, bs, hkv, d)
    rows = torch.from_numpy(rng.standard_normal((48, hkv, d)) * 1e6).float()
    rows[20, 0, 5] = float("nan")
    rows[32:] = 3.0
    bt = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    ops.kv_write_fp8(*dev, 0, bt, torch.tensor([0, 48], dtype=torch.int32, device="cuda"),
                     torch.tensor([48], dtype=torch.int32, device="cuda"), 48, bs, rows.cuda(), rows.cuda())
    slots = torch.tensor([b * bs + i for b in (2, 0, 1) for i in range(bs)], dtype=torch.int32, device="cuda")
    got, _ = ops.kv_read_fp8(*dev, 0, slots, bs, torch.float16)
    wide, _ = ops.kv_read_fp8(*dev, 0, slots, bs, torch.float32)
    top = torch.finfo(torch.float16).max
    assert got[16:32].isnan().all() and wide[16:32].isnan().all()
    for part in (slice(0, 16), slice(32, 48)):
        assert torch.equal(got[part], wide[part].clamp(-top, top).half())
    assert wide[:16].abs().max() > 1e6
