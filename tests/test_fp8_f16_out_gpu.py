"""Attention in f16 over values near the type's limit: an output is a mean of finite rows, so it is
finite, in each of the kernels (few rows, many rows, CUDA cores). Stored values are within 2^-4 of
the rows; an output past 65,504, f16's largest finite value, is that."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
TOP = torch.finfo(torch.float16).max


@pytest.mark.parametrize("d,bs", [(64, 16), (128, 16), (40, 16), (64, 8)])
@pytest.mark.parametrize("q_len", [None, 2, 130])
@pytest.mark.parametrize("long", [False, True])
def test_means_of_the_largest_rows_are_finite(ops, d, bs, q_len, long):
    hq, hkv = 6, 2
    rng = np.random.default_rng(d + bs)
    n, rows = 3, q_len or 1
    ctx = [rows + (3000 if long else 5)] * n  # long: sequences cut over several units
    need = -(-ctx[0] // bs)
    bt = torch.arange(n * need, dtype=torch.int32, device="cuda").view(n, need)
    new = torch.full((sum(ctx), hkv, d), TOP, dtype=torch.float16)
    new[:, :, ::2] = -TOP
    dev = [torch.zeros(1, n * need * bs, hkv, d, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2)]
    dev += [torch.zeros(1, n * need, hkv, device="cuda") for _ in range(2)]
    cu = torch.tensor([0, *np.cumsum(ctx)], dtype=torch.int32, device="cuda")
    c = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    keys = torch.from_numpy(rng.standard_normal((sum(ctx), hkv, d))).half()
    ops.kv_write_fp8(*dev, 0, bt, cu, c, ctx[0], bs, keys.cuda(), new.cuda())
    q = torch.from_numpy(rng.standard_normal((n * rows, hq, d))).half().cuda()
    if q_len is None:
        got = ops.paged_decode_fp8(q, *dev, 0, bt, c, bs, d ** -0.5)
    else:
        at = torch.arange(0, n * rows + 1, rows, dtype=torch.int32, device="cuda")
        got = ops.paged_prefill_fp8(q, *dev, 0, bt, at, c, rows, bs, d ** -0.5)
    # the mean of equal values is that value: rounding of weights and sums moves it by 2^-9 at most
    assert got.isfinite().all()
    assert (got[..., 1::2].double() >= TOP * (1 - 2.0 ** -9)).all()
    assert (got[..., ::2].double() <= -TOP * (1 - 2.0 ** -9)).all()
