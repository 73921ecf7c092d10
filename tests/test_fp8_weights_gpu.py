"""Few-row attention over the 8-bit cache where one key outweighs all others and its value is zero
(an attention sink): the output is the sum of many small weights.

Tolerances are those of test_fp8_cache_gpu.py, which are relative to sum p|v| and so to what the
small weights bring. The product of a weight and its block's scale is rounded to f16 against a
reference that puts the largest one at 2^10 or above: a weight at least 2^-24 of it is a normal f16
number, rounded by 2^-11 of itself at most; below that the rounding is 2^-25 against
2^10 times the weight, 2^(d - 35) of a weight that is 2^-d of the largest."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ref

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def check(got, want, dtype, head_dim, n, p_eps):
    from test_fp8_cache_gpu import check as within

    within(got, want, dtype, head_dim, n, p_eps)


def sink_pool(rng, keys, bs, hkv, d):
    """One history of `keys` tokens: dim 0 of every key is what a query (that has only dim 0) scores
    by: 8 for the first token, 0 for the others. The first token's value is zero; the others' have
    a mean, so that their weighted sum is near sum p|v|."""
    blocks = keys // bs
    k = rng.standard_normal((keys, hkv, d)) * 60
    k[:, :, 0] = 0.0
    k[0, :, 0] = 8.0
    v = 150.0 + 60 * rng.standard_normal((keys, hkv, d))
    v[0] = 0.0
    kc, vc = (torch.from_numpy(ref.encode(np.clip(x, -448, 448))) for x in (k, v))
    ks = torch.ones(blocks, hkv, dtype=torch.float64)
    vs = torch.full((blocks, hkv), 2.0 ** -7, dtype=torch.float64)
    dev = [t[None].cuda().view(FP8) for t in (kc, vc)] + [t[None].float().cuda() for t in (ks, vs)]
    return (kc, ks, vc, vs), dev


GAPS = [4.0, 12.0, 18.0, 20.5, 22.0, 23.5, 24.0]  # log2 of the first key's weight over each other's


def queries(rows, hq, d, dtype):
    """Row r puts GAPS[r % 7] log2 units between the first key and the others (scale 1)."""
    q = torch.zeros(rows, hq, d, dtype=torch.float64)
    for r in range(rows):
        q[r, :, 0] = GAPS[r % len(GAPS)] * np.log(2.0) / 8.0
    return q.to(dtype)  # bf16 rounds a gap by up to 2^-9 of it: 24 stays below 24.1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("keys", [2048, 16384])
def test_decode_of_small_weights_next_to_a_sink(ops, keys, dtype):
    """As many sequences (over the same blocks) as make every warp walk a whole history, so that the
    first key's reference holds for all the others."""
    hq, hkv, d, bs = 2, 1, 64, 16
    n = 1400
    rng = np.random.default_rng(keys)
    plain, dev = sink_pool(rng, keys, bs, hkv, d)
    q = queries(n, hq, d, dtype)
    table = list(range(keys // bs))
    bt = torch.tensor(table, dtype=torch.int32, device="cuda")[None].expand(n, -1).contiguous()
    ctx = torch.full((n,), keys, dtype=torch.int32, device="cuda")
    got = ops.paged_decode_fp8(q.cuda(), *dev, 0, bt, ctx, bs, 1.0)
    some = list(range(0, n, 97)) + list(range(700, 714))
    want = ref.attend(q[some], *plain, bs, [table] * len(some), [1] * len(some), [keys] * len(some), 1.0)
    # gaps up to 24.1: 2^(24.1 - 35) where a weight is below the normal range
    check(got[some], want, dtype, d, keys, 2 * 2.0 ** -10.9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_drafted_rows_of_small_weights_next_to_a_sink(ops, dtype):
    """The same with two rows a sequence (twelve columns)."""
    hq, hkv, d, bs, keys, n = 6, 1, 128, 16, 4096, 1300
    rng = np.random.default_rng(3)
    plain, dev = sink_pool(rng, keys, bs, hkv, d)
    q = queries(2 * n, hq, d, dtype)
    bt = torch.arange(keys // bs, dtype=torch.int32, device="cuda")[None].expand(n, -1).contiguous()
    ctx = torch.full((n,), keys, dtype=torch.int32, device="cuda")
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    got = ops.paged_prefill_fp8(q.cuda(), *dev, 0, bt, cu, ctx, 2, bs, 1.0)
    seqs = list(range(0, n, 131)) + list(range(600, 607))
    some = [r for s in seqs for r in (2 * s, 2 * s + 1)]
    want = ref.attend(q[some], *plain, bs, [list(range(keys // bs))] * len(seqs), [2] * len(seqs),
                      [keys] * len(seqs), 1.0)
    check(got[some], want, dtype, d, keys, 2 * 2.0 ** -10.9)


def test_a_gap_grows_while_a_sequence_is_walked(ops):
    """Scores that climb by less than a reference's slack per tile and by 40 log2 units in all, with value
    scales that fall meanwhile: the reference follows, and what is stored never passes f16."""
    hq, hkv, d, bs, keys, n = 2, 1, 64, 16, 2048, 1300
    rng = np.random.default_rng(4)
    plain, dev = sink_pool(rng, keys, bs, hkv, d)
    kc, ks, vc, vs = plain
    climb = np.repeat(np.arange(keys // 32), 32) / (keys / 32)  # 0 .. 1 by tile
    kc[:, 0, 0] = torch.from_numpy(ref.encode(climb * 448))
    vs[:, 0] = 2.0 ** torch.from_numpy(rng.integers(-60, 60, keys // bs)).double()
    dev[0] = kc[None].cuda().view(FP8)
    dev[3] = vs[None].float().cuda()
    q = torch.zeros(n, hq, d, dtype=torch.float64)
    q[:, :, 0] = 40 * np.log(2.0) / 448
    q = q.to(torch.bfloat16)
    bt = torch.arange(keys // bs, dtype=torch.int32, device="cuda")[None].expand(n, -1).contiguous()
    ctx = torch.full((n,), keys, dtype=torch.int32, device="cuda")
    got = ops.paged_decode_fp8(q.cuda(), *dev, 0, bt, ctx, bs, 1.0)
    assert got.isfinite().all()
    some = list(range(0, n, 173))
    want = ref.attend(q[some], *plain, bs, [list(range(keys // bs))] * len(some), [1] * len(some),
                      [keys] * len(some), 1.0)
    check(got[some], want, torch.bfloat16, d, keys, torch.finfo(torch.float16).eps)
