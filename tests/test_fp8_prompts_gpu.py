"""Many-row attention over the 8-bit cache (the histories widened to 16 bits) where its numbers are
unusual: scales over their whole range, blocks with a NaN scale, values past f16. Tolerances are
those of test_fp8_cache_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ref
from test_fp8_cache_gpu import Pool, check, p_step, tables_for

pytestmark = pytest.mark.gpu

WHOLE = [(0, 200), (60, 140), (0, 3)]   # query tiles enough to run whole
SPLIT = [(2300, 170), (5, 30)]          # few query tiles over a long history: keys in runs
FEW = [(92, 6), (30, 5), (0, 4)]        # the few-row kernel


def make(seqs, hq, hkv, d, bs, seed, exps=(-9, 1)):
    rng = np.random.default_rng(seed)
    q_lens, ctx = [b for _, b in seqs], [a + b for a, b in seqs]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d, exps)
    q = torch.from_numpy(rng.standard_normal((sum(q_lens), hq, d)))
    return rng, q_lens, ctx, tables, bt, pool, q


def attend(ops, q, pool, bt, q_lens, ctx, bs, scale, err=None):
    cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
    return ops.paged_prefill_fp8(q.cuda(), *pool.device(), 0, bt.cuda(), cu,
                                 torch.tensor(ctx, dtype=torch.int32, device="cuda"), max(q_lens), bs, scale,
                                 err_flag=err)


@pytest.mark.parametrize("seqs", [WHOLE, SPLIT, FEW])
@pytest.mark.parametrize("low,high", [(-110, -104), (-40, 40), (90, 104)])
def test_value_scales_over_the_whole_range(ops, seqs, low, high):
    hq, hkv, d, bs = 6, 2, 128, 16
    rng, q_lens, ctx, tables, bt, pool, q = make(seqs, hq, hkv, d, bs, low + 600)
    pool.vs = torch.from_numpy(2.0 ** rng.integers(low, high, size=pool.vs.shape))
    q = q.to(torch.bfloat16)
    got = attend(ops, q, pool, bt, q_lens, ctx, bs, d ** -0.5)
    want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, q_lens, ctx, d ** -0.5)
    check(got, want, torch.bfloat16, d, max(ctx), p_step(torch.bfloat16, True))


@pytest.mark.parametrize("seqs", [WHOLE, SPLIT, FEW])
@pytest.mark.parametrize("exp", [-100, -60, 60, 100])
def test_key_scales_far_from_one(ops, seqs, exp):
    """Keys of 2^exp and queries of 2^-exp: the scores are ordinary."""
    hq, hkv, d, bs = 6, 2, 64, 16
    rng, q_lens, ctx, tables, bt, pool, q = make(seqs, hq, hkv, d, bs, exp + 700, (exp - 9, exp + 1))
    pool.vs = torch.from_numpy(2.0 ** rng.integers(-9, 1, size=pool.vs.shape))
    q = (q * 2.0 ** -exp).to(torch.bfloat16)
    got = attend(ops, q, pool, bt, q_lens, ctx, bs, d ** -0.5)
    want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, q_lens, ctx, d ** -0.5)
    check(got, want, torch.bfloat16, d, max(ctx), p_step(torch.bfloat16, True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("seqs", [WHOLE, SPLIT, FEW])
@pytest.mark.parametrize("which", ["keys", "values"])
def test_a_nan_block_shows_in_the_rows_that_see_it_only(ops, which, seqs, dtype):
    hq, hkv, d, bs = 6, 2, 64, 16
    rng, q_lens, ctx, tables, bt, pool, q = make(seqs, hq, hkv, d, bs, 800)
    q = q.to(dtype)
    past = seqs[0][0]
    col = (past + 2) // bs + 1  # some rows lie before it, some behind
    first = col * bs  # its first position
    scales = pool.ks if which == "keys" else pool.vs
    scales[0, tables[0][col], 1] = float("nan")
    got = attend(ops, q, pool, bt, q_lens, ctx, bs, d ** -0.5)
    sees = torch.tensor([past + j >= first for j in range(q_lens[0])])
    assert sees.any() and not sees.all()
    heads = torch.arange(hq) // (hq // hkv) == 1
    want = torch.zeros(sum(q_lens), hq, dtype=torch.bool)
    want[:q_lens[0]] = sees[:, None] & heads[None]
    assert torch.equal(got.isnan().all(-1).cpu(), want) and torch.equal(got.isnan().any(-1).cpu(), want)
    scales[0, tables[0][col], 1] = 1.0  # the other rows do not see this value
    plain = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, q_lens, ctx, d ** -0.5)
    row, head = (~want).nonzero(as_tuple=True)
    out, mass, score = (t[row, head][:, None] for t in plain)
    check(got.cpu()[row, head][:, None], (out, mass, score), dtype, d, max(ctx), p_step(dtype, True))


@pytest.mark.parametrize("seqs", [WHOLE, SPLIT, FEW])
def test_f16_queries_over_what_f16_rows_give(ops, seqs):
    """Value scales from 2^-20 to 2^7 and codes as rows of f16 leave them (multiples of 2^-24): the
    16-bit copy holds each of them. Outputs below the normal range are rounded by 2^-25."""
    hq, hkv, d, bs = 6, 2, 64, 16
    rng, q_lens, ctx, tables, bt, pool, q = make(seqs, hq, hkv, d, bs, 900)
    pool.vs = torch.from_numpy(2.0 ** rng.integers(-20, 8, size=pool.vs.shape))
    wide = pool.vs[0].repeat_interleave(bs, 0)[:, :, None]
    values = (torch.from_numpy(ref.VALUES)[pool.v[0].long()] * wide * 2.0 ** 24).round() * 2.0 ** -24
    pool.v[0] = torch.from_numpy(ref.encode((values / wide).numpy()))
    q = q.to(torch.float16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = attend(ops, q, pool, bt, q_lens, ctx, bs, d ** -0.5, err)
    out, mass, score = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, q_lens, ctx, d ** -0.5)
    eps = torch.finfo(torch.float16).eps
    rel = eps / 2 + 2.0 ** -11 + 2 * d * 2.0 ** -23 * score + (max(ctx) + 64) * 2.0 ** -24 + 2.0 ** -21
    bound = eps / 2 * out.abs() + 2.0 ** -25 + (rel * mass)[:, :, None] * (1 + eps)
    if seqs is not FEW:
        # The tile kernel rounds each weight to f16 relative to a reference no larger than the row's
        # largest, whose own weight is then 1 or more, as is the sum: below 2^-14 by up to 2^-25,
        # which a value of 2^27 times the others' carries into the output. Over the visible keys:
        # 2^-25 * sum |v| / sum of weights <= 2^-25 * sum |v|.
        sums = torch.zeros_like(mass)
        row = 0
        for t, a, c in zip(tables, q_lens, ctx):
            slot = torch.tensor([t[x // bs] * bs + x % bs for x in range(c)])
            v = (torch.from_numpy(ref.VALUES)[pool.v[0].long()] * wide)[slot].abs().max(-1).values  # (tokens, heads)
            run = v.cumsum(0)[c - a:]
            sums[row:row + a] = run.repeat_interleave(hq // hkv, 1)
            row += a
        bound = bound + (2.0 ** -25 * sums)[:, :, None]
    assert ((got.double().cpu() - out).abs() <= bound).all()
    assert err.item() == 0


@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("seqs", [WHOLE, SPLIT])
def test_f16_queries_over_values_past_f16_are_flagged(ops, seqs, which):
    """One stored value past 65,536 that a sequence sees: flagged. 65,536, which rows of 65,504 leave, is
    not, and neither are larger ones that no sequence sees. bf16 queries take them all."""
    hq, hkv, d, bs = 6, 2, 64, 16
    rng, q_lens, ctx, tables, bt, pool, q = make(seqs, hq, hkv, d, bs, 1000)
    codes, scales = (pool.k, pool.ks) if which == "keys" else (pool.v, pool.vs)
    block = tables[0][0]
    spare = next(b for b in range(scales.shape[1]) if not any(b in t for t in tables))
    scales[0, spare] = 2.0 ** 40
    scales[0, block, 1] = 2.0 ** 8
    codes[0, block * bs:(block + 1) * bs, 1] = 0x20  # 2^-3
    for code, flag in ((0x78, 0), (0x79, 32), (0xF8, 0), (0xF9, 32)):  # +-256 and the codes above
        codes[0, block * bs + 7, 1, 21] = code
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = attend(ops, q.half(), pool, bt, q_lens, ctx, bs, d ** -0.5, err)
        assert err.item() == flag and got.isfinite().all()
        err.zero_()
        attend(ops, q.bfloat16(), pool, bt, q_lens, ctx, bs, d ** -0.5, err)
        assert err.item() == 0
