"""The 8-bit KV cache against its 64-bit plain forms: rows in and out, attention over it.

Tolerances. Writes and reads are exact (codes are rounded once, by the same rule). Attention:
an output is rounded to its type (half a step, eps/2 of its value); P is rounded to 16 bits
before P.V (eps_p/2 of each weight, so at most eps_p/2 * sum p|v|); a sequence split over units
leaves partial rows in f16 scaled by the row's largest value (2^-11 of it); a score's error d
changes a weight by 2d (its own and the sum's). Scores are sums of D products in fp32 that the
tensor cores may truncate: d <= D * 2^-23 * sum|q k| * scale. Sums of n weights in fp32 add
(n + 64) * 2^-24, exp2 its 2^-21.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ref

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def tables_for(rng, ctx, bs, spare=3):
    need = [-(-c // bs) for c in ctx]
    ids = rng.permutation(sum(need) + spare).tolist()
    out, used = [], 0
    for n in need:
        out.append(ids[used:used + n])
        used += n
    width = max(1, max(need))
    bt = torch.full((len(ctx), width), -1, dtype=torch.int32)
    for i, t in enumerate(out):
        bt[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    return out, bt, sum(need) + spare


class Pool:
    """A pool filled with every code (NaN codes among them in slots no context reaches)."""

    def __init__(self, rng, layers, blocks, bs, hkv, d, exps=(-9, 1)):
        self.bs = bs
        shape = (layers, blocks * bs, hkv, d)
        self.k, self.v = (torch.from_numpy(self._codes(rng, shape)) for _ in range(2))
        s = (layers, blocks, hkv)
        self.ks, self.vs = (torch.from_numpy(2.0 ** rng.integers(*exps, size=s)) for _ in range(2))

    @staticmethod
    def _codes(rng, shape):
        # normal values rather than uniform codes: scores of a few units, as a model's
        return ref.encode(np.clip(rng.standard_normal(shape) * 60, -448, 448))

    def device(self):
        return [t.cuda().view(FP8) for t in (self.k, self.v)] + [t.float().cuda() for t in (self.ks, self.vs)]

    def poison_unused(self, tables, ctx):
        """NaN codes in every slot that no context covers, NaN scales in unused blocks."""
        used = torch.zeros(self.k.shape[1], dtype=torch.bool)
        blocks = torch.zeros(self.ks.shape[1], dtype=torch.bool)
        for t, c in zip(tables, ctx):
            for p in range(c):
                used[t[p // self.bs] * self.bs + p % self.bs] = True
                blocks[t[p // self.bs]] = True
        for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
            codes[:, ~used] = 0x7F
            scales[:, ~blocks] = float("nan")


def check(got, want, dtype, head_dim, n, p_eps):
    out, mass, score = want
    eps = torch.finfo(dtype).eps
    d = head_dim * 2.0 ** -23 * score
    rel = p_eps / 2 + 2.0 ** -11 * (dtype != torch.float32) + 2 * d + (n + 64) * 2.0 ** -24 + 2.0 ** -21
    bound = eps / 2 * out.abs() + (rel * mass)[:, :, None] * (1 + eps)
    err = (got.double().cpu() - out).abs()
    worst = (err - bound).max().item()
    assert worst <= 0, (worst, err.max().item())


def p_step(dtype, prefill):
    """Step of the type that P is rounded to: the query's in the prompt kernel, f16 elsewhere;
    fp32 queries keep P in fp32."""
    if dtype == torch.float32:
        return 0.0
    return torch.finfo(dtype if prefill else torch.float16).eps


SHAPES = [
    # (hq, hkv, d, bs)
    (12, 2, 128, 16),
    (14, 2, 64, 16),
    (28, 4, 128, 16),
    (12, 2, 128, 32),
    (8, 1, 128, 64),
    (32, 2, 128, 16),   # group of 16
    (4, 4, 64, 16),     # no GQA
    (6, 2, 128, 48),    # a block size that is not a power of two
    (20, 1, 64, 16),    # a group of 20: two column passes
    (6, 2, 128, 8),     # CUDA-core kernel: block size below 16
    (200, 1, 64, 16),   # ... group above 160
    (4, 2, 40, 16),     # ... head_dim
    (4, 2, 256, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_decode(ops, shape, dtype):
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(hq * 1000 + d + bs)
    ctx = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 130, 257, 400]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 2, blocks, bs, hkv, d)
    pool.poison_unused(tables, ctx)
    q = torch.from_numpy(rng.standard_normal((len(ctx), hq, d))).to(dtype)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_decode_fp8(q.cuda(), *pool.device(), 1, bt.cuda(),
                               torch.tensor(ctx, dtype=torch.int32, device="cuda"), bs, d ** -0.5,
                               err_flag=err)
    want = ref.attend(q, pool.k[1], pool.ks[1], pool.v[1], pool.vs[1], bs, tables, [1] * len(ctx), ctx,
                      d ** -0.5)
    check(got, want, dtype, d, max(ctx), p_step(dtype, False))
    assert err.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,lo,hi", [(1, 1, 1), (1, 5000, 5000), (3, 900, 2500), (150, 1, 90), (300, 1, 40)])
def test_decode_split_and_crowded(ops, n, lo, hi, dtype):
    """Long sequences cut over many units, many short ones in one unit; one workspace throughout."""
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(n)
    ws = ops.make_fp8_workspace(n, hq, hkv, d, torch.device("cuda"))
    for trial in range(2):
        ctx = rng.integers(lo, hi + 1, n).tolist()
        tables, bt, blocks = tables_for(rng, ctx, bs)
        pool = Pool(rng, 1, blocks, bs, hkv, d)
        q = torch.from_numpy(rng.standard_normal((n, hq, d))).to(dtype)
        got = ops.paged_decode_fp8(q.cuda(), *pool.device(), 0, bt.cuda(),
                                   torch.tensor(ctx, dtype=torch.int32, device="cuda"), bs, d ** -0.5,
                                   workspace=ws)
        want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, [1] * n, ctx,
                          d ** -0.5)
        check(got, want, dtype, d, max(ctx), p_step(dtype, False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("low,high", [(-110, -104), (-40, 40), (90, 104)])
def test_decode_extreme_scales(ops, low, high, dtype):
    """Value scales over the whole range: P is scaled by 2^e before it is rounded, and a block
    with a far larger scale than another must not flush the other's weights."""
    hq, hkv, d, bs = 6, 1, 128, 16
    rng = np.random.default_rng(low + 500)
    ctx = [70, 33, 700]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    pool.vs = torch.from_numpy(2.0 ** rng.integers(low, high, size=pool.vs.shape))
    if dtype == torch.float16:  # the result has to fit its type
        pool.vs = torch.clamp(pool.vs, max=2.0 ** 4)
    q = torch.from_numpy(rng.standard_normal((len(ctx), hq, d))).to(dtype)
    got = ops.paged_decode_fp8(q.cuda(), *pool.device(), 0, bt.cuda(),
                               torch.tensor(ctx, dtype=torch.int32, device="cuda"), bs, d ** -0.5)
    out, mass, score = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, [1] * 3, ctx,
                                  d ** -0.5)
    if dtype == torch.float16:  # below the normal range a step is 2^-24
        err = (got.double().cpu() - out).abs()
        eps = 2.0 ** -10
        bound = eps / 2 * out.abs() + 2.0 ** -25 + (mass * (eps + 2 * d * 2.0 ** -23 * score + 2.0 ** -14))[:, :, None]
        assert (err <= bound).all()
    else:
        check(got, (out, mass, score), dtype, d, max(ctx), p_step(dtype, False))


def test_decode_strided_query_and_out(ops):
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(5)
    ctx = [40, 7, 100]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    q = torch.from_numpy(rng.standard_normal((3, hq, d))).to(torch.bfloat16)
    hf = torch.zeros(1, hq, 3, d, dtype=torch.bfloat16, device="cuda")  # (1, heads, tokens, dim)
    hf[0] = q.transpose(0, 1).cuda()
    out = torch.full((3, 2 * hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    args = (*pool.device(), 0, bt.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"), bs, d ** -0.5)
    got = ops.paged_decode_fp8(hf[0].transpose(0, 1), *args, out=out[:, :hq])
    assert torch.equal(got, ops.paged_decode_fp8(q.cuda(), *args))
    assert (out[:, hq:] == 7).all()


def test_decode_empty_and_bad_rows(ops):
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(6)
    ctx = [0, 20, 0, 5, 33]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    bt[3, 0] = blocks + 4  # outside the pool
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    q = torch.from_numpy(rng.standard_normal((5, hq, d))).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_decode_fp8(q.cuda(), *pool.device(), 0, bt.cuda(),
                               torch.tensor(ctx, dtype=torch.int32, device="cuda"), bs, d ** -0.5, err_flag=err)
    assert (got[[0, 2]] == 0).all()
    assert err.item() == 8 | 2  # a length that does not fit, a block outside the pool
    tables[3] = tables[4][:1]
    want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, [1] * 5, ctx, d ** -0.5)
    keep = [1, 4]
    check(got[keep], tuple(t[keep] for t in want), torch.bfloat16, d, 33, p_step(torch.bfloat16, False))


def test_a_nan_block_shows_and_stays_inside_its_sequence(ops):
    hq, hkv, d, bs = 4, 2, 64, 16
    rng = np.random.default_rng(8)
    ctx = [50, 50]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    pool.vs[0, tables[0][1], 1] = float("nan")
    q = torch.from_numpy(rng.standard_normal((2, hq, d))).to(torch.float16)
    got = ops.paged_decode_fp8(q.cuda(), *pool.device(), 0, bt.cuda(),
                               torch.tensor(ctx, dtype=torch.int32, device="cuda"), bs, d ** -0.5)
    assert got[0, 2:].isnan().all() and got[0, :2].isfinite().all() and got[1].isfinite().all()


PREFILL = [
    # (hq, hkv, d, bs, [(past, q_len)])
    (12, 2, 128, 16, [(100, 5), (0, 1), (15, 1), (16, 4), (63, 2), (300, 6)]),
    (12, 2, 128, 16, [(600, 1), (7, 3), (700, 2)]),
    (14, 2, 64, 32, [(100, 5), (31, 4), (0, 8)]),
    (28, 4, 128, 16, [(200, 4), (0, 7), (90, 3)]),
    (8, 1, 128, 16, [(130, 16), (0, 9), (257, 12)]),
    (32, 2, 128, 16, [(60, 3), (500, 5)]),
    (4, 4, 64, 16, [(33, 9), (0, 2)]),
    (12, 2, 128, 16, [(0, 130), (0, 1), (40, 128), (257, 200), (0, 64)]),
    (14, 2, 64, 16, [(0, 129), (300, 70), (0, 5)]),
    (6, 2, 128, 48, [(10, 140), (200, 33)]),
    (5, 5, 64, 64, [(0, 260), (64, 64)]),
    (12, 2, 128, 16, [(90, 26), (0, 20), (500, 17)]),   # ten passes of 16 columns
    (2, 2, 64, 32, [(0, 150), (33, 160), (10, 1)]),     # no GQA: 160 rows in as many columns
    (40, 2, 64, 16, [(70, 3), (0, 4)]),                 # a group of 20
    (12, 2, 128, 16, [(2300, 130), (5, 200)]),          # the tile kernel with split keys
    (14, 2, 64, 32, [(4200, 180), (0, 3), (129, 128)]),
    (6, 2, 128, 8, [(10, 40), (0, 3)]),
    (4, 2, 40, 16, [(10, 20), (0, 3)]),
    (4, 2, 256, 16, [(10, 20)]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", PREFILL)
def test_prefill(ops, case, dtype):
    hq, hkv, d, bs, seqs = case
    rng = np.random.default_rng(hq + d + bs + len(seqs))
    q_lens, ctx = [b for _, b in seqs], [a + b for a, b in seqs]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 2, blocks, bs, hkv, d)
    pool.poison_unused(tables, ctx)
    q = torch.from_numpy(rng.standard_normal((sum(q_lens), hq, d))).to(dtype)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_prefill_fp8(q.cuda(), *pool.device(), 1, bt.cuda(), cu,
                                torch.tensor(ctx, dtype=torch.int32, device="cuda"), max(q_lens), bs,
                                d ** -0.5, err_flag=err)
    want = ref.attend(q, pool.k[1], pool.ks[1], pool.v[1], pool.vs[1], bs, tables, q_lens, ctx, d ** -0.5)
    check(got, want, dtype, d, max(ctx), p_step(dtype, True))
    assert err.item() == 0


@pytest.mark.parametrize("q_lens", [[3, 2, 5], [40, 150, 2]])
def test_prefill_trailing_slice_and_rows_behind(ops, q_lens):
    """cu_seqlens_q that starts past 0 (a slice of a packed batch), rows behind the last
    sequence left as they were, a sequence without rows, max_q_len above the longest."""
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(11)
    lens = [4] + q_lens + [0]
    past = [9, 70, 0, 33, 12]
    ctx = [a + b for a, b in zip(past, lens)]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    rows = sum(lens) + 3
    q = torch.from_numpy(rng.standard_normal((rows, hq, d))).to(torch.bfloat16)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    c = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 3.0).cuda()
    ops.paged_prefill_fp8(q.cuda(), *pool.device(), 0, bt.cuda()[1:], cu[1:], c[1:], max(lens) + 2, bs,
                          d ** -0.5, out=out)
    want = ref.attend(q[4:-3], pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables[1:], lens[1:], ctx[1:],
                      d ** -0.5)
    check(out[4:-3], want, torch.bfloat16, d, max(ctx), p_step(torch.bfloat16, True))
    assert (out[:4] == 3).all() and (out[-3:] == 3).all()


@pytest.mark.parametrize("long", [3, 150])
def test_prefill_flags_what_does_not_fit(ops, long):
    """A q_len above its context: its early rows see nothing and are zeros; the others are right."""
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(12)
    lens, ctx = [long, 2], [long - 2, 40]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    q = torch.from_numpy(rng.standard_normal((sum(lens), hq, d))).to(torch.bfloat16)
    cu = torch.tensor([0, long, long + 2], dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_prefill_fp8(q.cuda(), *pool.device(), 0, bt.cuda(), cu,
                                torch.tensor(ctx, dtype=torch.int32, device="cuda"), long, bs, d ** -0.5,
                                err_flag=err)
    want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, lens, ctx, d ** -0.5)
    check(got, want, torch.bfloat16, d, max(ctx), p_step(torch.bfloat16, True))
    assert (got[:2] == 0).all() and err.item() == 8


@pytest.mark.parametrize("shape", [(12, 2, 128, 16), (4, 2, 40, 16)])
def test_a_context_beyond_its_table_is_cut_and_flagged(ops, shape):
    """Lengths of 2^31 - 1: what the table names is attended, nothing else is read, no call runs on."""
    hq, hkv, d, bs = shape
    rng = np.random.default_rng(13)
    tables, bt, blocks = tables_for(rng, [64, 30], bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    q = torch.from_numpy(rng.standard_normal((2, hq, d))).to(torch.float16)
    ctx = torch.tensor([2 ** 31 - 1, 30], dtype=torch.int32, device="cuda")
    for max_q, cu in ((1, None), (1, [0, 1, 2]), (200, [0, 1, 2])):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        if cu is None:
            got = ops.paged_decode_fp8(q.cuda(), *pool.device(), 0, bt.cuda(), ctx, bs, d ** -0.5, err_flag=err)
        else:
            got = ops.paged_prefill_fp8(q.cuda(), *pool.device(), 0, bt.cuda(),
                                        torch.tensor(cu, dtype=torch.int32, device="cuda"), ctx, max_q, bs,
                                        d ** -0.5, err_flag=err)
        want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, [1, 1], [64, 30], d ** -0.5)
        check(got, want, torch.float16, d, 64, p_step(torch.float16, True))
        assert err.item() == 2


@pytest.mark.parametrize("max_q", [4, 300])
def test_offsets_outside_the_rows_write_nothing_there(ops, max_q):
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(14)
    ctx = [40, 50, 60]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    q = torch.from_numpy(rng.standard_normal((8, hq, d))).to(torch.bfloat16)
    out = torch.full((16, hq, d), 5.0, dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged_prefill_fp8(q.cuda()[:8], *pool.device(), 0, bt.cuda(),
                          torch.tensor([0, 3, 6, 10], dtype=torch.int32, device="cuda"),
                          torch.tensor(ctx, dtype=torch.int32, device="cuda"), max_q, bs, d ** -0.5,
                          out=out[4:12], err_flag=err)
    assert err.item() == 8 and (out[:4] == 5).all() and (out[12:] == 5).all()
    want = ref.attend(q[:6], pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables[:2], [3, 3], ctx[:2],
                      d ** -0.5)
    check(out[4:10], want, torch.bfloat16, d, 50, p_step(torch.bfloat16, True))


# ------------------------------------------------------------------ rows in and out
WRITES = [
    # (hkv, d, bs, [(past, q_len)])
    (2, 128, 16, [(0, 1), (1, 1), (15, 1), (16, 1), (31, 1), (300, 1)]),
    (2, 64, 16, [(0, 40), (10, 3), (13, 7), (15, 1), (5, 100)]),
    (4, 128, 32, [(31, 2), (0, 32), (32, 64), (20, 30)]),
    (1, 40, 8, [(3, 2), (0, 9), (7, 20)]),
    (3, 256, 64, [(60, 10), (0, 0), (0, 65)]),
    (2, 24, 5, [(4, 3), (0, 11)]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("case", WRITES)
def test_write_and_read_back(ops, case, dtype):
    hkv, d, bs, seqs = case
    rng = np.random.default_rng(d + bs)
    q_lens, ctx = [b for _, b in seqs], [a + b for a, b in seqs]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 2, blocks, bs, hkv, d)
    # magnitudes from 2^-20 to 2^14, so that scales grow by anything from nothing to everything
    shape = (sum(q_lens), hkv, d)
    new = [torch.from_numpy(rng.standard_normal(shape) * 2.0 ** rng.integers(-20, 12, (shape[0], hkv, 1))).to(dtype)
           for _ in range(2)]
    dev = pool.device()
    hf = [torch.empty(1, hkv, shape[0], d, dtype=dtype, device="cuda") for _ in range(2)]
    for t, x in zip(hf, new):
        t[0] = x.transpose(0, 1).cuda()
    cu = torch.tensor(np.concatenate([[0], np.cumsum(q_lens)]), dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_write_fp8(*dev, 1, bt.cuda(), cu, torch.tensor(ctx, dtype=torch.int32, device="cuda"),
                     max(q_lens), bs, *(t[0].transpose(0, 1) for t in hf), err_flag=err)
    assert err.item() == 0
    for codes, scales, x in ((pool.k, pool.ks, new[0]), (pool.v, pool.vs, new[1])):
        c, s = codes[1].numpy(), scales[1].numpy()
        ref.write(c, s, bs, tables, q_lens, ctx, x.double().numpy())
    used = np.zeros(blocks * bs, dtype=bool)  # slots of the touched blocks behind the context are free
    for t, a, cx in zip(tables, q_lens, ctx):
        if a:
            used[t[-1] * bs + (cx - 1) % bs + 1:(t[-1] + 1) * bs] = True
    for got, want in zip(dev[:2], (pool.k, pool.v)):
        got = got.view(torch.uint8).cpu()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][~used], want[1][~used])
    for got, want in zip(dev[2:], (pool.ks, pool.vs)):
        assert torch.equal(got.double().cpu(), want)
    slots = torch.from_numpy(np.flatnonzero(~used).astype(np.int32))
    slots = torch.cat([slots, torch.tensor([-1], dtype=torch.int32)])
    for out_dtype in (torch.float32, dtype):
        keys, values = ops.kv_read_fp8(*dev, 1, slots.cuda(), bs, out_dtype)
        for got, codes, scales in ((keys, pool.k, pool.ks), (values, pool.v, pool.vs)):
            at = slots[:-1].long()
            want = torch.from_numpy(ref.VALUES)[codes[1][at].long()] * scales[1][at // bs][:, :, None]
            assert torch.equal(got[:-1].double().cpu(), want.float().to(out_dtype).double())
            assert (got[-1] == 0).all()


def test_write_edges(ops):
    """Zeros, the type's largest values, NaN and infinity; a fresh block clears a NaN scale."""
    hkv, d, bs = 1, 64, 16
    rng = np.random.default_rng(1)
    ctx = [16, 16, 16, 16, 17]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    pool.ks[0, tables[4][1], 0] = float("nan")
    pool.vs[0, tables[4][1], 0] = float("nan")
    dev = pool.device()
    new = torch.zeros(65, hkv, d)
    new[16:32] = torch.from_numpy(rng.standard_normal((16, hkv, d))).float()
    new[20, 0, 3] = float("inf")
    new[32:48] = 1.0
    new[40, 0, 5] = float("nan")
    new[48:64] = 3.3e38
    new[64] = 2.0
    cu = torch.tensor([0, 16, 32, 48, 64, 65], dtype=torch.int32, device="cuda")
    ops.kv_write_fp8(*dev, 0, bt.cuda(), cu, torch.tensor(ctx, dtype=torch.int32, device="cuda"), 16, bs,
                     new.cuda(), -new.cuda())
    for scales, codes, sign in ((dev[2], dev[0], 1), (dev[3], dev[1], -1)):
        s = scales.cpu()[0, :, 0]
        assert s[tables[0][0]] == 2.0 ** -110
        assert s[tables[1][0]].isnan() and s[tables[2][0]].isnan()
        assert s[tables[3][0]] == 2.0 ** 120
        assert s[tables[4][1]] == 2.0 ** -7  # 256 * 2^-7: started anew
    slots = torch.tensor([tables[3][0] * bs, tables[0][0] * bs, tables[1][0] * bs, tables[4][1] * bs],
                         dtype=torch.int32, device="cuda")
    keys, values = ops.kv_read_fp8(*dev, 0, slots, bs, torch.float32)
    assert (keys[0] == 1.875 * 2.0 ** 127).all() and (values[0] == -1.875 * 2.0 ** 127).all()
    assert (keys[1] == 0).all() and keys[2].isnan().all() and (keys[3] == 2).all()


def test_write_appended_one_by_one_keeps_the_rows(ops):
    """Sixteen one-token writes whose magnitudes grow: each older row stays within half a step of
    e4m3 per re-rounding (none while it is in the normal range)."""
    hkv, d, bs = 2, 128, 16
    rng = np.random.default_rng(3)
    tables, bt, blocks = tables_for(rng, [16], bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    dev = pool.device()
    c, s = pool.k[0].numpy(), pool.ks[0].numpy()
    new = rng.standard_normal((16, hkv, d)) * 2.0 ** np.arange(16)[:, None, None]
    new = torch.from_numpy(new).float()
    for t in range(16):
        ops.kv_write_fp8(*dev, 0, bt.cuda(), torch.tensor([0, 1], dtype=torch.int32, device="cuda"),
                         torch.tensor([t + 1], dtype=torch.int32, device="cuda"), 1, bs,
                         new[t:t + 1].cuda(), new[t:t + 1].cuda())
        ref.write(c, s, bs, tables, [1], [t + 1], new[t:t + 1].double().numpy())
    assert torch.equal(dev[0].view(torch.uint8).cpu(), pool.k)
    assert torch.equal(dev[2].double().cpu(), pool.ks)


def test_write_skips_and_flags(ops):
    hkv, d, bs = 2, 64, 16
    rng = np.random.default_rng(2)
    tables, bt, blocks = tables_for(rng, [20, 20, 20], bs)
    bt[1, 1] = blocks
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    before = [t.clone() for t in (pool.k, pool.v)]
    dev = pool.device()
    new = torch.ones(12, hkv, d, dtype=torch.bfloat16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 5, 9, 12], dtype=torch.int32, device="cuda")
    # five rows where four is the bound; a block outside the pool; three rows for a context of 2
    ops.kv_write_fp8(*dev, 0, bt.cuda(), cu, torch.tensor([20, 20, 2], dtype=torch.int32, device="cuda"), 4, bs,
                     new, new, err_flag=err)
    assert err.item() == 8 | 2
    for got, want in zip(dev[:2], before):
        assert torch.equal(got.view(torch.uint8).cpu(), want)
    slots = torch.tensor([blocks * bs], dtype=torch.int32, device="cuda")
    err.zero_()
    keys, _ = ops.kv_read_fp8(*dev, 0, slots, bs, torch.float32, err_flag=err)
    assert err.item() == 1 and (keys == 0).all()


def test_a_second_stream_and_a_captured_step(ops):
    """Write + attend captured once and replayed with new inputs, on a stream of its own."""
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(4)
    ctx = [33, 80, 16]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    dev = pool.device()
    q = torch.zeros(3, hq, d, dtype=torch.bfloat16, device="cuda")
    new = torch.zeros(3, hkv, d, dtype=torch.bfloat16, device="cuda")
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    c, b = torch.tensor(ctx, dtype=torch.int32, device="cuda"), bt.cuda()
    ws = ops.make_fp8_workspace(3, hq, hkv, d, torch.device("cuda"))
    out = torch.empty_like(q)

    def step():
        ops.kv_write_fp8(*dev, 0, b, cu, c, 1, bs, new, new)
        ops.paged_decode_fp8(q, *dev, 0, b, c, bs, d ** -0.5, out=out, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for trial in range(3):
            qh = torch.from_numpy(rng.standard_normal(tuple(q.shape))).to(q.dtype)
            nh = torch.from_numpy(rng.standard_normal(tuple(new.shape))).to(q.dtype)
            q.copy_(qh)
            new.copy_(nh)
            graph.replay()
            side.synchronize()
            for codes, scales in ((dev[0], dev[2]), (dev[1], dev[3])):
                assert codes.is_contiguous() and scales.is_contiguous()
            k8, v8 = (t.view(torch.uint8).cpu()[0] for t in dev[:2])
            ks, vs = (t.double().cpu()[0] for t in dev[2:])
            want = ref.attend(qh, k8, ks, v8, vs, bs, tables, [1] * 3, ctx, d ** -0.5)
            check(out, want, torch.bfloat16, d, max(ctx), p_step(torch.bfloat16, False))
    torch.cuda.current_stream().wait_stream(side)


def test_captured_prompts_replayed_side_by_side(ops):
    """Two captured calls, 64 calls apart, replayed at once on two streams: nothing that one of them
    counts in may be the other's."""
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(11)
    q_lens, ctx = [400, 700, 333], [1500, 700, 2000]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    dev = pool.device()
    q = torch.from_numpy(rng.standard_normal((sum(q_lens), hq, d))).to(torch.bfloat16).cuda()
    cu = torch.tensor([0, *np.cumsum(q_lens)], dtype=torch.int32, device="cuda")
    c, b = torch.tensor(ctx, dtype=torch.int32, device="cuda"), bt.cuda()

    def call(out=None):
        return ops.paged_prefill_fp8(q, *dev, 0, b, cu, c, max(q_lens), bs, d ** -0.5, out=out)

    want = call()
    outs = [torch.empty_like(q) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for out, stream in zip(outs, streams):
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(out)
        graphs.append(graph)
        for _ in range(63):
            call()
    torch.cuda.synchronize()
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out, want)


@pytest.mark.parametrize("hkv,d,dtype", [(3, 64, torch.bfloat16), (1, 128, torch.float16), (5, 32, torch.float32)])
@pytest.mark.parametrize("even", [False, True])
def test_write_of_more_blocks_than_run_at_once(ops, hkv, d, dtype, even):
    """Warps that take many blocks in turn, with sequences that bring nothing or do not fit between them."""
    bs, n = 16, 60
    rng = np.random.default_rng(hkv + d)
    q_lens = [470] * n if even else [int(x) for x in rng.choice([0, 1, 15, 40, 700, 1100], n)]
    past = [int(x) for x in rng.integers(0, 40, n)]
    ctx = [a + b for a, b in zip(past, q_lens)]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    new = [torch.from_numpy(rng.standard_normal((sum(q_lens), hkv, d)) * s).to(dtype) for s in (3.0, 0.01)]
    cu = [0, *np.cumsum(q_lens)]
    dev = pool.device()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = int(np.argmax(q_lens))  # its context is one short of its rows: refused
    told = list(ctx)
    told[bad] = q_lens[bad] - 1
    ops.kv_write_fp8(*dev, 0, bt.cuda(), torch.tensor(cu, dtype=torch.int32, device="cuda"),
                     torch.tensor(told, dtype=torch.int32, device="cuda"), max(q_lens), bs, new[0].cuda(),
                     new[1].cuda(), err_flag=err)
    assert err.item() == 8
    fits = [i for i in range(n) if i != bad]
    rows = np.concatenate([np.arange(cu[i], cu[i + 1]) for i in fits])
    for codes, scales, x in ((pool.k, pool.ks, new[0]), (pool.v, pool.vs, new[1])):
        ref.write(codes[0].numpy(), scales[0].numpy(), bs, [tables[i] for i in fits], [q_lens[i] for i in fits],
                  [ctx[i] for i in fits], x.double().numpy()[rows])
    used = np.zeros(blocks * bs, dtype=bool)  # slots of the touched blocks behind the context are free
    for i in fits:
        if q_lens[i]:
            last = tables[i][(ctx[i] - 1) // bs]
            used[last * bs + (ctx[i] - 1) % bs + 1:(last + 1) * bs] = True
    for got, want in zip(dev[:2], (pool.k, pool.v)):
        assert torch.equal(got.view(torch.uint8).cpu()[0][~used], want[0][~used])
    for got, want in zip(dev[2:], (pool.ks, pool.vs)):
        assert torch.equal(got.double().cpu(), want)
