"""Many-row calls over the 8-bit cache whose tables are wider than the pool: the 16-bit copy then keeps
the pool's block ids. Tolerances are those of test_fp8_cache_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ref
from test_fp8_cache_gpu import Pool, check, p_step, tables_for

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def widened(bt, width):
    wide = torch.full((bt.shape[0], width), -1, dtype=torch.int32)
    wide[:, :bt.shape[1]] = bt
    return wide


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,bs", [(128, 16), (64, 32), (64, 48)])
def test_tables_wider_than_the_pool(ops, d, bs, dtype):
    """The same histories through narrow tables and through ones that name more blocks than there are."""
    hq, hkv = 6, 2
    rng = np.random.default_rng(d + bs)
    q_lens, past = [200, 1, 90, 300], [40, 700, 0, 513]
    ctx = [a + b for a, b in zip(past, q_lens)]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    pool.poison_unused(tables, ctx)
    q = torch.from_numpy(rng.standard_normal((sum(q_lens), hq, d))).to(dtype)
    cu = i32([0, *np.cumsum(q_lens)])
    want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, q_lens, ctx, d ** -0.5)
    for width in (bt.shape[1], blocks, 3000):
        err = i32([0])
        got = ops.paged_prefill_fp8(q.cuda(), *pool.device(), 0, widened(bt, width).cuda(), cu, i32(ctx), max(q_lens),
                                    bs, d ** -0.5, err_flag=err)
        check(got, want, dtype, d, max(ctx), p_step(dtype, True))
        assert err.item() == 0


@pytest.mark.parametrize("width", [30, 400])
def test_sequences_that_share_blocks(ops, width):
    """Forks: shared full blocks, and two sequences that end at different tokens of one block."""
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(2)
    tables = [list(range(20)), list(range(12)) + [25, 26], list(range(18)), [26, 25, 3]]
    q_lens, ctx = [150, 40, 130, 37], [313, 217, 280, 37]
    bt = torch.full((4, width), -1, dtype=torch.int32)
    for row, t in zip(bt, tables):
        row[:len(t)] = torch.tensor(t, dtype=torch.int32)
    pool = Pool(rng, 1, 40, bs, hkv, d)
    q = torch.from_numpy(rng.standard_normal((sum(q_lens), hq, d))).to(torch.bfloat16)
    cu = i32([0, *np.cumsum(q_lens)])
    got = ops.paged_prefill_fp8(q.cuda(), *pool.device(), 0, bt.cuda(), cu, i32(ctx), max(q_lens), bs, d ** -0.5)
    want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, q_lens, ctx, d ** -0.5)
    check(got, want, torch.bfloat16, d, max(ctx), p_step(torch.bfloat16, True))


def test_a_bad_block_is_flagged_in_a_wide_table(ops):
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(3)
    q_lens, ctx = [140, 150], [180, 150]
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    q = torch.from_numpy(rng.standard_normal((290, hq, d))).to(torch.bfloat16)
    want = ref.attend(q, pool.k[0], pool.ks[0], pool.v[0], pool.vs[0], bs, tables, q_lens, ctx, d ** -0.5)
    for bad in (blocks, 2 ** 31 - 1, -5):
        wide = widened(bt, 500)
        wide[0, 3] = bad
        err = i32([0])
        got = ops.paged_prefill_fp8(q.cuda(), *pool.device(), 0, wide.cuda(), i32([0, 140, 290]), i32(ctx), 150, bs,
                                    d ** -0.5, err_flag=err)
        assert err.item() == 2
        check(got[140:], tuple(t[140:] for t in want), torch.bfloat16, d, 180, p_step(torch.bfloat16, True))


def test_what_a_call_allocates_follows_the_pool(ops):
    """Sixteen short prompts through tables of 65,536 tokens: 1.07 GB by the entries, 3.5 MB by the pool."""
    hq, hkv, d, bs, n = 12, 2, 128, 16, 16
    rng = np.random.default_rng(4)
    ctx = [200] * n
    tables, bt, blocks = tables_for(rng, ctx, bs)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    dev = pool.device()
    q = torch.from_numpy(rng.standard_normal((sum(ctx), hq, d))).to(torch.bfloat16).cuda()
    bt, cu, c = widened(bt, 4096).cuda(), i32([0, *np.cumsum(ctx)]), i32(ctx)
    out = torch.empty_like(q)
    ws = ops.make_fp8_workspace(n, hq, hkv, d, torch.device("cuda"))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    ops.paged_prefill_fp8(q, *dev, 0, bt, cu, c, 200, bs, d ** -0.5, out=out, workspace=ws)
    taken = torch.cuda.max_memory_allocated() - before
    # K and V of the pool in 16 bits, and the partial results of at most eight runs
    assert taken <= 2 * blocks * bs * hkv * d * 2 + 8 * q.numel() * 4 * (1 + 1 / d) + (1 << 20)


@pytest.mark.parametrize("q_lens,past", [([200, 90, 300], [40, 0, 513]), ([130], [2300]), ([5, 3], [90, 7])])
def test_a_bound_on_the_contexts(ops, q_lens, past):
    """Wide tables with a bound: the narrow tables' results, bit for bit, and their scratch. A context
    past the bound is cut to the blocks that the bound covers, and flagged, in the many-row form."""
    hq, hkv, d, bs = 12, 2, 128, 16
    rng = np.random.default_rng(len(q_lens))
    ctx = [a + b for a, b in zip(past, q_lens)]
    tables, bt, blocks = tables_for(rng, ctx, bs, spare=4000)
    pool = Pool(rng, 1, blocks, bs, hkv, d)
    dev = pool.device()
    q = torch.from_numpy(rng.standard_normal((sum(q_lens), hq, d))).to(torch.bfloat16).cuda()
    cu = i32([0, *np.cumsum(q_lens)])
    ws = ops.make_fp8_workspace(len(ctx), hq, hkv, d, torch.device("cuda"), max(q_lens))

    def call(table, **kw):
        err, out = i32([0]), torch.empty_like(q)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        ops.paged_prefill_fp8(q, *dev, 0, table, cu, i32(ctx), max(q_lens), bs, d ** -0.5, out=out, workspace=ws,
                              err_flag=err, **kw)
        taken = torch.cuda.max_memory_allocated() - before
        return out, err.item(), taken

    narrow, flag, least = call(bt.cuda())
    assert flag == 0
    for bound in (max(ctx), bt.shape[1] * bs):
        got, flag, taken = call(widened(bt, 1000).cuda(), max_context=bound)
        assert torch.equal(got, narrow) and taken <= least + (1 << 16) and flag == 0
    if max(q_lens) > 5:
        got, flag, _ = call(widened(bt, 1000).cuda(), max_context=max(ctx) - 20)
        assert flag == 2
    with pytest.raises(ValueError, match="max_context"):
        call(bt.cuda(), max_context=-1)
