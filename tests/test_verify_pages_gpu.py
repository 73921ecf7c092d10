"""Draft verification and page moves against their plain forms. Every result is a whole number or
a copy, so everything has to be equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ref

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def run_verify(ops, target, draft, tokens, cu, accept, sample, max_k, err=None, rows=None):
    got = ops.verify_drafts(target if rows is None else rows, torch.tensor(tokens, dtype=torch.int64, device="cuda"),
                            i32(cu), torch.tensor(accept, dtype=torch.float32, device="cuda"),
                            torch.tensor(sample, dtype=torch.float32, device="cuda"), max_k,
                            draft_probs=draft, err_flag=err)
    want = ref.verify(target.double().cpu().numpy(), None if draft is None else draft.double().cpu().numpy(),
                      tokens, cu, np.float32(accept).astype(np.float64), np.float32(sample).astype(np.float64), max_k)
    assert got[0].tolist() == want[0]
    assert got[1].tolist() == want[1]
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 7, 100, 1001, 32000, 151936])
def test_verify(ops, vocab, with_draft, dtype):
    rng = np.random.default_rng(vocab)
    ks = [0, 1, 3, 5, 0, 2, 8, 4]
    cu = np.concatenate([[0], np.cumsum(ks)]).tolist()
    n, t = len(ks), cu[-1]
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(t + n, vocab, generator=g) * 3
    target = torch.softmax(logits, -1).to(dtype).cuda()
    rows = torch.arange(t) + torch.repeat_interleave(torch.arange(n), torch.tensor(ks))
    q = torch.softmax(logits[rows] + torch.randn(t, vocab, generator=g) * 0.5, -1)
    tokens = torch.multinomial(q, 1, generator=g)[:, 0].tolist()
    draft = q.to(dtype).cuda() if with_draft else None
    run_verify(ops, target, draft, tokens, cu, rng.random(t), rng.random(n), 8)


def test_verify_extreme_draws_and_ties(ops):
    """Equal rows (p = q: every draft stands), draws of 0 and of the largest fp32 below 1, exact
    borders of the running sum, zeros in front, behind and between."""
    top = float(np.nextafter(np.float32(1), np.float32(0)))
    p = torch.zeros(8, 64)
    p[:, 4:8] = 0.25
    target = p.cuda()
    for sample, token in ((0.0, 4), (0.25, 5), (0.5, 6), (top, 7)):
        want = run_verify(ops, target, None, [], [0] * 9, [], [sample] * 8, 0)
        assert [w[0] for w in want[0]] == [token] * 8
    # p = q: u q < p for every u < 1
    q = p[:4].cuda()
    want = run_verify(ops, p[:6].cuda(), q, [4, 5, 6, 7], [0, 2, 4], [top, 0.5, 0.0, top], [0.1, 0.9], 2)
    assert want[1] == [2, 2]
    # the residual is zero everywhere but the draft is rejected (q above p): the target row itself
    q2 = torch.full((1, 64), 0.5).cuda()
    want = run_verify(ops, p[:2].cuda(), q2, [4], [0, 1], [0.9], [0.6], 1)
    assert want[0][0][0] == 6
    # the rejected token is the only one of the target row: it is drawn again only without p - q
    only = torch.zeros(2, 64)
    only[:, 3] = 1.0
    run_verify(ops, only.cuda(), None, [9], [0, 1], [0.5], [0.5], 1)
    run_verify(ops, torch.zeros(2, 64).cuda(), None, [9], [0, 1], [0.5], [0.5], 1)  # token 0


def test_verify_nan_and_negative_entries_count_as_zero(ops):
    p = torch.rand(3, 500)
    p[:, 100:200] = float("nan")
    p[:, 300:310] = -1.0
    q = torch.rand(2, 500) * 2
    q[0, 50] = float("nan")
    for draft in (None, q.cuda()):
        run_verify(ops, p.cuda(), draft, [150, 7], [0, 2], [0.1, 0.9], [0.77], 2)


def test_verify_strided_rows_and_unaligned_starts(ops):
    g = torch.Generator().manual_seed(3)
    big = torch.rand(9, 1003, generator=g)
    big /= big.sum(1, keepdim=True)
    target = big.cuda()[:, 1:1000]   # rows 1003 apart, first element 4 bytes past a boundary
    draft = big.cuda()[:6, 3:1002]
    ks = [2, 1, 3]
    run_verify(ops, target, draft, [4, 100, 998, 5, 6, 7], [0, 2, 3, 6], [0.9, 0.2, 0.7, 0.1, 0.99, 0.5],
               [0.3, 0.5, 0.99], max(ks), rows=target)


def test_verify_flags(ops):
    err = i32([0])
    p = torch.softmax(torch.randn(7, 50), -1).cuda()
    # an id outside the vocabulary is rejected
    want = run_verify(ops, p[:5], None, [3, 50, -1], [0, 2, 3], [0.0, 0.0, 0.0], [0.5, 0.5], 3, err)
    assert want[1] == [1, 0] and err.item() == 16
    # more drafts than max_drafts: -1 everywhere, the others are right
    err.zero_()
    got = ops.verify_drafts(p[:6], torch.tensor([1, 2, 3, 4], device="cuda"), i32([0, 3, 4]),
                            torch.zeros(4, device="cuda"), torch.zeros(2, device="cuda"), 2, err_flag=err)
    assert got[0][0].tolist() == [-1, -1, -1] and got[1].tolist() == [0, 1]
    assert got[0][1][0] == 4 and err.item() == 8


def test_verify_follows_the_target_distribution(ops):
    """What speculative sampling promises: the first token is distributed as p, whatever q is. A
    count of N draws with probability p is within 6 standard deviations of N p (2e-9 a side)."""
    vocab, n = 6, 40000
    p = torch.tensor([0.4, 0.05, 0.2, 0.05, 0.25, 0.05])
    q = torch.tensor([0.1, 0.3, 0.2, 0.15, 0.05, 0.2])
    g = torch.Generator(device="cuda").manual_seed(0)
    target = p.repeat(2 * n, 1).cuda()
    draft = q.repeat(n, 1).cuda()
    tokens = torch.multinomial(draft, 1, generator=g)[:, 0]
    got, _ = ops.verify_drafts(target, tokens, torch.arange(n + 1, dtype=torch.int32, device="cuda"),
                               torch.rand(n, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda"),
                               1, draft_probs=draft)
    counts = torch.bincount(got[:, 0], minlength=vocab).double().cpu()
    assert ((counts - n * p.double()).abs() <= 6 * (n * p * (1 - p)).double().sqrt()).all(), counts / n


def test_verify_greedy(ops):
    rng = np.random.default_rng(0)
    ks = [0, 1, 4, 40, 33, 2]
    cu = np.concatenate([[0], np.cumsum(ks)]).tolist()
    ids = torch.from_numpy(rng.integers(0, 3, cu[-1] + len(ks)))
    tokens, want, counts = [], [], []
    for i, k in enumerate(ks):
        line = ids[cu[i] + i:cu[i] + i + k].tolist()
        if k and i != 3:  # sequence 3 keeps every draft
            line[int(rng.integers(0, k))] += 1
        n = next((j for j, x in enumerate(line) if x != ids[cu[i] + i + j]), k)
        tokens += line
        want.append(line[:n] + [int(ids[cu[i] + i + n])] + [-1] * (40 - n))
        counts.append(n)
    got = ops.verify_drafts_greedy(ids.cuda(), torch.tensor(tokens, device="cuda"), i32(cu), 40)
    assert got[0].tolist() == want and got[1].tolist() == counts


# ------------------------------------------------------------------ pages
def pool(seed, dtype, layers, blocks, bs, hkv, d):
    g = torch.Generator().manual_seed(seed)
    shape = (layers, blocks * bs, hkv, d)
    if dtype == FP8:
        k, v = (torch.randint(0, 256, shape, generator=g, dtype=torch.uint8) for _ in range(2))
        ks, vs = (torch.rand(layers, blocks, hkv, generator=g) for _ in range(2))
        return [k.cuda().view(FP8), v.cuda().view(FP8), ks.cuda(), vs.cuda()]
    return [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2)] + [None, None]


def raw(t, bs):
    """(layers, blocks, bytes) of a pool tensor, (layers, blocks, heads) of scales."""
    if t is None or t.dim() == 3:
        return t
    return t.view(torch.uint8).reshape(t.shape[0], t.shape[1] // bs, -1)


PAGES = [(3, 40, 16, 2, 128), (1, 65, 5, 1, 24), (28, 33, 16, 2, 64), (2, 12, 64, 4, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, FP8])
@pytest.mark.parametrize("shape", PAGES)
def test_copy_blocks(ops, shape, dtype):
    layers, blocks, bs, hkv, d = shape
    p = pool(1, dtype, *shape)
    ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(2)).tolist()
    src, dst = [ids[0], ids[0], -1, ids[1], ids[2], ids[3]], [ids[4], ids[5], ids[6], -1, ids[7], ids[3]]
    want = [None if t is None else raw(t, bs).clone() for t in p]
    for s, t in zip(src, dst):
        if s >= 0 and t >= 0:
            for w in want:
                if w is not None:
                    w[:, t] = w[:, s]
    err = i32([0])
    ops.copy_blocks(p[0], p[1], i32(src + [blocks]), i32(dst + [ids[8]]), bs, p[2], p[3], err_flag=err)
    assert err.item() == 2  # the block past the pool: skipped
    for t, w in zip(p, want):
        assert t is None or torch.equal(raw(t, bs), w)
    ops.copy_blocks(p[0], p[1], i32([]), i32([]), bs, p[2], p[3])


@pytest.mark.parametrize("dtype", [torch.float16, FP8])
@pytest.mark.parametrize("blocks,fill", [(64, 0.0), (64, 1.0), (40, 0.5), (333, 0.3), (333, 0.9), (5000, 0.6)])
def test_compact_blocks(ops, blocks, fill, dtype):
    layers, bs, hkv, d = 2, 16, 2, 64
    rng = np.random.default_rng(blocks + int(fill * 10))
    p = pool(blocks, dtype, layers, blocks, bs, hkv, d)
    ids = rng.permutation(blocks)[:round(blocks * fill)].tolist()
    n = 7
    tables = [ids[i::n] for i in range(n)]
    if len(tables[1]) > 1:
        tables[1] = tables[0][:1] + tables[1][1:]  # a shared first page
    ctx = [max(0, len(t) * bs - int(rng.integers(0, bs))) for t in tables]
    ctx[2] = 0  # a finished sequence: its row names blocks that are not live
    width = max(1, max(len(t) for t in tables) + 2)
    bt = torch.full((n, width), -1, dtype=torch.int32)
    for i, t in enumerate(tables):
        bt[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    moves, new, live = ref.compact(tables, ctx, bs, blocks)
    want = [None if t is None else raw(t, bs).clone() for t in p]
    for s, t in moves:
        for w in want:
            if w is not None:
                w[:, t] = w[:, s]
    want_bt = bt.clone()
    for i, c in enumerate(ctx):
        for j in range(-(-c // bs)):
            want_bt[i, j] = new[bt[i, j]]
    err, dev_bt = i32([0]), bt.cuda()
    got_new, got_live = ops.compact_blocks(p[0], p[1], dev_bt, i32(ctx), bs, p[2], p[3], err_flag=err)
    assert err.item() == 0 and got_live.tolist() == [live] and got_new.tolist() == new
    assert torch.equal(dev_bt.cpu(), want_bt)
    for t, w in zip(p, want):
        assert t is None or torch.equal(raw(t, bs), w)


def test_compact_flags_bad_tables(ops):
    p = pool(0, torch.bfloat16, 1, 10, 16, 1, 64)
    before = [t.clone() for t in p[:2]]
    bt, err = i32([[9, 12, 3], [-1, 0, 1]]), i32([0])
    new, live = ops.compact_blocks(p[0], p[1], bt, i32([40, 70]), 16, err_flag=err)
    assert err.item() == 8 | 2 and live.item() == 4  # blocks 9, 3, 0, 1
    assert new.tolist() == [0, 1, -1, 3, -1, -1, -1, -1, -1, 2]
    assert bt.tolist() == [[2, 12, 3], [-1, 0, 1]]
    for t, b in zip(p, before):
        assert torch.equal(t[:, 32:48], b[:, 144:160])


@pytest.mark.parametrize("blocks,width", [(3000, 1170), (3000, 1171), (2049, 4000), (40, 9000)])
def test_compact_wide_tables(ops, blocks, width):
    """Tables of up to and over what one CTA looks through, pools that end inside a word of bits."""
    n, bs = 7, 16
    rng = np.random.default_rng(width)
    p = pool(3, torch.bfloat16, 1, blocks, bs, 1, 8)
    ids = rng.permutation(blocks)[:blocks * 3 // 5].tolist()
    cuts = sorted(rng.integers(0, len(ids) + 1, n - 1).tolist())
    tables = [ids[a:b][:width] for a, b in zip([0, *cuts], [*cuts, len(ids)])]
    ctx = [max(0, len(t) * bs - int(rng.integers(0, bs))) for t in tables]
    bt = torch.from_numpy(rng.integers(0, blocks, (n, width))).to(torch.int32)  # stale ids behind the context
    for i, t in enumerate(tables):
        bt[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
    moves, new, live = ref.compact(tables, ctx, bs, blocks)
    want = [raw(t, bs).clone() for t in p[:2]]
    for s, t in moves:
        for w in want:
            w[:, t] = w[:, s]
    want_bt = bt.clone()
    for i, c in enumerate(ctx):
        used = -(-c // bs)
        want_bt[i, :used] = torch.tensor(new, dtype=torch.int32)[bt[i, :used].long()]
    err, dev_bt = i32([0]), bt.cuda()
    got_new, got_live = ops.compact_blocks(p[0], p[1], dev_bt, i32(ctx), bs, err_flag=err)
    assert err.item() == 0 and got_live.tolist() == [live] and got_new.tolist() == new
    assert torch.equal(dev_bt.cpu(), want_bt)
    for t, w in zip(p, want):
        assert torch.equal(raw(t, bs), w)
