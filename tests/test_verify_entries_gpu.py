"""Draft verification with NaN and negative probabilities on either side: they count as zero, in
the acceptance, in the residual and in the row that is drawn from. Whole numbers: all equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import fp8 as ref

pytestmark = pytest.mark.gpu


def verify(ops, target, draft, tokens, cu, accept, sample, max_k):
    got = ops.verify_drafts(target.cuda(), torch.tensor(tokens, dtype=torch.int64, device="cuda"),
                            torch.tensor(cu, dtype=torch.int32, device="cuda"),
                            torch.tensor(accept, dtype=torch.float32, device="cuda"),
                            torch.tensor(sample, dtype=torch.float32, device="cuda"), max_k,
                            draft_probs=draft.cuda())
    return got[0].tolist(), got[1].tolist()


NAN = float("nan")


def test_one_entry_at_the_drafted_token(ops):
    """(q, p) of the drafted token: what is not positive is zero, and the draft stands while
    u * q < p."""
    cases = [(NAN, 0.5, True), (-1.0, 0.5, True), (NAN, 0.0, False), (-1.0, 0.0, False), (-1.0, -0.5, False),
             (NAN, NAN, False), (0.5, NAN, False), (0.5, -1.0, False), (-2.0, -1.0, False), (0.25, 0.5, True)]
    for q, p, stands in cases:
        target = torch.full((2, 8), 0.125)
        draft = torch.full((1, 8), 0.125)
        target[0, 3], draft[0, 3] = p, q
        _, accepted = verify(ops, target, draft, [3], [0, 1], [0.5], [0.5], 1)
        assert accepted == [int(stands)], (q, p)


def test_draft_entries_that_are_not_positive_take_nothing_away(ops):
    """The residual of a rejected row: p where q is NaN or negative, 0 where p is."""
    target = torch.zeros(2, 64)
    draft = torch.zeros(1, 64)
    target[0, [5, 9, 20]] = torch.tensor([0.25, 0.25, 0.5])
    draft[0, 5], draft[0, 9], draft[0, 40] = NAN, -3.0, 1.0
    target[0, 50], draft[0, 50] = -0.25, -4.0
    target[0, 51], draft[0, 51] = NAN, -4.0
    for u, token in ((0.0, 5), (0.2, 5), (0.25, 9), (0.45, 9), (0.5, 20), (0.99, 20)):
        tokens, accepted = verify(ops, target, draft, [40], [0, 1], [0.5], [u], 1)
        assert accepted == [0] and tokens[0][0] == token, u


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [3, 129, 5000, 151936])
def test_rows_with_entries_of_both_kinds(ops, vocab, dtype):
    rng = np.random.default_rng(vocab)
    g = torch.Generator().manual_seed(vocab)
    ks = [3, 1, 0, 4, 2, 5]
    cu = np.concatenate([[0], np.cumsum(ks)]).tolist()
    t, n = cu[-1], len(ks)
    target = torch.softmax(torch.randn(t + n, vocab, generator=g) * 2, -1).to(dtype)
    draft = torch.softmax(torch.randn(t, vocab, generator=g) * 2, -1).to(dtype)
    for rows, share in ((target, 0.2), (draft, 0.4)):
        pick = torch.rand(rows.shape, generator=g)
        rows[pick < share / 2] = NAN
        rows[(pick >= share / 2) & (pick < share)] *= -1
    tokens = rng.integers(0, vocab, t).tolist()
    accept = rng.random(t).astype(np.float32)
    sample = rng.random(n).astype(np.float32)
    got = verify(ops, target, draft, tokens, cu, accept, sample, 5)
    want = ref.verify(target.double().numpy(), draft.double().numpy(), tokens, cu, accept.astype(np.float64),
                      sample.astype(np.float64), 5)
    assert got == (want[0], want[1])
