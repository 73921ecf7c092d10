"""Plain 64-bit forms of the 8-bit cache, of attention over it, of draft verification and of
page moves (test infrastructure: the product never imports it).

An 8-bit cache is held here as uint8 codes and float64 scales. The 256 code values are built
from the e4m3 definition, and rounding is a search of that table (ties to the even code), so
nothing here shares arithmetic with the kernels.
"""

from __future__ import annotations

import numpy as np
import torch

MIN_EXP = -110
SATURATE = 1.875 * 2.0 ** 127  # finite rows above this are stored as this


def _code_values() -> np.ndarray:
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if e == 15 and m == 7:
            v = np.nan
        out[c] = -v if c & 128 else v
    return out


VALUES = _code_values()
_POSITIVE = VALUES[:127]


def encode(x: np.ndarray) -> np.ndarray:
    """The nearest code of each |x| <= 448, ties to the even code."""
    a = np.abs(x)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 1, 126)
    lo = hi - 1
    dl, dh = a - _POSITIVE[lo], _POSITIVE[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def block_scale(amax: float) -> float:
    e = MIN_EXP
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write(codes, scales, block_size, tables, q_lens, ctx, new):
    """Append packed rows ``new`` (rows, heads, dim; float64) to one layer's codes [slots, heads,
    dim] and scales [blocks, heads], in place."""
    row = 0
    for i, (a, c) in enumerate(zip(q_lens, ctx)):
        start = c - a
        for b in range(start // block_size, -(-c // block_size)):
            lo, hi = max(start, b * block_size), min(c, (b + 1) * block_size)
            if lo >= hi:
                continue
            blk = tables[i][b]
            off = lo - b * block_size
            base = blk * block_size
            for h in range(new.shape[1]):
                x = new[row + lo - start:row + hi - start, h]
                old = scales[blk, h]
                if not np.isfinite(x).all() or (off and not np.isfinite(old)):
                    scales[blk, h] = np.nan
                    codes[base + off:base + off + hi - lo, h] = 0
                    continue
                x = np.clip(x, -SATURATE, SATURATE)
                s = block_scale(np.abs(x).max())
                if off:
                    s = max(s, old)
                    if s != old:
                        held = VALUES[codes[base:base + off, h]] * (old / s)
                        codes[base:base + off, h] = encode(held)
                scales[blk, h] = s
                codes[base + off:base + off + hi - lo, h] = encode(x / s)
        row += a


def attend(q, kc, ks, vc, vs, block_size, tables, q_lens, ctx, scale):
    """(out, mass, score) in float64: the attention rows; per (row, head) the largest over the
    head dims of sum_t p_t |v_t|; and the largest of sum_d |q_d k_d| * scale (what rounding
    errors of P, V and of the scores are relative to)."""
    q = q.double()
    kc, vc = torch.from_numpy(VALUES)[kc.long()], torch.from_numpy(VALUES)[vc.long()]
    out = torch.zeros_like(q)
    mass, score = torch.zeros(q.shape[:2]).double(), torch.zeros(q.shape[:2]).double()
    row, group = 0, q.shape[1] // kc.shape[1]
    for i, (a, c) in enumerate(zip(q_lens, ctx)):
        if a == 0:
            continue
        pos = torch.arange(c)
        blk = torch.tensor(tables[i], dtype=torch.int64)[pos // block_size] if c else pos
        slot = blk * block_size + pos % block_size
        k, v = kc[slot] * ks[blk][:, :, None], vc[slot] * vs[blk][:, :, None]
        for j in range(a):
            n = c - a + j + 1
            if n <= 0:
                continue
            for h in range(q.shape[1]):
                x, g = q[row + j, h], h // group
                p = torch.softmax(k[:n, g] @ x * scale, 0)
                out[row + j, h] = p @ v[:n, g]
                mass[row + j, h] = (p @ v[:n, g].abs()).max()
                score[row + j, h] = (k[:n, g].abs() @ x.abs()).max() * scale
        row += a
    return out, mass, score


def verify(target, draft, tokens, cu, accept, sample, max_drafts):
    """(tokens, accepted) as lists; target/draft float64 arrays, draft None for certain drafts.
    NaN and negative entries of either count as zero."""
    target = np.where(target > 0, target, 0.0)
    draft = None if draft is None else np.where(draft > 0, draft, 0.0)
    out, counts = [], []
    for i in range(len(cu) - 1):
        k, n = cu[i + 1] - cu[i], 0
        vocab = target.shape[1]
        while n < k:
            t = cu[i] + n
            x = tokens[t]
            if not 0 <= x < vocab:
                break
            qx = draft[t, x] if draft is not None else 1.0
            if not accept[t] * qx < target[t + i, x]:
                break
            n += 1
        p = target[cu[i] + i + n]
        r = p
        if n < k:
            t = cu[i] + n
            if draft is not None:
                d = target[t + i] - draft[t]
                r = np.where(d > 0, d, 0.0)
            else:
                r = p.copy()
                if 0 <= tokens[t] < vocab:
                    r[tokens[t]] = 0.0
            if not r.sum() > 0:
                r = p
        cdf = np.cumsum(r)
        past = np.nonzero(cdf > sample[i] * cdf[-1])[0]
        some = np.nonzero(r > 0)[0]
        pick = int(past[0]) if past.size else int(some[-1]) if some.size else 0
        out.append([int(t) for t in tokens[cu[i]:cu[i] + n]] + [pick] + [-1] * (max_drafts - n))
        counts.append(n)
    return out, counts


def compact(tables, ctx, block_size, num_blocks):
    """(moves [(src, dst)], new_ids, num_live) of packing the live blocks to the front."""
    live = sorted({b for t, c in zip(tables, ctx) for b in t[:-(-c // block_size)]})
    n = len(live)
    free = [b for b in range(n) if b not in set(live)]
    moves = list(zip([b for b in live if b >= n], free))
    new = [-1] * num_blocks
    for b in live:
        new[b] = b
    for s, d in moves:
        new[s] = d
    return moves, new, n
