"""Workloads of the 8-bit KV cache, the verification of drafted tokens and the page moves.

Three families of operators, each in its plain form (elementary torch operations in 32 or
64 bits) and, where ``own`` is true, through the framework's calls:

* ``rows``    new K/V rows into an 8-bit paged cache and the touched rows back as values;
* ``attend``  causal attention over the 8-bit cache: one query token per sequence
              (``decode``), or ``q_len`` of them (drafted tokens, prompt slices, prompts);
* ``drafts``  verification of drafted tokens against target probabilities;
* ``fork``    copies of pages over all layers (the partial last pages of forked sequences);
* ``compact`` live pages moved to the front of the pool, block tables rewritten.

The 8-bit cache holds e4m3 codes and one power-of-two scale for each (layer, block, KV
head): 2**e with the smallest e >= -110 for which the block's largest magnitude is at most
448 * 2**e. A write that covers a block's first slot starts the block anew; any other write
keeps the larger of the old scale and the one its rows need, and the rows already there are
rounded to the new scale.
"""

import math
import random

import torch

own = False

FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}
MIN_EXP = -110


# ---------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step's new rows of 256 running sequences (latency of a small call)
        {"name": "rows-step", "op": "rows", "n": 256, "q_lo": 1, "q_hi": 1, "past_lo": 512,
         "past_hi": 4095, "hkv": 2, "d": 128, "bs": 16, "type": "bf16", "layers": 2},
        # a whole packed prefill of 32 prompts enters the cache
        {"name": "rows-prompts", "op": "rows", "n": 32, "q_lo": 64, "q_hi": 8192, "past_lo": 0,
         "past_hi": 0, "hkv": 2, "d": 128, "bs": 16, "type": "f16", "layers": 1},
        # one user, one short history: the smallest decode call
        {"name": "decode-one", "op": "decode", "n": 1, "lo": 333, "hi": 333, "hq": 14, "hkv": 2,
         "d": 64, "bs": 16, "type": "f16", "layers": 2},
        # the ordinary decode step: 256 sequences, contexts 512 to 4096
        {"name": "decode-256", "op": "decode", "n": 256, "lo": 512, "hi": 4096, "hq": 12, "hkv": 2,
         "d": 128, "bs": 16, "type": "bf16", "layers": 1},
        # long contexts, where an 8-bit cache matters most
        {"name": "decode-long", "op": "decode", "n": 64, "lo": 8192, "hi": 32768, "hq": 28, "hkv": 4,
         "d": 128, "bs": 16, "type": "bf16", "layers": 1},
        # drafted tokens of 128 sequences scored in one call (1 to 6 rows each)
        {"name": "rows-of-drafts", "op": "attend", "n": 128, "q_lo": 1, "q_hi": 6, "past_lo": 512,
         "past_hi": 4090, "hq": 12, "hkv": 2, "d": 128, "bs": 16, "type": "bf16", "layers": 1},
        # four 512-token prompt slices over the history before them, as a mixed step carries
        {"name": "slices", "op": "attend", "n": 4, "q_lo": 512, "q_hi": 512, "past_lo": 100,
         "past_hi": 7777, "hq": 14, "hkv": 2, "d": 64, "bs": 16, "type": "f16", "layers": 1},
        # 32 whole prompts, 64 to 8192 tokens
        {"name": "prompts", "op": "attend", "n": 32, "q_lo": 64, "q_hi": 8192, "past_lo": 0,
         "past_hi": 0, "hq": 12, "hkv": 2, "d": 128, "bs": 16, "type": "bf16", "layers": 1},
        # one user with four drafted tokens
        {"name": "drafts-one", "op": "drafts", "n": 1, "k_lo": 4, "k_hi": 4, "vocab": 151936,
         "type": "f32", "draft_probs": True, "match": 0.6},
        # 256 users with 1 to 5 drafted tokens, a draft model's probabilities at hand
        {"name": "drafts-256", "op": "drafts", "n": 256, "k_lo": 1, "k_hi": 5, "vocab": 151936,
         "type": "f32", "draft_probs": True, "match": 0.8},
        # 64 sequences forked: their last pages copied in every layer of an 8-bit cache
        {"name": "fork-64", "op": "fork", "pairs": 64, "blocks": 4096, "layers": 28, "hkv": 2,
         "d": 128, "bs": 16, "type": "fp8"},
        # a 28-layer cache, 55 % in use and scattered, packed to its front
        {"name": "compact-28", "op": "compact", "n": 48, "blocks": 4096, "live": 0.55, "layers": 28,
         "hkv": 2, "d": 128, "bs": 16, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = ((12, 2, 128), (14, 2, 64), (28, 4, 128), (8, 1, 128), (32, 2, 128), (4, 4, 64), (16, 8, 128))


def draw(rng):
    op = rng.choice(("rows", "decode", "decode", "attend", "attend", "drafts", "fork", "compact"))
    hq, hkv, d = rng.choice(HEADS)
    bs = rng.choice((16, 16, 32, 64))
    kind = rng.choice(("bf16", "f16"))
    if op == "decode":
        n = _log(rng, 1, 256)
        hi = _log(rng, 17, min(32768, max(64, 1200000 // n)))
        return {"op": op, "n": n, "lo": rng.randint(1, hi), "hi": hi, "hq": hq, "hkv": min(hkv, 4),
                "d": d, "bs": bs, "type": kind, "layers": rng.randint(1, 2)} if hq % min(hkv, 4) == 0 else draw(rng)
    if op in ("rows", "attend"):
        few = rng.random() < 0.5
        n = _log(rng, 1, 192 if few else 32)
        q_hi = rng.randint(1, 9) if few else _log(rng, 16, 4096)
        past = _log(rng, 1, 4000) if few or rng.random() < 0.5 else 0
        case = {"op": op, "n": n, "q_lo": rng.randint(1, q_hi), "q_hi": q_hi,
                "past_lo": rng.randint(0, past), "past_hi": past, "hkv": hkv, "d": d, "bs": bs,
                "type": kind if op == "attend" else rng.choice(("bf16", "f16", "f32")),
                "layers": rng.randint(1, 2)}
        if op == "attend":
            case["hq"] = hq
        heavy = work(case)
        return draw(rng) if heavy["flops"] > 4e11 or heavy["bytes"] > 2e8 else case
    if op == "drafts":
        n, k_hi = _log(rng, 1, 200), rng.randint(1, 8)
        vocab = _log(rng, 1000, 151936)
        if n * (k_hi + 1) * vocab > 1.5e8:
            return draw(rng)
        return {"op": op, "n": n, "k_lo": rng.randint(0, k_hi), "k_hi": k_hi, "vocab": vocab,
                "type": rng.choice(("f32", "bf16", "f16")), "draft_probs": rng.random() < 0.6,
                "match": round(rng.uniform(0.2, 0.95), 2)}
    layers, blocks = rng.randint(1, 28), _log(rng, 64, 4096)
    kind = rng.choice(("fp8", "bf16"))
    size = {"layers": layers, "blocks": blocks, "hkv": hkv, "d": d, "bs": bs, "type": kind}
    if blocks * _page_bytes(size) > 2e9:
        return draw(rng)
    if op == "fork":
        return {"op": op, "pairs": _log(rng, 1, max(1, blocks // 3)), **size}
    return {"op": op, "n": rng.randint(1, 64), "live": round(rng.uniform(0.05, 0.95), 2), **size}


# ---------------------------------------------------------------------------- lengths
def _spread(lo, hi, n):
    """n lengths from lo to hi: even steps, or even steps of the logarithm over a factor of ten."""
    if lo > 0 and hi > 10 * lo:
        return [round(lo * (hi / lo) ** ((i + 0.5) / n)) for i in range(n)]
    return [lo + round((hi - lo) * (i + 0.5) / n) for i in range(n)]


def _lengths(case):
    """(query lengths, context lengths) of an attend or rows case, before they are shuffled."""
    if case["op"] == "decode":
        ctx = _spread(case["lo"], case["hi"], case["n"])
        return [1] * case["n"], ctx
    q = _spread(case["q_lo"], case["q_hi"], case["n"])
    past = _spread(case["past_lo"], case["past_hi"], case["n"])
    past = [past[(7 * i + 3) % len(past)] for i in range(len(past))]
    return q, [a + b for a, b in zip(q, past)]


def _page_bytes(case):
    """Bytes of one block's K and V over all layers, scales included."""
    scales = 8 * case["hkv"] if case["type"] == "fp8" else 0
    return case["layers"] * (2 * case["bs"] * case["hkv"] * case["d"] * BYTES[case["type"]] + scales)


def work(case):
    op = case["op"]
    if op in ("rows", "decode", "attend"):
        q, ctx = _lengths(case)
        row, bs = case["hkv"] * case["d"], case["bs"]
        if op == "rows":
            # rows in, their codes out; of each touched block the codes in and the values out
            back = sum(c - (c - a) // bs * bs for a, c in zip(q, ctx))
            per = BYTES[case["type"]]
            return {"bytes": 2 * row * (sum(q) * (per + 1) + back * (1 + per)), "flops": 0}
        kv = sum(ctx) * 2 * row + sum(-(-c // bs) for c in ctx) * (8 * case["hkv"] + 4)
        io = 2 * sum(q) * case["hq"] * case["d"] * BYTES[case["type"]]
        pairs = sum(a * (c - a) + a * (a + 1) // 2 for a, c in zip(q, ctx))
        return {"bytes": kv + io, "flops": 4 * case["hq"] * case["d"] * pairs}
    if op == "drafts":
        k = _spread(case["k_lo"], case["k_hi"], case["n"])
        per = BYTES[case["type"]]
        # one row of target probabilities a sequence, one of draft probabilities where a token is rejected
        rejects = sum(1 - case["match"] ** j for j in k)
        rows = case["n"] + (rejects if case["draft_probs"] else 0)
        return {"bytes": rows * case["vocab"] * per + 40 * sum(k) + 8 * (sum(k) + 2 * case["n"]), "flops": 0}
    if op == "fork":
        return {"bytes": 2 * case["pairs"] * _page_bytes(case) + 8 * case["pairs"], "flops": 0}
    moved = case["blocks"] * case["live"] * (1 - case["live"])
    return {"bytes": 2 * moved * _page_bytes(case) + 12 * case["blocks"], "flops": 0}


# ---------------------------------------------------------------------------- inputs
def _block_scales(amax):
    """2**e with the smallest e >= MIN_EXP for which amax <= 448 * 2**e (448 = 0.875 * 2**9)."""
    m, e = torch.frexp(amax.float())
    e = (e - 9 + (m > 0.875).int()).clamp(min=MIN_EXP)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))
    return torch.ldexp(torch.ones_like(m), e)


def _values(gen, shape, spread):
    """Normal values; every 32nd channel is `spread` times as large, as keys of trained models have."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    x[..., ::32] *= spread
    return x


def _pool8(gen, layers, blocks, bs, hkv, d, spread):
    """(codes [layers, slots, hkv, d], scales [layers, blocks, hkv]) of a filled 8-bit pool."""
    codes = torch.empty((layers, blocks * bs, hkv, d), dtype=FP8, device="cuda")
    scales = torch.empty((layers, blocks, hkv), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 26) // (bs * hkv * d))
    for lay in range(layers):
        for b in range(0, blocks, step):
            n = min(step, blocks - b)
            x = _values(gen, (n, bs, hkv, d), spread)
            s = _block_scales(x.abs().amax(dim=(1, 3)))
            scales[lay, b:b + n] = s
            codes[lay, b * bs:(b + n) * bs] = (x / s[:, None, :, None]).to(FP8).view(n * bs, hkv, d)
    return codes, scales


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op in ("rows", "decode", "attend"):
        q, ctx = _lengths(case)
        order = list(range(len(q)))
        rng.shuffle(order)
        q, ctx = [q[i] for i in order], [ctx[i] for i in order]
        bs, hkv, d, dtype = case["bs"], case["hkv"], case["d"], DTYPES[case["type"]]
        need = [-(-c // bs) for c in ctx]
        blocks = sum(need) + sum(need) // 8 + 3
        ids = list(range(blocks))
        rng.shuffle(ids)
        table, cu, used = torch.full((len(q), max(need)), -1, dtype=torch.int32), [0], 0
        for i, w in enumerate(need):
            table[i, :w] = torch.tensor(ids[used:used + w], dtype=torch.int32)
            used += w
            cu.append(cu[-1] + q[i])
        s = {"case": case, "q_lens": q, "ctx_lens": ctx, "bs": bs, "layer": case["layers"] - 1,
             "tables": table.cuda(), "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
             "ctx": torch.tensor(ctx, dtype=torch.int32, device="cuda"), "max_q": max(q)}
        s["kc"], s["ks"] = _pool8(gen, case["layers"], blocks, bs, hkv, d, 6.0)
        s["vc"], s["vs"] = _pool8(gen, case["layers"], blocks, bs, hkv, d, 1.0)
        if op == "rows":
            s["keys"] = _values(gen, (cu[-1], hkv, d), 6.0).to(dtype)
            s["values"] = _values(gen, (cu[-1], hkv, d), 1.0).to(dtype)
            # what the step's metadata gives: the slot of each new row; and the slots of every
            # row of the touched blocks that is in use after the write
            pos = [(i, p) for i, (a, c) in enumerate(zip(q, ctx)) for p in range(c - a, c)]
            back = [(i, p) for i, (a, c) in enumerate(zip(q, ctx)) for p in range((c - a) // bs * bs, c)]
            for name, at in (("slots", pos), ("back", back)):
                seq, p = (torch.tensor(v) for v in zip(*at))
                s[name] = (table[seq, p // bs] * bs + p % bs).to(torch.int32).cuda()
        else:
            s["q"] = torch.randn((cu[-1], case["hq"], d), generator=gen, device="cuda").to(dtype)
            s["scale"] = d ** -0.5
        return s
    if op == "drafts":
        k = _spread(case["k_lo"], case["k_hi"], case["n"])
        rng.shuffle(k)
        cu, n, v, dtype = [0], case["n"], case["vocab"], DTYPES[case["type"]]
        for j in k:
            cu.append(cu[-1] + j)
        t = cu[-1]
        seq = torch.tensor([i for i, j in enumerate(k) for _ in range(j)], dtype=torch.int64, device="cuda")
        logits = torch.randn((t + n, v), generator=gen, device="cuda") * 3.0
        target = torch.softmax(logits, -1)
        rows = torch.arange(t, device="cuda") + seq
        # the draft model: the target's logits with noise, less of it the better they match
        draft = torch.softmax(logits[rows] + torch.randn((t, v), generator=gen, device="cuda") * (2.5 * (1 - case["match"])), -1)
        del logits
        tokens = torch.multinomial(draft, 1, generator=gen)[:, 0] if t else torch.zeros(0, dtype=torch.int64, device="cuda")
        return {"case": case, "k": k, "max_k": max(k), "target": target.to(dtype),
                "draft": draft.to(dtype) if case["draft_probs"] else None, "tokens": tokens,
                "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
                "accept": torch.rand(t, generator=gen, device="cuda"),
                "sample": torch.rand(n, generator=gen, device="cuda")}
    layers, blocks, bs, hkv, d = (case[x] for x in ("layers", "blocks", "bs", "hkv", "d"))
    s = {"case": case, "bs": bs, "ks": None, "vs": None}
    for c, scales in (("kc", "ks"), ("vc", "vs")):
        if case["type"] == "fp8":
            raw = torch.randint(0, 127, (layers, blocks * bs, hkv, d), generator=gen, device="cuda", dtype=torch.uint8)
            s[c] = raw.view(FP8)
            s[scales] = torch.ldexp(torch.ones((), device="cuda"), torch.randint(-12, 3, (layers, blocks, hkv), generator=gen, device="cuda"))
        else:
            s[c] = torch.empty((layers, blocks * bs, hkv, d), dtype=DTYPES[case["type"]], device="cuda")
            s[c].normal_(generator=gen)
    ids = list(range(blocks))
    rng.shuffle(ids)
    if op == "fork":
        p = case["pairs"]
        # several children of one parent copy the same page
        s["src"] = torch.tensor([ids[i // 2] for i in range(p)], dtype=torch.int32, device="cuda")
        s["dst"] = torch.tensor(ids[blocks - p:], dtype=torch.int32, device="cuda")
        return s
    live = max(case["n"], round(blocks * case["live"]))
    n = min(case["n"], live)
    need = [live // n + (i < live % n) for i in range(n)]
    table, used = torch.full((n, max(need) + 1), -1, dtype=torch.int32), 0
    for i, w in enumerate(need):
        table[i, :w] = torch.tensor(ids[used:used + w], dtype=torch.int32)
        if i and w > 2:  # a shared prefix: forked sequences hold their first pages together
            table[i, 0] = table[0, 0]
        used += w
    s["tables"] = table.cuda()
    s["ctx"] = torch.tensor([w * bs - rng.randrange(bs) for w in need], dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------- plain forms
def _plain_rows(s):
    """New rows into the pool, rows of the touched blocks back as values."""
    lay, bs, slots = s["layer"], s["bs"], s["slots"].long()
    blk, first = slots // bs, s["cu"][:-1].long()
    for cache, scales, new in ((s["kc"], s["ks"], s["keys"]), (s["vc"], s["vs"], s["values"])):
        new, sc, pool = new.float(), scales[lay], cache[lay]
        hkv, d = new.shape[1:]
        amax = torch.zeros_like(sc).scatter_reduce_(0, blk[:, None].expand(-1, hkv), new.abs().amax(-1), "amax")
        need = _block_scales(amax)
        # the block that a sequence's first new row falls into keeps its older rows unless that row is its first
        part, keep = blk[first], (slots[first] % bs != 0)
        old = sc[part]
        grown = torch.where(keep[:, None], torch.maximum(old, need[part]), need[part])
        raw = pool.view(torch.uint8).view(-1, bs, hkv, d)
        held = raw[part].view(FP8).float() * (old / grown)[:, None, :, None]
        held = torch.where(keep[:, None, None, None], held.clamp(-448, 448).to(FP8).float(), raw[part].view(FP8).float())
        raw[part] = held.to(FP8).view(torch.uint8)
        sc[blk] = need[blk]
        sc[part] = grown
        pool.view(torch.uint8)[slots] = (new / sc[blk][:, :, None]).to(FP8).view(torch.uint8)
    back = s["back"].long()
    out = {"key_scales": s["ks"], "value_scales": s["vs"]}
    for name, cache, scales, like in (("keys", s["kc"], s["ks"], s["keys"]), ("values", s["vc"], s["vs"], s["values"])):
        codes = cache[lay].view(torch.uint8)[back].view(FP8).float()
        out[name] = (codes * scales[lay][back // bs][:, :, None]).to(like.dtype)
    return out


def _history(cache, scales, layer, tables, bs):
    """Values of the given tables' blocks: [sequences, tokens, hkv, d] in 32 bits."""
    hkv, d = cache.shape[2:]
    at = tables.clamp(min=0).long()
    codes = cache[layer].view(torch.uint8).view(-1, bs, hkv, d)[at].view(FP8).float()
    return (codes * scales[layer][at][:, :, None, :, None]).flatten(1, 2)


def _plain_attend(s):
    """softmax(q k' scale + causal mask) v, a batch of sequences at a time."""
    q, cu, bs = s["q"], s["cu"], s["bs"]
    hq, d = q.shape[1:]
    hkv = s["kc"].shape[2]
    n, top = len(s["q_lens"]), s["max_q"]
    # few rows: every sequence in one batch; many: one sequence at a time, for its matrix of scores
    batches = [(0, n)] if top <= 16 else [(i, i + 1) for i in range(n)]

    def some(i, j):
        rows, width = max(s["q_lens"][i:j]), -(-max(s["ctx_lens"][i:j]) // bs)
        k = _history(s["kc"], s["ks"], s["layer"], s["tables"][i:j, :width], bs)
        v = _history(s["vc"], s["vs"], s["layer"], s["tables"][i:j, :width], bs)
        lens, ctx = (cu[i + 1:j + 1] - cu[i:j]).long(), s["ctx"][i:j].long()
        r = torch.arange(rows, device=q.device)
        inside = r < lens[:, None]
        at = torch.where(inside, cu[i:j, None].long() + r, 0)
        x = q[at].float().view(j - i, rows, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(j - i, hkv, -1, d)
        scores = torch.matmul(x, k.permute(0, 2, 3, 1)).view(j - i, hkv, hq // hkv, rows, -1) * s["scale"]
        seen = torch.arange(k.shape[1], device=q.device) <= (ctx[:, None] - lens[:, None] + r)[:, :, None]
        scores.masked_fill_(~seen[:, None, None], float("-inf"))
        scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        scores /= scores.sum(-1, keepdim=True)
        v = torch.where((torch.arange(k.shape[1], device=q.device) < ctx[:, None])[:, :, None, None], v, 0.0)
        o = torch.matmul(scores.view(j - i, hkv, -1, k.shape[1]), v.permute(0, 2, 1, 3))
        o = o.view(j - i, hq, rows, d).permute(0, 2, 1, 3)
        return o[inside].to(q.dtype)

    return torch.cat([some(i, j) for i, j in batches])


def _plain_drafts(s):
    """Accepted drafts, then one token from the residual (or, with all accepted, from the target)."""
    p, q, tok, cu = s["target"], s["draft"], s["tokens"], s["cu"].long()
    n, t, dev = cu.numel() - 1, tok.numel(), p.device
    lens = cu[1:] - cu[:-1]
    j = torch.arange(s["max_k"], device=dev)
    inside = j < lens[:, None]
    at = torch.where(inside, cu[:-1, None] + j, 0)
    if t:
        rows = at + torch.arange(n, device=dev)[:, None]
        drafted = tok[at]
        px = p[rows, drafted].double()
        qx = q[at, drafted].double() if q is not None else torch.ones_like(px)
        ok = inside & (s["accept"][at].double() * qx < px)
        count = ok.int().cumprod(1).sum(1)
    else:
        drafted, count = at, torch.zeros(n, dtype=torch.int64, device=dev)
    rejected = count < lens
    r = p[cu[:-1] + torch.arange(n, device=dev) + count].double()
    whole = r.clone()
    if t:
        at = torch.where(rejected, cu[:-1] + count, 0)
        if q is not None:
            r -= torch.where(rejected[:, None], q[at].double(), 0.0)
        else:
            r[torch.arange(n, device=dev), tok[at]] -= rejected.double()
        r.clamp_(min=0)
        r = torch.where(r.sum(1, keepdim=True) > 0, r, whole)
    cdf = r.cumsum(1)
    token = torch.searchsorted(cdf, (s["sample"].double() * cdf[:, -1])[:, None], right=True)[:, 0]
    last = r.shape[1] - 1 - (r > 0).flip(1).int().argmax(1)
    token = torch.minimum(token, last)
    j = torch.arange(s["max_k"] + 1, device=dev)
    out = torch.full((n, s["max_k"] + 1), -1, dtype=torch.int64, device=dev)
    if t:
        out[:, :-1] = torch.where(j[:-1] < count[:, None], drafted, -1)
    out = torch.where(j == count[:, None], token[:, None], out)
    return {"tokens": out, "accepted": count.int()}


def _buffers(s):
    """The pool's tensors, those that move with a page."""
    got = {"key_cache": s["kc"], "value_cache": s["vc"]}
    if s["ks"] is not None:
        got |= {"key_scales": s["ks"], "value_scales": s["vs"]}
    return got


def _move(s, src, dst):
    bs = s["bs"]
    for t in _buffers(s).values():
        if t.dim() == 4:
            t = t.view(torch.uint8 if t.dtype == FP8 else t.dtype).view(t.shape[0], -1, bs, *t.shape[2:])
        t[:, dst] = t[:, src]


def _plain_compact(s):
    bs, blocks = s["bs"], s["case"]["blocks"]
    tables, dev = s["tables"].clone(), s["tables"].device
    used = torch.arange(tables.shape[1], device=dev) < ((s["ctx"] + bs - 1) // bs)[:, None]
    live = torch.zeros(blocks, dtype=torch.bool, device=dev)
    live[tables[used].long()] = True
    count = live.sum()
    index = torch.arange(blocks, device=dev)
    src, dst = torch.nonzero(live & (index >= count))[:, 0], torch.nonzero(~live & (index < count))[:, 0]
    _move(s, src, dst)
    new = torch.where(live, index, -1)
    new[src] = dst
    tables = torch.where(used, new[tables.clamp(min=0).long()].int(), tables)
    return {"tables": tables, "new_ids": new.int(), "num_live": count.int().view(1), **_buffers(s)}


# ---------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        import __graft_entry__

        __graft_entry__.load_package()
        from llm_engineering_b200 import ops

        if op == "rows":
            ops.kv_write_fp8(s["kc"], s["vc"], s["ks"], s["vs"], s["layer"], s["tables"], s["cu"], s["ctx"],
                             s["max_q"], s["bs"], s["keys"], s["values"])
            keys, values = ops.kv_read_fp8(s["kc"], s["vc"], s["ks"], s["vs"], s["layer"], s["back"], s["bs"],
                                           s["keys"].dtype)
            return {"keys": keys, "values": values, "key_scales": s["ks"], "value_scales": s["vs"]}
        if op in ("decode", "attend"):
            if "workspace" not in s:
                s["workspace"] = ops.make_fp8_workspace(s["ctx"].numel(), s["q"].shape[1], s["kc"].shape[2],
                                                        s["q"].shape[2], s["q"].device, s["max_q"])
            args = (s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["layer"], s["tables"])
            if op == "decode":
                return ops.paged_decode_fp8(*args, s["ctx"], s["bs"], s["scale"], workspace=s["workspace"])
            return ops.paged_prefill_fp8(*args, s["cu"], s["ctx"], s["max_q"], s["bs"], s["scale"],
                                         workspace=s["workspace"])
        if op == "drafts":
            tokens, accepted = ops.verify_drafts(s["target"], s["tokens"], s["cu"], s["accept"], s["sample"],
                                                 s["max_k"], draft_probs=s["draft"])
            return {"tokens": tokens, "accepted": accepted}
        if op == "fork":
            ops.copy_blocks(s["kc"], s["vc"], s["src"], s["dst"], s["bs"], s["ks"], s["vs"])
            return _buffers(s)
        tables = s["tables"].clone()
        new, count = ops.compact_blocks(s["kc"], s["vc"], tables, s["ctx"], s["bs"], s["ks"], s["vs"])
        return {"tables": tables, "new_ids": new, "num_live": count, **_buffers(s)}
    if op == "rows":
        return _plain_rows(s)
    if op in ("decode", "attend"):
        return _plain_attend(s)
    if op == "drafts":
        return _plain_drafts(s)
    if op == "fork":
        _move(s, s["src"].long(), s["dst"].long())
        return _buffers(s)
    return _plain_compact(s)


# ---------------------------------------------------------------------------- 64 bits
def _round8(x):
    """x (64 bits, |x| <= 448) to the nearest e4m3 value, ties to even: steps of 2**(e - 3), e >= -6."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _scale_of(amax):
    """The block scale of one (block, head) from its largest magnitude, counted up from below."""
    e = MIN_EXP
    if amax > 0:
        e = max(MIN_EXP, math.floor(math.log2(amax)) - 10)
        while amax > 448.0 * 2.0 ** e:
            e += 1
    return 2.0 ** e


def _exact_rows(s):
    lay, bs = s["layer"], s["bs"]
    out = {"key_scales": s["ks"].double(), "value_scales": s["vs"].double(), "keys": [], "values": []}
    cu = s["cu"].tolist()
    for cache, scales, new, name in ((s["kc"], s["ks"], s["keys"], "keys"), (s["vc"], s["vs"], s["values"], "values")):
        top = new.abs().amax(-1).double().tolist()
        into = out["key_scales" if name == "keys" else "value_scales"]
        old = scales[lay].tolist()
        tables = s["tables"].tolist()
        grown, lists = [], []
        for i, (a, c) in enumerate(zip(s["q_lens"], s["ctx_lens"])):
            for b in range((c - a) // bs, -(-c // bs)):
                first, last = max(b * bs, c - a), min(c, (b + 1) * bs)
                rows = range(cu[i] + first - (c - a), cu[i] + last - (c - a))
                line = [_scale_of(max(top[r][h] for r in rows)) for h in range(new.shape[1])]
                if first > b * bs:
                    line = [max(x, y) for x, y in zip(line, old[tables[i][b]])]
                grown.append(line)
                lists.append((tables[i][b], first - b * bs, rows.start, last - first))
        grown = torch.tensor(grown, dtype=torch.float64, device="cuda")
        into[lay][torch.tensor([x[0] for x in lists], device="cuda")] = grown
        # the rows that each touched block holds afterwards, in order: older ones, then new ones
        held = [x for x in range(len(lists)) if lists[x][1]]
        whole = _round8(new.double() / grown.repeat_interleave(torch.tensor([x[3] for x in lists], device="cuda"), 0)[:, :, None]) \
            * grown.repeat_interleave(torch.tensor([x[3] for x in lists], device="cuda"), 0)[:, :, None]
        parts = []
        codes = cache[lay].view(torch.uint8).view(-1, bs, *new.shape[1:])
        older = codes[torch.tensor([lists[x][0] for x in held], dtype=torch.int64, device="cuda")].view(FP8).double() if held else None
        for x, (block, before, start, count) in enumerate(lists):
            if before:
                h = older[held.index(x), :before] * scales[lay][block].double()[None, :, None]
                parts.append(_round8(h / grown[x][None, :, None]) * grown[x][None, :, None])
            parts.append(whole[start:start + count])
        out[name] = torch.cat(parts)
    return out


def _exact_attend(s):
    cu, bs, q = s["cu"].tolist(), s["bs"], s["q"]
    hkv, d = s["kc"].shape[2:]
    out = []
    for i, (a, c) in enumerate(zip(s["q_lens"], s["ctx_lens"])):
        at = torch.arange(c, device="cuda")
        block = s["tables"][i].long()[at // bs]
        slot = block * bs + at % bs
        k, v = ((t[s["layer"]].view(torch.uint8)[slot].view(FP8).double() * f[s["layer"]][block].double()[:, :, None])
                for t, f in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
        x = q[cu[i]:cu[i + 1]].double()
        got = torch.empty_like(x)
        mask = at[None, :] > (c - a + torch.arange(a, device="cuda"))[:, None]
        for h in range(x.shape[1]):
            g = h // (x.shape[1] // hkv)
            w = (x[:, h] @ k[:, g].T * s["scale"]).masked_fill(mask, -math.inf)
            got[:, h] = torch.softmax(w, -1) @ v[:, g]
        out.append(got)
    return torch.cat(out)


def _exact_drafts(s):
    cu, tokens, counts = s["cu"].tolist(), [], []
    drafts = s["tokens"].tolist()
    for i, k in enumerate(s["k"]):
        n = 0
        while n < k:
            row, x = cu[i] + n, drafts[cu[i] + n]
            px = float(s["target"][row + i, x])
            qx = float(s["draft"][row, x]) if s["draft"] is not None else 1.0
            if not float(s["accept"][row]) * qx < px:
                break
            n += 1
        p = s["target"][cu[i] + i + n].double()
        r = p
        if n < k:
            one = torch.zeros_like(p)
            one[drafts[cu[i] + n]] = 1.0
            r = (p - (s["draft"][cu[i] + n].double() if s["draft"] is not None else one)).clamp(min=0)
            r = r if float(r.sum()) > 0 else p
        cdf = r.cumsum(0)
        past = torch.nonzero(cdf > float(s["sample"][i]) * float(cdf[-1]))
        pick = int(past[0]) if past.numel() else int(torch.nonzero(r > 0)[-1])
        tokens.append(drafts[cu[i]:cu[i] + n] + [pick] + [-1] * (s["max_k"] - n))
        counts.append(n)
    return {"tokens": torch.tensor(tokens), "accepted": torch.tensor(counts, dtype=torch.int32)}


def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # copies of bits: nothing is computed
    s = prepare(case, seed)
    return _exact_rows(s) if op == "rows" else _exact_drafts(s) if op == "drafts" else _exact_attend(s)
