"""The 8-bit cache, draft verification, forks and compaction as one program uses them: by hand
against the 64-bit plain forms, and through the runner and the engine."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

from llm_engineering_b200 import engine as eng
from llm_engineering_b200 import runner as runner_module
from llm_engineering_b200.runner import B200PagedModelRunner
from llm_engineering_b200.storage import Fp8PagedKVStorage, PagedKVStorage
from oracle import fp8 as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Mirror:
    """One layer of an 8-bit pool in the plain form."""

    def __init__(self, storage):
        self.bs = storage.block_size
        self.k, self.v = (t.view(torch.uint8).cpu()[0].numpy().copy() for t in (storage.key_cache, storage.value_cache))
        self.ks, self.vs = (t.cpu()[0].double().numpy().copy() for t in (storage.key_scales, storage.value_scales))

    def write(self, tables, q_lens, ctx, keys, values):
        ref.write(self.k, self.ks, self.bs, tables, q_lens, ctx, keys.double().numpy())
        ref.write(self.v, self.vs, self.bs, tables, q_lens, ctx, values.double().numpy())

    def move(self, src, dst):
        for t in (self.k, self.v):
            t[dst * self.bs:(dst + 1) * self.bs] = t[src * self.bs:(src + 1) * self.bs]
        for t in (self.ks, self.vs):
            t[dst] = t[src]

    def attend(self, q, tables, q_lens, ctx, scale):
        return ref.attend(q, torch.from_numpy(self.k), torch.from_numpy(self.ks), torch.from_numpy(self.v),
                          torch.from_numpy(self.vs), self.bs, tables, q_lens, ctx, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_speculative_steps_with_forks_and_compaction(ops, dtype):
    """Prompts in, drafted rows scored and partly dropped, sequences forked, the pool compacted, and
    on; every attention call within the bound that its roundings give (test_fp8_cache_gpu.py)."""
    from test_fp8_cache_gpu import check, p_step

    hq, hkv, d, bs, blocks, vocab = 12, 2, 128, 16, 64, 97
    rng = np.random.default_rng(7)
    storage = Fp8PagedKVStorage(1, blocks, bs, hkv, d, DEV)
    storage.key_cache.view(torch.uint8).fill_(0x7F)  # NaN codes wherever nothing is written
    storage.value_cache.view(torch.uint8).fill_(0x7F)
    plain = Mirror(storage)
    table = eng.BlockTable(eng.BlockPool(blocks), bs)
    ctx = {"a": 75, "b": 16, "c": 150}
    for name, n in ctx.items():
        table.allocate_for_request(name, n)
    ws = ops.make_fp8_workspace(8, hq, hkv, d, DEV, 5)
    err = i32([0])

    def rows(n, heads):
        return torch.from_numpy(rng.standard_normal((n, heads, d))).to(dtype)

    def step(names, q_lens):
        """Append q_lens new rows each (contexts already grown) and attend them."""
        tables = [list(table.blocks_for_request(n)) for n in names]
        c = [ctx[n] for n in names]
        width = max(len(t) for t in tables)
        bt = i32([t + [-1] * (width - len(t)) for t in tables])
        cu = i32(np.concatenate([[0], np.cumsum(q_lens)]).tolist())
        k, v, q = rows(sum(q_lens), hkv), rows(sum(q_lens), hkv), rows(sum(q_lens), hq)
        storage.append(0, bt, cu, i32(c), max(q_lens), k.cuda(), v.cuda(), err)
        plain.write(tables, q_lens, c, k, v)
        pool = (storage.key_cache, storage.value_cache, storage.key_scales, storage.value_scales, 0, bt)
        if max(q_lens) == 1:
            got = ops.paged_decode_fp8(q.cuda(), *pool, i32(c), bs, d ** -0.5, workspace=ws, err_flag=err)
        else:
            got = ops.paged_prefill_fp8(q.cuda(), *pool, cu, i32(c), max(q_lens), bs, d ** -0.5, workspace=ws,
                                        err_flag=err)
        check(got, plain.attend(q, tables, q_lens, c, d ** -0.5), dtype, d, max(c),
              p_step(dtype, max(q_lens) > 1))

    step(list(ctx), list(ctx.values()))  # prompts
    for round_ in range(3):
        names = list(ctx)
        ks = [int(rng.integers(0, 5)) for _ in names]
        for n, k in zip(names, ks):
            for t in range(ctx[n], ctx[n] + k + 1):
                table.append_token(n, t)
            ctx[n] += k + 1
        step(names, [k + 1 for k in ks])  # the last token and k drafts
        cu = np.concatenate([[0], np.cumsum(ks)]).tolist()
        target = torch.softmax(torch.randn(cu[-1] + len(ks), vocab) * 2, -1)
        draft = torch.softmax(torch.randn(cu[-1], vocab), -1)
        tokens = torch.multinomial(draft, 1)[:, 0] if cu[-1] else torch.zeros(0, dtype=torch.int64)
        u, w = torch.rand(cu[-1]), torch.rand(len(ks))
        got, accepted = ops.verify_drafts(target.cuda(), tokens.cuda(), i32(cu), u.cuda(), w.cuda(), 4,
                                          draft_probs=draft.cuda(), err_flag=err)
        want = ref.verify(target.double().numpy(), draft.double().numpy(), tokens.tolist(), cu, u.double().numpy(),
                          w.double().numpy(), 4)
        assert got.tolist() == want[0] and accepted.tolist() == want[1]
        for n, k, a in zip(names, ks, accepted.tolist()):
            ctx[n] -= k - a  # rejected drafts leave; their rows are written over later
        if round_ == 0:  # fork "a" in the middle of a block
            copies = table.fork_request("a", "a2", ctx["a"])
            storage.copy_blocks([s for s, _ in copies], [t for _, t in copies])
            for s, t in copies:
                plain.move(s, t)
            ctx["a2"] = ctx["a"]
        if round_ == 1:  # "b" ends; the pool is packed
            table.free_request("b")
            del ctx["b"]
            before = table.tables()
            moves, new, live = ref.compact(list(before.values()), [len(t) * bs for t in before.values()], bs, blocks)
            assert storage.compact(table) == live
            for s, t in moves:
                plain.move(s, t)
            assert {n: tuple(new[b] for b in t) for n, t in before.items()} == table.tables()
        for n in ctx:  # the drawn token's row
            table.append_token(n, ctx[n])
            ctx[n] += 1
        step(list(ctx), [1] * len(ctx))
    assert err.item() == 0


def test_offsets_past_32_bits(ops):
    """A pool of 4.9 GB a tensor whose used blocks lie at its end: every entry point's byte offsets
    pass 2^32 (the few-row kernel, the tile kernel over the widened copy, rows in and out, copies,
    and verification rows past 2^31 elements)."""
    from test_fp8_cache_gpu import check, p_step

    hq, hkv, d, bs, blocks = 28, 4, 128, 16, 600_000
    rng = np.random.default_rng(1)
    storage = Fp8PagedKVStorage(1, blocks, bs, hkv, d, DEV)
    tables = [[blocks - 1 - 3 * i for i in range(12)], [blocks - 2 - 3 * i for i in range(2)]]
    ctx = [190, 31]
    bt = i32([tables[0], tables[1] + [-1] * 10])
    cu = i32([0, 190, 221])
    k, v = (torch.from_numpy(rng.standard_normal((221, hkv, d))).to(torch.bfloat16) for _ in range(2))
    storage.append(0, bt, cu, i32(ctx), 190, k.cuda(), v.cuda())
    ids = sorted(b for t in tables for b in t)
    small = {b: i for i, b in enumerate(ids)}  # the same blocks in a pool of their own
    codes, scales = ([np.zeros((len(ids) * bs, hkv, d), np.uint8) for _ in range(2)],
                     [np.zeros((len(ids), hkv)) for _ in range(2)])
    own = [[small[b] for b in t] for t in tables]
    for c, s, x in zip(codes, scales, (k, v)):
        ref.write(c, s, bs, own, ctx, ctx, x.double().numpy())
    plain = (torch.from_numpy(codes[0]), torch.from_numpy(scales[0]), torch.from_numpy(codes[1]),
             torch.from_numpy(scales[1]))
    slots = [tables[0][p // bs] * bs + p % bs for p in range(190)]
    got = storage.gather(0, slots)
    for x, c, s in zip(got, codes, scales):
        at = np.array([own[0][p // bs] * bs + p % bs for p in range(190)])
        assert torch.equal(x.double().cpu(), torch.from_numpy(ref.VALUES[c[at]] * s[at // bs][:, :, None]))
    pool = (storage.key_cache, storage.value_cache, storage.key_scales, storage.value_scales, 0, bt)
    q = torch.from_numpy(rng.standard_normal((221, hq, d))).to(torch.bfloat16)
    got = ops.paged_prefill_fp8(q.cuda(), *pool, cu, i32(ctx), 190, bs, d ** -0.5)
    rows = [0, 17, 100, 189, 190, 220]  # of all rows: enough for the offsets
    want = ref.attend(q, *plain, bs, own, ctx, ctx, d ** -0.5)
    check(got[rows], tuple(t[rows] for t in want), torch.bfloat16, d, 190, p_step(torch.bfloat16, True))
    last = torch.stack([q[189], q[220]])
    got = ops.paged_decode_fp8(last.cuda(), *pool, i32(ctx), bs, d ** -0.5)
    check(got, tuple(t[[189, 220]] for t in want), torch.bfloat16, d, 190, p_step(torch.bfloat16, False))
    storage.copy_blocks([tables[0][0]], [5])
    assert torch.equal(storage.key_cache[0, 80:96].view(torch.uint8).cpu(), plain[0][own[0][0] * bs:own[0][0] * bs + bs])
    del storage, got, pool
    vocab = 151936
    target = torch.zeros((14200, vocab), dtype=torch.bfloat16, device=DEV)  # 2.16e9 elements
    target[14199, 77] = 1.0
    target[:14199, 3] = 1.0
    n = 14199
    tokens, accepted = ops.verify_drafts(target, torch.full((1,), 3, dtype=torch.int64, device=DEV),
                                         i32([0] * n + [1])[:n + 1], torch.zeros(1, device=DEV),
                                         torch.full((n,), 0.5, device=DEV), 1)
    assert accepted.tolist() == [0] * (n - 1) + [1]
    assert tokens[-1].tolist() == [3, 77] and tokens[0].tolist() == [3, -1]


def small_model(dtype, seed=0):
    from transformers import Qwen2Config, Qwen2ForCausalLM

    cfg = Qwen2Config(vocab_size=1000, hidden_size=1536, intermediate_size=512, num_hidden_layers=2,
                      num_attention_heads=12, num_key_value_heads=2, max_position_embeddings=4096)
    torch.manual_seed(seed)
    return Qwen2ForCausalLM(cfg).eval().to(DEV, dtype)


def run_engine(model, storage, prompts, blocks, chunked=False, between=None):
    runner = B200PagedModelRunner(model, DEV, storage)
    cfg = eng.EngineConfiguration(device="cuda", block_size=16, num_blocks=blocks, max_sequences=8,
                                  max_batched_tokens=256 if chunked else 2048, enable_chunked_prefill=chunked)
    engine = eng.Engine(configuration=cfg, model_runner=runner)
    for i, p in enumerate(prompts):
        engine.submit(eng.Request(request_id=f"r{i}", prompt_token_ids=tuple(p), max_new_tokens=6 + i, ignore_eos=True))
    steps = 0
    while engine.has_unfinished_requests:
        engine.step()
        steps += 1
        if between is not None:
            between(steps, engine, runner, storage)
    assert runner.device_error() == 0
    return {s.request.request_id: list(s.generated_token_ids) for s in engine.finished_sequences}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_engine_over_the_8bit_pool(dtype):
    """The engine runs unchanged on the 8-bit storage, with whole and with chunked prefill: every
    request ends with the tokens it asked for and no device error."""
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (40, 17, 130, 300, 3)]
    model = small_model(dtype)
    got = run_engine(model, Fp8PagedKVStorage(2, 128, 16, 2, 128, DEV), prompts, 128)
    assert sorted(got) == [f"r{i}" for i in range(5)] and [len(got[f"r{i}"]) for i in range(5)] == [6, 7, 8, 9, 10]
    chunked = run_engine(model, Fp8PagedKVStorage(2, 128, 16, 2, 128, DEV), prompts, 128, chunked=True)
    assert [len(chunked[f"r{i}"]) for i in range(5)] == [6, 7, 8, 9, 10]


def test_first_token_logits_match_a_forward_over_the_dequantised_pool(ops, monkeypatch):
    """One prefill step on the 8-bit pool, then the same step on an fp32 pool filled with the values
    that the 8-bit pool holds: attention over equal values, so the next step's logits agree to
    fp32 rounding. Softmax and norms keep relative errors near 2^-24 * a few hundred operations:
    1e-4 of the logits' size is far above it and far below a cache error (2^-4 per value)."""
    rng = np.random.default_rng(5)
    model = small_model(torch.float32, seed=2)
    torch.backends.cuda.matmul.allow_tf32 = False
    prompts = [rng.integers(0, 1000, n).tolist() for n in (70, 33)]
    f8 = Fp8PagedKVStorage(2, 16, 16, 2, 128, DEV)
    f32 = PagedKVStorage(2, 16, 16, 2, 128, torch.float32, DEV)
    f32.key_cache.zero_(), f32.value_cache.zero_()

    class Ex:
        def __init__(self, name, tokens, blocks, phase, q_len):
            req = eng.Request(request_id=name, prompt_token_ids=tuple(tokens), max_new_tokens=4, ignore_eos=True)
            self.sequence = eng.SequenceState(request=req)
            self.phase, self.block_ids = phase, tuple(blocks)
            self.length, self.query_length = len(tokens), q_len

    blocks = [(3, 9, 1, 12, 5), (7, 0, 14)]
    r8 = B200PagedModelRunner(copy.deepcopy(model), DEV, f8)
    r8.forward([Ex(f"p{i}", p, b, eng.ExecutionPhase.PREFILL, len(p)) for i, (p, b) in enumerate(zip(prompts, blocks))])
    for i, (p, b) in enumerate(zip(prompts, blocks)):
        slots = [b[t // 16] * 16 + t % 16 for t in range(len(p))]
        for lay in range(2):
            k, v = f8.gather(lay, slots)
            f32.key_cache[lay, slots], f32.value_cache[lay, slots] = k, v
    r32 = B200PagedModelRunner(copy.deepcopy(model), DEV, f32)

    class ReadOnly:
        """The kernels without those that write rows: a new row would be rounded in one pool and not
        in the other, so the step runs the last prompt token again, whose rows are there."""

        def __getattr__(self, name):
            if name == "paged_decode_append":
                raise AttributeError(name)
            return (lambda *a, **k: None) if name in ("kv_write_fp8", "kv_write") else getattr(ops, name)

    monkeypatch.setattr(runner_module, "_ops", ReadOnly())
    again = [Ex(f"d{i}", p, b, eng.ExecutionPhase.DECODE, 1) for i, (p, b) in enumerate(zip(prompts, blocks))]
    got, want = (r.forward(again).float() for r in (r8, r32))
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()


def test_compaction_between_engine_steps_changes_no_token():
    """A fragmented pool packed after every second step: the same tokens, from moved pages."""
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (40, 17, 130, 60, 3, 90)]
    model = small_model(torch.bfloat16, seed=1)
    moved = []

    def pack(steps, engine, runner, storage):
        if steps % 2 == 0:
            table = engine.scheduler.block_table
            before = table.tables()
            live = storage.compact(table)
            runner.forget_tables()
            assert live == engine.scheduler.block_pool.num_allocated_blocks
            moved.append(sum(a != b for x, y in zip(before.values(), table.tables().values()) for a, b in zip(x, y)))

    for make in (lambda: PagedKVStorage(2, 64, 16, 2, 128, torch.bfloat16, DEV),
                 lambda: Fp8PagedKVStorage(2, 64, 16, 2, 128, DEV)):
        plain = run_engine(model, make(), prompts, 64)
        moved.clear()
        packed = run_engine(model, make(), prompts, 64, between=pack)
        assert packed == plain and sum(moved) > 0
