"""Host logic of the runner over an 8-bit pool: what it hands to the attention calls of a step that
mixes decode rows with prompts. The kernels are stand-ins that note their arguments."""

from __future__ import annotations

import pytest
import torch

from llm_engineering_b200 import engine as eng
from llm_engineering_b200 import runner as runner_mod
from llm_engineering_b200.runner import B200PagedModelRunner
from llm_engineering_b200.storage import Fp8PagedKVStorage
from test_runner_cpu import CpuKernels, tiny_model

BS = 16


class Notes(CpuKernels):
    def __init__(self):
        self.decode, self.prefill = [], []

    @staticmethod
    def fp8_workspace_size(*args):
        return 16

    def kv_write_fp8(self, *args):
        pass

    def paged_decode_fp8(self, q, kc, vc, ks, vs, layer, bt, ctx, bs, scale, out=None, **kw):
        self.decode.append((bt.clone(), ctx.tolist(), bt.is_contiguous()))
        return out.zero_()

    def paged_prefill_fp8(self, q, kc, vc, ks, vs, layer, bt, cu, ctx, max_q, bs, scale, out=None,
                          max_context=None, **kw):
        self.prefill.append((bt.clone(), cu.tolist(), ctx.tolist(), bt.is_contiguous(), max_context))
        return out


class Execution:
    def __init__(self, name, length, q_len, blocks):
        req = eng.Request(request_id=name, prompt_token_ids=tuple(range(1, length + 1)), max_new_tokens=4,
                          ignore_eos=True)
        self.sequence = eng.SequenceState(request=req)
        self.phase = eng.ExecutionPhase.DECODE if q_len == 1 else eng.ExecutionPhase.PREFILL
        self.block_ids, self.length, self.query_length = tuple(blocks), length, q_len


@pytest.mark.parametrize("decode", [[], [90], [5, 64]])
@pytest.mark.parametrize("prompts", [[(20, 20)], [(40, 8), (17, 17), (3, 2)]])
def test_prompts_are_bounded_by_their_own_contexts(monkeypatch, decode, prompts):
    notes = Notes()
    monkeypatch.setattr(runner_mod, "_ops", notes)
    model = tiny_model()
    storage = Fp8PagedKVStorage(2, 64, BS, 2, 16, torch.device("cpu"))
    runner = B200PagedModelRunner(model, torch.device("cpu"), storage)
    free = iter(range(63, -1, -1))
    lengths = decode + [n for n, _ in prompts]
    blocks = [[next(free) for _ in range(-(-n // BS))] for n in lengths]
    q_lens = [1] * len(decode) + [q for _, q in prompts]
    runner.forward([Execution(f"r{i}", n, q, b) for i, (n, q, b) in enumerate(zip(lengths, q_lens, blocks))])
    nd = len(decode)
    assert len(notes.prefill) == 2 and len(notes.decode) == (2 if nd else 0)  # one per layer
    for table, cu, ctx, contiguous, bound in notes.prefill:
        assert bound == max(lengths[nd:]) and contiguous and len(table) == len(prompts)
        assert [row[:len(b)].tolist() for row, b in zip(table, blocks[nd:])] == blocks[nd:]
        assert ctx == lengths[nd:] and cu[0] == nd and cu[-1] == sum(q_lens)
    for table, ctx, contiguous in notes.decode:
        assert contiguous and ctx == lengths[:nd]
        assert [row[:len(b)].tolist() for row, b in zip(table, blocks)] == blocks[:nd]


@pytest.mark.parametrize("make", [lambda: Fp8PagedKVStorage(2, 64, BS, 2, 16, torch.device("cpu")),
                                  lambda: plain_storage()])
def test_tables_are_uploaded_anew_after_a_compaction(monkeypatch, make):
    """The device copy of the tables learns of new blocks only: moved ones would be read where they were."""
    notes = Notes()
    monkeypatch.setattr(runner_mod, "_ops", notes)
    seen = []
    monkeypatch.setattr(Notes, "build_metadata", staticmethod(
        lambda *a, **k: seen.append(CpuKernels.build_metadata(*a, **k)) or seen[-1]))
    storage = make()
    runner = B200PagedModelRunner(tiny_model(), torch.device("cpu"), storage)
    step = Execution("r", 40, 40, [9, 5, 30])
    runner.forward([step])
    assert seen[-1]["block_tables"][0].tolist() == [9, 5, 30]
    storage.compactions += 1  # what compact() does when it has moved the pages
    step.block_ids = (0, 1, 2)
    runner.forward([step])
    assert seen[-1]["block_tables"][0].tolist() == [0, 1, 2]


def plain_storage():
    from llm_engineering_b200.storage import PagedKVStorage

    s = PagedKVStorage(2, 64, BS, 2, 16, torch.float32, torch.device("cpu"))
    s.key_cache.zero_(), s.value_cache.zero_()
    return s
