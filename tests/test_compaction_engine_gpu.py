"""A pool packed between engine steps by PagedKVStorage.compact alone: the runner sees that pages have
moved, and every request ends with the same tokens."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from llm_engineering_b200.storage import Fp8PagedKVStorage, PagedKVStorage
from test_speculative_gpu import DEV, run_engine, small_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("make", [lambda: PagedKVStorage(2, 64, 16, 2, 128, torch.bfloat16, DEV),
                                  lambda: Fp8PagedKVStorage(2, 64, 16, 2, 128, DEV)])
def test_compaction_needs_no_other_call(make):
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (40, 17, 130, 60, 3, 90)]
    model = small_model(torch.bfloat16, seed=1)
    moved = []

    def pack(steps, engine, runner, storage):
        table = engine.scheduler.block_table
        before = table.tables()
        storage.compact(table)
        moved.append(sum(a != b for x, y in zip(before.values(), table.tables().values()) for a, b in zip(x, y)))

    plain = run_engine(model, make(), prompts, 64)
    packed = run_engine(model, make(), prompts, 64, between=pack)
    assert packed == plain and sum(moved) > 0
