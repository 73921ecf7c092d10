"""Host bookkeeping of forks and compaction (block pool, block table, storage checks)."""

from __future__ import annotations

import pytest
import torch

from llm_engineering_b200 import engine as eng
from llm_engineering_b200.storage import Fp8PagedKVStorage, PagedKVStorage


def table(blocks=10, bs=4):
    return eng.BlockTable(eng.BlockPool(blocks), bs)


def test_fork_shares_full_blocks_and_copies_the_last():
    t = table()
    t.allocate_for_request("a", 10)  # blocks 0, 1 and half of 2
    assert t.fork_request("a", "b", 10) == ((2, 3),)
    assert t.blocks_for_request("b") == (0, 1, 3)
    assert [t.pool.block(i).ref_count for i in range(4)] == [2, 2, 1, 1]
    assert t.fork_request("b", "c", 8) == ()  # whole blocks only: nothing to copy
    assert t.blocks_for_request("c") == (0, 1)
    t.append_token("c", 8)
    assert t.blocks_for_request("c") == (0, 1, 4)
    t.free_request("a")
    assert [t.pool.block(i).ref_count for i in range(5)] == [2, 2, 0, 1, 1]
    t.free_request("b")
    t.free_request("c")
    assert t.pool.num_free_blocks == 10


def test_fork_refusals():
    t = table(blocks=3)
    t.allocate_for_request("a", 10)
    with pytest.raises(ValueError, match="Unknown request_id"):
        t.fork_request("x", "b", 4)
    with pytest.raises(ValueError, match="already has"):
        t.fork_request("a", "a", 4)
    with pytest.raises(ValueError, match="greater than zero"):
        t.fork_request("a", "b", 0)
    with pytest.raises(ValueError, match="more than"):
        t.fork_request("a", "b", 13)
    with pytest.raises(RuntimeError, match="free blocks"):
        t.fork_request("a", "b", 9)
    assert [t.pool.block(i).ref_count for i in range(3)] == [1, 1, 1]  # nothing half done


def test_apply_moves_keeps_references_and_resets_the_free_queue():
    t = table(blocks=6)
    t.allocate_for_request("a", 8)      # 0, 1
    t.allocate_for_request("b", 12)     # 2, 3, 4
    t.fork_request("b", "c", 8)         # shares 2, 3
    t.free_request("a")
    # live: 2 (twice), 3 (twice), 4 -> 3 and 4 move to 0 and 1
    t.apply_moves([-1, -1, 2, 0, 1, -1])
    assert t.blocks_for_request("b") == (2, 0, 1) and t.blocks_for_request("c") == (2, 0)
    assert [t.pool.block(i).ref_count for i in range(6)] == [2, 1, 2, 0, 0, 0]
    assert t.pool.allocate(3) == (3, 4, 5)
    for bad in ([0, 1, 2, 3, 4], [-1] * 6, [0, 0, 2, 3, 4, 5], [9, 1, 2, 3, 4, 5]):
        with pytest.raises(ValueError):
            t.apply_moves(bad)


def test_storage_refusals():
    dev = torch.device("cpu")
    s = PagedKVStorage(1, 4, 16, 1, 8, torch.float32, dev)
    with pytest.raises(ValueError, match="one entry per pair"):
        s.copy_blocks([0], [1, 2])
    with pytest.raises(ValueError, match="physical blocks"):
        s.copy_blocks([0], [4])
    with pytest.raises(ValueError, match="distinct"):
        s.copy_blocks([0, 1], [2, 2])
    with pytest.raises(ValueError, match="distinct"):
        s.copy_blocks([0, 1], [1, 2])
    s.copy_blocks([], [])
    with pytest.raises(ValueError, match="this pool"):
        s.compact(table(blocks=10, bs=16))
    t = table(blocks=4, bs=16)
    t.allocate_for_request("a", 20)
    t.pool.allocate(1)  # held by nobody's table: it would be taken for free
    with pytest.raises(ValueError, match="no request"):
        s.compact(t)
    f = Fp8PagedKVStorage(2, 4, 16, 1, 8, dev)
    assert f.key_cache.dtype == torch.float8_e4m3fn and f.key_scales.shape == (2, 4, 1)
    with pytest.raises(ValueError, match="append"):
        f.scatter(0, [0], torch.zeros(1, 1, 8), torch.zeros(1, 1, 8))
    with pytest.raises(ValueError, match="layer_index"):
        f.gather(2, [0])
    with pytest.raises(ValueError, match="multiple of 8"):
        Fp8PagedKVStorage(1, 4, 16, 1, 12, dev)
