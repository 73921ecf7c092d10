"""Paged KV storage with the reference layout, written through the K1 kernel.

Interface of ``PagedKVStorage`` (serving/engine/paged_kv_storage.py:6-174): the same
constructor, attributes (``key_cache``/``value_cache`` of shape
``[num_layers, num_blocks * block_size, num_kv_heads, head_dim]``, ``num_slots`` ...) and
``ValueError`` messages. ``scatter`` runs the CUDA KV-write kernel; ``gather`` exists for
callers that still want materialised histories (the paged attention kernels never call
it). ``copy_blocks`` and ``compact`` move pages for forked requests and a fragmented pool.

``Fp8PagedKVStorage`` holds the same pool in 8 bits: e4m3 codes with one power-of-two scale
for each (layer, block, KV head), half the bytes per token. Rows enter it by ``append``
(a block's scale depends on all of its rows, so single slots cannot be set), and the runner
takes it in place of ``PagedKVStorage``.
"""

from __future__ import annotations

from collections.abc import Sequence

import numpy as np
import torch

from . import ops


class PagedKVStorage:
    key_scales: torch.Tensor | None = None
    value_scales: torch.Tensor | None = None
    compactions = 0  # how often pages of this pool have moved

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int,
                 head_dim: int, dtype: torch.dtype, device: torch.device) -> None:
        for name, value in (("num_layers", num_layers), ("num_blocks", num_blocks),
                            ("block_size", block_size), ("num_kv_heads", num_kv_heads),
                            ("head_dim", head_dim)):
            if value <= 0:
                raise ValueError(f"{name} must be greater than zero.")
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = torch.device(device)
        self.num_slots = num_blocks * block_size
        shape = (num_layers, self.num_slots, num_kv_heads, head_dim)
        self.key_cache = torch.empty(shape, dtype=dtype, device=self.device)
        self.value_cache = torch.empty(shape, dtype=dtype, device=self.device)

    def _check_layer(self, layer_index: int) -> None:
        if not 0 <= layer_index < self.num_layers:
            raise ValueError("layer_index must be within the configured layers.")

    def _slot_tensor(self, slot_ids: Sequence[int] | torch.Tensor) -> torch.Tensor:
        if isinstance(slot_ids, torch.Tensor):
            arr = slot_ids.detach().to("cpu", torch.int64).numpy()
        else:
            arr = np.asarray(slot_ids, dtype=np.int64).reshape(-1)
        if arr.size and (arr.min() < 0 or arr.max() >= self.num_slots):
            raise ValueError("slot_ids must be within the configured physical slots.")
        return torch.from_numpy(arr.astype(np.int32)).to(self.key_cache.device, non_blocking=True)

    def copy_blocks(self, src_blocks: Sequence[int], dst_blocks: Sequence[int]) -> None:
        """Copy block src_blocks[i] to block dst_blocks[i] in every layer (what
        ``BlockTable.fork_request`` asks for). Targets must be distinct and not be sources."""
        src = np.asarray(src_blocks, dtype=np.int64).reshape(-1)
        dst = np.asarray(dst_blocks, dtype=np.int64).reshape(-1)
        if src.size != dst.size:
            raise ValueError("src_blocks and dst_blocks must have one entry per pair.")
        if src.size == 0:
            return
        if min(src.min(), dst.min()) < 0 or max(src.max(), dst.max()) >= self.num_blocks:
            raise ValueError("block ids must be within the configured physical blocks.")
        if np.unique(dst).size != dst.size or np.intersect1d(src, dst).size:
            raise ValueError("dst_blocks must be distinct and must not contain a source.")
        pairs = torch.from_numpy(np.stack([src, dst]).astype(np.int32)).to(self.key_cache.device)
        ops.copy_blocks(self.key_cache, self.value_cache, pairs[0], pairs[1], self.block_size,
                        self.key_scales, self.value_scales)

    def compact(self, block_table) -> int:
        """Move the blocks of every request in ``block_table`` (engine.BlockTable) to the front of
        the pool, in every layer, and rewrite the tables and the block pool. Returns the number
        of blocks in use. A runner on this pool uploads its tables anew in its next step. (It
        frees no memory: the pool's size is fixed. It is for programs that hand the pool's unused
        end to something else, or that want pages in few places.)"""
        lists = list(block_table.tables().values())
        if block_table.block_size != self.block_size or block_table.pool.num_blocks != self.num_blocks:
            raise ValueError("block_table must be over this pool's blocks.")
        if len({b for t in lists for b in t}) != block_table.pool.num_allocated_blocks:
            raise ValueError("blocks are allocated that no request of block_table holds.")
        width = max([1, *(len(t) for t in lists)])
        host = np.full((len(lists) + 1, width), -1, dtype=np.int32)
        for row, t in zip(host, lists):
            row[:len(t)] = t
        used = [len(t) * self.block_size for t in lists] + [0]
        dev = self.key_cache.device
        err = torch.zeros(1, dtype=torch.int32, device=dev)
        new_ids, live = ops.compact_blocks(
            self.key_cache, self.value_cache, torch.from_numpy(host).to(dev),
            torch.tensor(used, dtype=torch.int32, device=dev), self.block_size, self.key_scales,
            self.value_scales, err_flag=err)
        if int(err.item()):
            raise RuntimeError("block_table names blocks outside the pool.")
        self.compactions += 1
        block_table.apply_moves(new_ids.tolist())
        return int(live.item())

    def scatter(self, layer_index: int, slot_ids: Sequence[int] | torch.Tensor,
                keys: torch.Tensor, values: torch.Tensor) -> None:
        """Write row t of keys/values into slot slot_ids[t] of one layer (K1)."""
        self._check_layer(layer_index)
        slots = self._slot_tensor(slot_ids)
        expected = (slots.numel(), self.num_kv_heads, self.head_dim)
        if tuple(keys.shape) != expected:
            raise ValueError(f"keys must have shape {expected}.")
        if tuple(values.shape) != expected:
            raise ValueError(f"values must have shape {expected}.")
        if keys.dtype != self.dtype:
            raise ValueError("keys dtype must match the KV-cache dtype.")
        if values.dtype != self.dtype:
            raise ValueError("values dtype must match the KV-cache dtype.")
        if keys.device != self.key_cache.device:
            raise ValueError("keys device must match the KV-cache device.")
        if values.device != self.key_cache.device:
            raise ValueError("values device must match the KV-cache device.")
        ops.kv_write(self.key_cache, self.value_cache, layer_index, slots, keys, values)

    def gather(self, layer_index: int,
               slot_ids: Sequence[int] | torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows of the given slots in logical order (materialised copy)."""
        self._check_layer(layer_index)
        idx = self._slot_tensor(slot_ids).long()
        return (self.key_cache[layer_index].index_select(0, idx),
                self.value_cache[layer_index].index_select(0, idx))


class Fp8PagedKVStorage(PagedKVStorage):
    """The pool in 8 bits: ``key_cache``/``value_cache`` are float8_e4m3fn, and an element stands for
    its code times ``key_scales``/``value_scales`` [num_layers, num_blocks, num_kv_heads]."""

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int,
                 head_dim: int, device: torch.device) -> None:
        if head_dim % 8:
            raise ValueError("head_dim must be a multiple of 8 for an 8-bit cache.")
        super().__init__(num_layers, num_blocks, block_size, num_kv_heads, head_dim,
                         ops.FP8_DTYPE, device)
        shape = (num_layers, num_blocks, num_kv_heads)
        self.key_scales = torch.zeros(shape, dtype=torch.float32, device=self.device)
        self.value_scales = torch.zeros(shape, dtype=torch.float32, device=self.device)

    def append(self, layer_index: int, block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor,
               context_lens: torch.Tensor, max_q_len: int, keys: torch.Tensor,
               values: torch.Tensor, err_flag: torch.Tensor | None = None) -> None:
        """Append a packed batch's rows to its sequences (``ops.kv_write_fp8``)."""
        self._check_layer(layer_index)
        ops.kv_write_fp8(self.key_cache, self.value_cache, self.key_scales, self.value_scales,
                         layer_index, block_tables, cu_seqlens_q, context_lens, max_q_len,
                         self.block_size, keys, values, err_flag)

    def scatter(self, layer_index: int, slot_ids: Sequence[int] | torch.Tensor,
                keys: torch.Tensor, values: torch.Tensor) -> None:
        raise ValueError("an 8-bit cache takes rows by append, not by slot.")

    def gather(self, layer_index: int, slot_ids: Sequence[int] | torch.Tensor,
               dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows of the given slots in logical order, as values of ``dtype``."""
        self._check_layer(layer_index)
        return ops.kv_read_fp8(self.key_cache, self.value_cache, self.key_scales,
                               self.value_scales, layer_index, self._slot_tensor(slot_ids),
                               self.block_size, dtype)
