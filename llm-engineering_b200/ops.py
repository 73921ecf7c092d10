"""Torch-facing wrappers of the C-ABI kernels.

Each function takes CUDA tensors, checks shapes/dtypes on the host, passes raw device
pointers, element strides and ``torch.cuda.current_stream()`` to the library, and
returns without synchronising. Nothing here computes attention itself: a tensor on the
wrong device or a missing library raises instead of falling back.
"""

from __future__ import annotations

import functools

import torch

from . import _lib

_DTYPE_CODES = {
    torch.bfloat16: _lib.B2P_BF16,
    torch.float16: _lib.B2P_F16,
    torch.float32: _lib.B2P_F32,
}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODES[dtype]
    except KeyError as exc:
        raise ValueError(f"unsupported KV dtype {dtype}") from exc


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (got {t.device}); the paged kernels have "
                         "no CPU path.")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _tok_head_strides(name: str, t: torch.Tensor) -> tuple[int, int]:
    if t.dim() != 3:
        raise ValueError(f"{name} must have shape (tokens, heads, head_dim)")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must have a contiguous head_dim")
    return t.stride(0), t.stride(1)


def _check_pool(key_cache: torch.Tensor, value_cache: torch.Tensor) -> None:
    _require_cuda("key_cache", key_cache)
    _require_cuda("value_cache", value_cache)
    if key_cache.shape != value_cache.shape or key_cache.dim() != 4:
        raise ValueError("key_cache/value_cache must both be [layers, slots, kv_heads, head_dim]")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("key_cache/value_cache must be contiguous")
    if key_cache.dtype != value_cache.dtype:
        raise ValueError("key_cache/value_cache dtypes differ")


def _int32(name: str, t: torch.Tensor) -> None:
    _require_cuda(name, t)
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 CUDA tensor")


def kv_write(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    layer_index: int,
    slot_mapping: torch.Tensor,
    keys: torch.Tensor,
    values: torch.Tensor,
    err_flag: torch.Tensor | None = None,
) -> None:
    """K1: write row t of keys/values into slot slot_mapping[t] of layer ``layer_index``.

    keys/values: (tokens, kv_heads, head_dim) views (any token/head strides).
    slot_mapping: int32 (tokens,); negative entries are skipped.
    """
    _check_pool(key_cache, value_cache)
    _require_cuda("keys", keys)
    _require_cuda("values", values)
    _int32("slot_mapping", slot_mapping)
    layers, slots, hkv, d = key_cache.shape
    if keys.shape != values.shape or keys.dim() != 3 or tuple(keys.shape[1:]) != (hkv, d):
        raise ValueError(f"keys/values must have shape (tokens, {hkv}, {d})")
    if keys.dtype != key_cache.dtype or values.dtype != key_cache.dtype:
        raise ValueError("keys/values dtype must match the KV-cache dtype")
    if slot_mapping.numel() != keys.shape[0]:
        raise ValueError("slot_mapping must have one entry per token")
    kt, kh = _tok_head_strides("keys", keys)
    vt, vh = _tok_head_strides("values", values)
    rc = _lib.load().b2p_kv_write(
        keys.data_ptr(), kt, kh, values.data_ptr(), vt, vh, key_cache.data_ptr(),
        value_cache.data_ptr(), slot_mapping.data_ptr(), keys.shape[0], layer_index, layers,
        slots, hkv, d, dtype_code(key_cache.dtype), _ptr(err_flag), _stream(key_cache.device),
    )
    _lib.check(rc, "b2p_kv_write")


def cuda_core_fallbacks() -> tuple[int, int]:
    """bf16/f16 launches of (decode, prefill) so far that ran on the CUDA-core kernels
    because the tensor-core kernels' preconditions were not met."""
    lib = _lib.load()
    return int(lib.b2p_cuda_core_fallbacks(2)), int(lib.b2p_cuda_core_fallbacks(3))


def reset_scratch(device: torch.device) -> None:
    """Zero the library's device-resident prefill claim counters on ``device`` (on its
    current stream), after a launch whose bounded waits gave up."""
    with torch.cuda.device(device):
        _lib.check(_lib.load().b2p_reset_scratch(_stream(torch.device(device))),
                   "b2p_reset_scratch")


def decode_workspace_size(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int) -> int:
    return int(_lib.load().b2p_paged_decode_workspace_size(num_seqs, num_q_heads, num_kv_heads,
                                                            head_dim))


def make_decode_workspace(max_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                          device: torch.device) -> torch.Tensor:
    """Zero-filled scratch for the split-K decode kernel (reusable across launches)."""
    n = decode_workspace_size(max_seqs, num_q_heads, num_kv_heads, head_dim)
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=device)


def paged_decode(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    layer_index: int,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    scale: float,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """K2: one query token per sequence attends its paged history.

    q: (num_seqs, num_q_heads, head_dim); returns out of the same shape.
    """
    _check_pool(key_cache, value_cache)
    _require_cuda("q", q)
    _int32("block_tables", block_tables)
    _int32("context_lens", context_lens)
    layers, slots, hkv, d = key_cache.shape
    n, hq, dq = q.shape
    if dq != d or q.dtype != key_cache.dtype:
        raise ValueError("q must match the pool's head_dim and dtype")
    if block_tables.dim() != 2 or block_tables.shape[0] < n or context_lens.numel() < n:
        raise ValueError("block_tables/context_lens must cover every sequence")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    qt, qhs = _tok_head_strides("q", q)
    ot, ohs = _tok_head_strides("out", out)
    if workspace is None:
        workspace = make_decode_workspace(n, hq, hkv, d, q.device)
    rc = _lib.load().b2p_paged_decode(
        q.data_ptr(), qt, qhs, key_cache.data_ptr(), value_cache.data_ptr(), layer_index, layers,
        slots, block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), n, hq,
        hkv, d, block_size, float(scale), out.data_ptr(), ot, ohs, workspace.data_ptr(),
        workspace.numel(), dtype_code(q.dtype), _ptr(err_flag), _stream(q.device),
    )
    _lib.check(rc, "b2p_paged_decode")
    return out


def paged_decode_append(
    q: torch.Tensor,
    new_keys: torch.Tensor,
    new_values: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    layer_index: int,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    scale: float,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """K1 + K2 for decode rows in one launch: stores each sequence's new K/V row (position
    ``context_lens[i] - 1``, slot from its block table) into the pool and attends over the
    whole history. q: (num_seqs, HQ, D); new_keys / new_values: (num_seqs, Hkv, D)."""
    _check_pool(key_cache, value_cache)
    _require_cuda("q", q)
    _int32("block_tables", block_tables)
    _int32("context_lens", context_lens)
    layers, slots, hkv, d = key_cache.shape
    n, hq, dq = q.shape
    if dq != d or q.dtype != key_cache.dtype:
        raise ValueError("q must match the pool's head_dim and dtype")
    for name, t in (("new_keys", new_keys), ("new_values", new_values)):
        _require_cuda(name, t)
        if t.dtype != key_cache.dtype or t.dim() != 3 or t.shape[0] < n or t.shape[1:] != (hkv, d):
            raise ValueError(f"{name} must be (num_seqs, num_kv_heads, head_dim) in the pool dtype")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a contiguous head_dim")
    if block_tables.dim() != 2 or block_tables.shape[0] < n or context_lens.numel() < n:
        raise ValueError("block_tables/context_lens must cover every sequence")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    qt, qhs = _tok_head_strides("q", q)
    ot, ohs = _tok_head_strides("out", out)
    if workspace is None:
        workspace = make_decode_workspace(n, hq, hkv, d, q.device)
    rc = _lib.load().b2p_paged_decode_append(
        q.data_ptr(), qt, qhs, new_keys.data_ptr(), new_keys.stride(0), new_keys.stride(1),
        new_values.data_ptr(), new_values.stride(0), new_values.stride(1),
        key_cache.data_ptr(), value_cache.data_ptr(), layer_index, layers, slots,
        block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), n, hq, hkv, d,
        block_size, float(scale), out.data_ptr(), ot, ohs, workspace.data_ptr(),
        workspace.numel(), dtype_code(q.dtype), _ptr(err_flag), _stream(q.device),
    )
    _lib.check(rc, "b2p_paged_decode_append")
    return out


def paged_prefill(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    layer_index: int,
    block_tables: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    context_lens: torch.Tensor,
    max_q_len: int,
    block_size: int,
    scale: float,
    out: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """K3: packed variable-length causal attention over the paged history.

    q: (rows, num_q_heads, head_dim); sequence i owns rows [cu_seqlens_q[i],
    cu_seqlens_q[i+1]) of q (int32, num_seqs + 1 entries, need not start at 0, so a
    trailing slice of a packed batch can be run with views of its metadata).
    """
    _check_pool(key_cache, value_cache)
    _require_cuda("q", q)
    _int32("block_tables", block_tables)
    _int32("cu_seqlens_q", cu_seqlens_q)
    _int32("context_lens", context_lens)
    layers, slots, hkv, d = key_cache.shape
    total_q, hq, dq = q.shape
    if dq != d or q.dtype != key_cache.dtype:
        raise ValueError("q must match the pool's head_dim and dtype")
    num_seqs = cu_seqlens_q.numel() - 1
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    qt, qhs = _tok_head_strides("q", q)
    ot, ohs = _tok_head_strides("out", out)
    rc = _lib.load().b2p_paged_prefill(
        q.data_ptr(), qt, qhs, key_cache.data_ptr(), value_cache.data_ptr(), layer_index, layers,
        slots, block_tables.data_ptr(), block_tables.stride(0), cu_seqlens_q.data_ptr(),
        context_lens.data_ptr(), num_seqs, total_q, max_q_len, hq, hkv, d, block_size,
        float(scale), out.data_ptr(), ot, ohs, dtype_code(q.dtype), _ptr(err_flag),
        _stream(q.device),
    )
    _lib.check(rc, "b2p_paged_prefill")
    return out


def build_metadata(
    query_lens: torch.Tensor,
    context_lens: torch.Tensor,
    table_rows: torch.Tensor,
    block_mirror: torch.Tensor,
    block_size: int,
    total_q: int,
    max_blocks_per_seq: int,
    err_flag: torch.Tensor | None = None,
) -> dict[str, torch.Tensor]:
    """K4: packed batch metadata from a per-step execution descriptor (all int32 CUDA)."""
    for name, t in (("query_lens", query_lens), ("context_lens", context_lens),
                    ("table_rows", table_rows), ("block_mirror", block_mirror)):
        _int32(name, t)
    n = query_lens.numel()
    dev = query_lens.device
    out = {
        "cu_seqlens_q": torch.empty(n + 1, dtype=torch.int32, device=dev),
        "cu_seqlens_k": torch.empty(n + 1, dtype=torch.int32, device=dev),
        "positions": torch.empty(total_q, dtype=torch.int64, device=dev),
        "slot_mapping": torch.empty(total_q, dtype=torch.int32, device=dev),
        "logit_indices": torch.empty(n, dtype=torch.int64, device=dev),
        "block_tables": torch.empty((n, max(max_blocks_per_seq, 1)), dtype=torch.int32,
                                    device=dev),
    }
    rc = _lib.load().b2p_build_metadata(
        query_lens.data_ptr(), context_lens.data_ptr(), table_rows.data_ptr(), n,
        block_mirror.data_ptr(), block_mirror.stride(0), block_mirror.shape[0], block_size,
        out["cu_seqlens_q"].data_ptr(), out["cu_seqlens_k"].data_ptr(),
        out["positions"].data_ptr(), out["slot_mapping"].data_ptr(),
        out["logit_indices"].data_ptr(), out["block_tables"].data_ptr(), max_blocks_per_seq,
        total_q, _ptr(err_flag), _stream(dev),
    )
    _lib.check(rc, "b2p_build_metadata")
    return out


def lm_head_argmax_workspace_size(rows: int) -> int:
    """Bytes of the K6 workspace for up to ``rows`` rows (keys and a counter; rows are
    counted rounded up to the kernel's 128-row tiles)."""
    return int(_lib.load().b2p_lm_head_argmax_workspace_size(rows + (-rows) % 128))


def lm_head_argmax(
    hidden: torch.Tensor,
    weight: torch.Tensor,
    workspace: torch.Tensor,
    out_ids: torch.Tensor | None = None,
    out_max: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
    rows: int | None = None,
) -> torch.Tensor | None:
    """K6: greedy token ids ``argmax_v round(hidden[r] . weight[v])`` for the first ``rows``
    rows of hidden (default: all).

    hidden (n, hidden_size) and weight (vocab, hidden_size) are bf16 or f16 CUDA tensors
    with contiguous rows; the logits are rounded to their dtype before the argmax (the LM
    head's own output type) and never written. The kernel takes rows in tiles of 128: a
    hidden whose n is a multiple of 128 is used as it is (rows past ``rows`` are computed
    and dropped), any other is copied into a zero-padded one first. ``workspace`` is a uint8
    CUDA tensor of at least ``lm_head_argmax_workspace_size(n rounded up to 128)`` bytes,
    zero before its first use (each launch leaves it zero). Returns the int64 ids of the
    first ``rows`` rows, or None when the dtype or shape is outside what the kernel takes
    (the caller then computes logits).
    """
    _require_cuda("hidden", hidden)
    _require_cuda("weight", weight)
    _require_cuda("workspace", workspace)
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError("hidden must be (rows, hidden_size) and weight (vocab, hidden_size)")
    if hidden.dtype != weight.dtype:
        raise ValueError("hidden and weight dtypes differ")
    if hidden.stride(1) != 1 or weight.stride(1) != 1:
        raise ValueError("hidden and weight rows must be contiguous")
    if hidden.dtype not in (torch.bfloat16, torch.float16) or hidden.shape[1] % 64:
        return None
    n = hidden.shape[0]
    rows = n if rows is None else rows
    if not 0 <= rows <= n:
        raise ValueError("rows must lie within hidden's rows")
    if n % 128:
        padded = hidden.new_zeros((n + (-n) % 128, hidden.shape[1]))
        padded[:n] = hidden
        hidden = padded
    n = hidden.shape[0]
    dev = hidden.device
    for name, t, dt in (("out_ids", out_ids, torch.int64), ("out_max", out_max, torch.float32)):
        if t is not None and (t.dtype != dt or not t.is_contiguous() or t.numel() < rows):
            raise ValueError(f"{name} must be a contiguous {dt} tensor of at least rows entries")
    # the kernel writes one entry per padded row: the caller's tensors when they are large
    # enough, else scratch whose first rows are copied back
    ids = out_ids if out_ids is not None and out_ids.numel() >= n else \
        torch.empty(n, dtype=torch.int64, device=dev)
    mx = out_max if out_max is None or out_max.numel() >= n else \
        torch.empty(n, dtype=torch.float32, device=dev)
    rc = _lib.load().b2p_lm_head_argmax(
        hidden.data_ptr(), hidden.stride(0), weight.data_ptr(), weight.stride(0), n,
        weight.shape[0], hidden.shape[1], dtype_code(hidden.dtype), ids.data_ptr(),
        _ptr(mx), workspace.data_ptr(), workspace.numel(), _ptr(err_flag), _stream(dev),
    )
    if rc == _lib.B2P_EUNSUPPORTED:
        return None
    _lib.check(rc, "b2p_lm_head_argmax")
    if out_ids is not None and ids is not out_ids:
        out_ids[:rows].copy_(ids[:rows])
        ids = out_ids
    if out_max is not None and mx is not out_max:
        out_max[:rows].copy_(mx[:rows])
    return ids[:rows]


# ---------------------------------------------------------------------- 8-bit cache, K7 - K9
FP8_DTYPE = torch.float8_e4m3fn


# The current stream's handle and the current device's index without torch.cuda's wrappers: the
# calls below take a few microseconds on the host, of which those two would be one. For the same
# reason outputs come from torch.empty_strided, in two thirds of torch.empty's time.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _call(name: str, index: int, *args) -> None:
    """Launch on CUDA device ``index``'s current stream, whichever device is current."""
    fn = getattr(_lib.load(), name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _index_of(name: str, t: torch.Tensor) -> int:
    """CUDA device index of t."""
    index = t.get_device()
    if index < 0:
        _require_cuda(name, t)
    return index


def _on(index: int, name: str, t: torch.Tensor) -> None:
    if t.get_device() != index:
        _require_cuda(name, t)
        raise ValueError(f"{name} is on {t.device}, the other tensors on cuda:{index}")


def _vector(index: int, name: str, t: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dtype is not dtype or not t.is_contiguous():
        _require_cuda(name, t)
        raise ValueError(f"{name} must be a contiguous {dtype} CUDA tensor")
    if t.get_device() != index:
        _on(index, name, t)


def _err_flag(index: int, err_flag: torch.Tensor | None) -> int | None:
    if err_flag is None:
        return None
    _vector(index, "err_flag", err_flag, torch.int32)
    return err_flag.data_ptr()


def _check_fp8_pool(key_cache: torch.Tensor, value_cache: torch.Tensor, key_scales: torch.Tensor,
                    value_scales: torch.Tensor, block_size: int) -> tuple[int, torch.Size]:
    """(device index, pool shape) of a valid 8-bit pool."""
    index = key_cache.get_device()
    if index < 0:
        _require_cuda("key_cache", key_cache)
    shape = key_cache.shape
    if value_cache.shape != shape or len(shape) != 4:
        raise ValueError("key_cache/value_cache must both be [layers, slots, kv_heads, head_dim]")
    if key_cache.dtype is not FP8_DTYPE or value_cache.dtype is not FP8_DTYPE:
        raise ValueError(f"an 8-bit pool must be {FP8_DTYPE} (got {key_cache.dtype}, {value_cache.dtype})")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise ValueError("key_cache/value_cache must be contiguous")
    layers, slots, hkv, _ = shape
    if block_size <= 0 or slots % block_size:
        raise ValueError("the pool's slots must be a multiple of block_size")
    want = (layers, slots // block_size, hkv)
    if key_scales.shape != want or value_scales.shape != want:
        raise ValueError(f"key_scales/value_scales must have shape {want}")
    if value_cache.get_device() != index:
        _on(index, "value_cache", value_cache)
    _vector(index, "key_scales", key_scales, torch.float32)
    _vector(index, "value_scales", value_scales, torch.float32)
    return index, shape


def _check_tables(index: int, num_seqs: int, block_tables: torch.Tensor,
                  context_lens: torch.Tensor) -> int:
    """The block tables' width."""
    _vector(index, "block_tables", block_tables, torch.int32)
    _vector(index, "context_lens", context_lens, torch.int32)
    shape = block_tables.shape
    if len(shape) != 2 or shape[0] < num_seqs or context_lens.numel() < num_seqs or num_seqs < 0:
        raise ValueError("block_tables/context_lens must cover every sequence")
    return shape[1]


def kv_write_fp8(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    layer_index: int,
    block_tables: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    context_lens: torch.Tensor,
    max_q_len: int,
    block_size: int,
    keys: torch.Tensor,
    values: torch.Tensor,
    err_flag: torch.Tensor | None = None,
) -> None:
    """K7: append a packed batch's new K/V rows to an 8-bit cache.

    key_cache/value_cache: float8_e4m3fn [layers, slots, kv_heads, head_dim]; key_scales/
    value_scales: float32 [layers, blocks, kv_heads]; an element stands for code * scale.
    Sequence i owns rows [cu_seqlens_q[i], cu_seqlens_q[i+1]) of keys/values (bf16, f16 or fp32,
    any token/head strides) and appends them at positions ``context_lens[i] - q_len ..
    context_lens[i] - 1`` through its block table. ``max_q_len`` bounds the q_len (a longer
    sequence is skipped and flagged). A block's scale is the smallest power of two (from 2**-110)
    that holds its rows; a write that covers the block's first slot starts it anew, any other one
    rounds the rows before it to the new scale where that grows. A non-finite row makes the
    scale NaN. Two sequences of one call must not append to the same block.
    """
    index, (layers, slots, hkv, d) = _check_fp8_pool(key_cache, value_cache, key_scales,
                                                     value_scales, block_size)
    n = cu_seqlens_q.numel() - 1
    _vector(index, "cu_seqlens_q", cu_seqlens_q, torch.int32)
    width = _check_tables(index, n, block_tables, context_lens)
    _on(index, "keys", keys)
    _on(index, "values", values)
    shape = keys.shape
    if values.shape != shape or len(shape) != 3 or shape[1] != hkv or shape[2] != d:
        raise ValueError(f"keys/values must have shape (tokens, {hkv}, {d})")
    if keys.dtype is not values.dtype:
        raise ValueError("keys/values dtypes differ")
    kt, kh, kd = keys.stride()
    vt, vh, vd = values.stride()
    if kd != 1 or vd != 1:
        raise ValueError("keys/values must have a contiguous head_dim")
    _call("b2p_kv_write_fp8", index, keys.data_ptr(), kt, kh, values.data_ptr(), vt, vh,
          key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(),
          value_scales.data_ptr(), block_tables.data_ptr(), width,
          cu_seqlens_q.data_ptr(), context_lens.data_ptr(), n, shape[0], max_q_len,
          layer_index, layers, slots, hkv, d, block_size, dtype_code(keys.dtype),
          _err_flag(index, err_flag))


def kv_read_fp8(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    layer_index: int,
    slot_mapping: torch.Tensor,
    block_size: int,
    dtype: torch.dtype,
    err_flag: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of the given slots (int32) as values of ``dtype``: (keys, values), each
    (rows, kv_heads, head_dim). Negative slots give zero rows; values past f16's range read as its
    largest finite one."""
    index, (layers, slots, hkv, d) = _check_fp8_pool(key_cache, value_cache, key_scales,
                                                     value_scales, block_size)
    _vector(index, "slot_mapping", slot_mapping, torch.int32)
    code = dtype_code(dtype)
    n = slot_mapping.numel()
    keys = torch.empty_strided((n, hkv, d), (hkv * d, d, 1), dtype=dtype, device=key_cache.device)
    values = torch.empty_like(keys)
    _call("b2p_kv_read_fp8", index, key_cache.data_ptr(), value_cache.data_ptr(),
          key_scales.data_ptr(), value_scales.data_ptr(), slot_mapping.data_ptr(), n,
          keys.data_ptr(), values.data_ptr(), layer_index, layers, slots, hkv, d, block_size, code,
          _err_flag(index, err_flag))
    return keys, values


@functools.cache
def _row_columns() -> int:
    """(row, query head of a KV head) pairs per sequence up to which a call needs no scratch."""
    return int(_lib.load().b2p_paged_fp8_row_columns())


def fp8_workspace_size(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                       max_q_len: int = 1) -> int:
    return int(_lib.load().b2p_paged_fp8_workspace_size(num_seqs, num_q_heads, num_kv_heads,
                                                        head_dim, max_q_len))


def make_fp8_workspace(max_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                       device: torch.device, max_q_len: int = 1) -> torch.Tensor:
    """Zero-filled scratch of the attention calls over the 8-bit cache: for up to ``max_seqs``
    sequences of up to ``max_q_len`` rows, reusable across layers and steps on one stream."""
    n = fp8_workspace_size(max_seqs, num_q_heads, num_kv_heads, head_dim, max_q_len)
    return torch.zeros(max(n, 16), dtype=torch.uint8, device=device)


def _fp8_query(index: int, head_dim: int, q: torch.Tensor, out: torch.Tensor | None):
    """(dtype code, out, q's and out's token and head strides) of a valid query."""
    _on(index, "q", q)
    if q.dim() != 3 or q.shape[2] != head_dim:
        raise ValueError("q must be (rows, num_q_heads, head_dim) with the pool's head_dim")
    code = dtype_code(q.dtype)
    qt, qh, qd = q.stride()
    if out is None:
        if q.is_contiguous():
            return code, torch.empty_like(q), qt, qh, q.shape[1] * head_dim, head_dim
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _on(index, "out", out)
        if out.shape != q.shape or out.dtype is not q.dtype:
            raise ValueError("out must have q's shape and dtype")
    ot, oh, od = out.stride()
    if qd != 1 or od != 1:
        raise ValueError("q and out must have a contiguous head_dim")
    return code, out, qt, qh, ot, oh


def _fp8_workspace(index: int, workspace: torch.Tensor | None, n: int, hq: int, hkv: int, d: int,
                   max_q_len: int) -> torch.Tensor:
    if workspace is None:
        return make_fp8_workspace(n, hq, hkv, d, torch.device("cuda", index), max_q_len)
    _vector(index, "workspace", workspace, torch.uint8)
    return workspace


def paged_decode_fp8(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    layer_index: int,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    scale: float,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
) -> torch.Tensor:
    """K2 over the 8-bit cache: one query token per sequence attends its paged history.

    q: (num_seqs, num_q_heads, head_dim) in bf16, f16 or fp32; returns out of the same shape.
    """
    index, (layers, slots, hkv, d) = _check_fp8_pool(key_cache, value_cache, key_scales,
                                                     value_scales, block_size)
    code, out, qt, qh, ot, oh = _fp8_query(index, d, q, out)
    n, hq, _ = q.shape
    width = _check_tables(index, n, block_tables, context_lens)
    workspace = _fp8_workspace(index, workspace, n, hq, hkv, d, 1)
    _call("b2p_paged_decode_fp8", index, q.data_ptr(), qt, qh, key_cache.data_ptr(),
          value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), layer_index,
          layers, slots, block_tables.data_ptr(), width, context_lens.data_ptr(), n, hq, hkv, d,
          block_size, scale, out.data_ptr(), ot, oh, workspace.data_ptr(), workspace.numel(), code,
          _err_flag(index, err_flag))
    return out


def paged_prefill_fp8(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    layer_index: int,
    block_tables: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    context_lens: torch.Tensor,
    max_q_len: int,
    block_size: int,
    scale: float,
    out: torch.Tensor | None = None,
    workspace: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
    max_context: int | None = None,
) -> torch.Tensor:
    """K3 over the 8-bit cache: packed variable-length causal attention over the paged history
    (the rows of drafted tokens, of prompt slices or of whole prompts).

    q: (rows, num_q_heads, head_dim); sequence i owns rows [cu_seqlens_q[i], cu_seqlens_q[i+1]) and
    row j of it sits at position ``context_lens[i] - q_len + j``. ``max_q_len`` bounds the q_len
    (rows of a longer sequence are flagged, or computed all the same). Rows of q that no sequence
    owns are left alone in out. Calls of many rows widen the histories into a 16-bit copy, allocated
    for the call, of one layer's blocks: ``num_seqs * block_tables.shape[1]`` of them or as many as the
    pool has, whichever are fewer (with fp32 partial results where few query tiles are spread over
    the SMs by their keys). ``max_context`` bounds the context_lens where the tables are wider than
    those need: the runs of keys are sized by it, else by the tables' width (a longer context is cut
    and flagged, or attended all the same). The copy is in q's type: with f16 queries over a pool that bf16 or fp32 rows
    went into, values past 65,536 are flagged (B2P_DEV_VALUE_RANGE) and cut.
    """
    index, (layers, slots, hkv, d) = _check_fp8_pool(key_cache, value_cache, key_scales,
                                                     value_scales, block_size)
    code, out, qt, qh, ot, oh = _fp8_query(index, d, q, out)
    total_q, hq, _ = q.shape
    n = cu_seqlens_q.numel() - 1
    _vector(index, "cu_seqlens_q", cu_seqlens_q, torch.int32)
    width = _check_tables(index, n, block_tables, context_lens)
    workspace = _fp8_workspace(index, workspace, n, hq, hkv, d, max_q_len)
    reach = width
    if max_context is not None:
        if max_context < 0:
            raise ValueError("max_context must not be negative")
        reach = min(width, max(1, -(-max_context // block_size)))
    scratch, size = None, 0
    if max_q_len * hq > _row_columns() * hkv:
        size = _lib.load().b2p_paged_prefill_fp8_pool_scratch_size(
            n, total_q, reach, slots, hq, hkv, d, block_size, max_q_len, code)
        scratch = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    _call("b2p_paged_prefill_fp8_reach", index, q.data_ptr(), qt, qh, key_cache.data_ptr(),
          value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), layer_index,
          layers, slots, block_tables.data_ptr(), width, reach, cu_seqlens_q.data_ptr(),
          context_lens.data_ptr(), n, total_q, max_q_len, hq, hkv, d, block_size, scale,
          out.data_ptr(), ot, oh, workspace.data_ptr(), workspace.numel(), _ptr(scratch), size,
          code, _err_flag(index, err_flag))
    return out


def _drafts_out(n: int, max_drafts: int, device: torch.device):
    row = max_drafts + 1
    return (torch.empty_strided((n, row), (row, 1), dtype=torch.int64, device=device),
            torch.empty_strided((n,), (1,), dtype=torch.int32, device=device))


def _check_drafts(index: int, draft_tokens: torch.Tensor, cu_drafts: torch.Tensor,
                  max_drafts: int) -> int:
    _vector(index, "cu_drafts", cu_drafts, torch.int32)
    _vector(index, "draft_tokens", draft_tokens, torch.int64)
    n = cu_drafts.numel() - 1
    if max_drafts < 0 or n < 0:
        raise ValueError("max_drafts must not be negative and cu_drafts needs an entry")
    return n


def verify_drafts(
    target_probs: torch.Tensor,
    draft_tokens: torch.Tensor,
    cu_drafts: torch.Tensor,
    accept_draws: torch.Tensor,
    sample_draws: torch.Tensor,
    max_drafts: int,
    draft_probs: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """K8: verify drafted tokens against the target model's probabilities.

    Sequence i drafted ``draft_tokens[cu_drafts[i]:cu_drafts[i+1]]`` (int64; cu_drafts int32) and
    owns the rows ``cu_drafts[i] + i .. cu_drafts[i+1] + i`` of target_probs (one more than it
    drafted; bf16, f16 or fp32, rows contiguous). draft_probs has one row per draft, or is None
    when every draft is certain (prompt lookup, greedy drafts). Draft j stands while
    ``accept_draws[j] * q_j(x_j) < p_j(x_j)``; one more token is drawn with ``sample_draws[i]``
    from max(p - q, 0) of the first rejected row, or from p of the last row. Draws are fp32 in
    [0, 1). NaN and negative probabilities, in either tensor, count as zero. Returns (tokens,
    accepted): int64 (num_seqs, max_drafts + 1), the standing drafts, then
    the drawn token, then -1; and int32 (num_seqs,), how many drafts stand.
    """
    index = _index_of("target_probs", target_probs)
    n = _check_drafts(index, draft_tokens, cu_drafts, max_drafts)
    total = draft_tokens.numel()
    dtype = target_probs.dtype
    code = dtype_code(dtype)
    if target_probs.dim() != 2 or target_probs.shape[0] != total + n:
        raise ValueError(f"target_probs must be ({total + n}, vocab)")
    vocab = target_probs.shape[1]
    t_row, one = target_probs.stride()
    if one != 1 and vocab > 1:
        raise ValueError("target_probs must have contiguous rows")
    q_ptr, q_row = None, 0
    if draft_probs is not None:
        _on(index, "draft_probs", draft_probs)
        if draft_probs.shape != (total, vocab) or draft_probs.dtype is not dtype:
            raise ValueError(f"draft_probs must be ({total}, {vocab}) in target_probs' dtype")
        q_row, one = draft_probs.stride()
        if one != 1 and vocab > 1:
            raise ValueError("draft_probs must have contiguous rows")
        q_ptr = draft_probs.data_ptr() or None  # no drafts: an empty tensor
    _vector(index, "accept_draws", accept_draws, torch.float32)
    _vector(index, "sample_draws", sample_draws, torch.float32)
    if accept_draws.numel() != total or sample_draws.numel() != n:
        raise ValueError(f"accept_draws must have {total} entries and sample_draws {n}")
    tokens, accepted = _drafts_out(n, max_drafts, target_probs.device)
    _call("b2p_verify_drafts", index, target_probs.data_ptr(), t_row, q_ptr, q_row,
          draft_tokens.data_ptr(), cu_drafts.data_ptr(), accept_draws.data_ptr(),
          sample_draws.data_ptr(), n, total, max_drafts, vocab, code, tokens.data_ptr(),
          max_drafts + 1, accepted.data_ptr(), _err_flag(index, err_flag))
    return tokens, accepted


def verify_drafts_greedy(
    target_ids: torch.Tensor,
    draft_tokens: torch.Tensor,
    cu_drafts: torch.Tensor,
    max_drafts: int,
    err_flag: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The greedy form of ``verify_drafts``: target_ids (int64, drafts + num_seqs) holds the
    arg-max of each target row (what ``lm_head_argmax`` gives); drafts stand while they equal it."""
    index = _index_of("target_ids", target_ids)
    n = _check_drafts(index, draft_tokens, cu_drafts, max_drafts)
    total = draft_tokens.numel()
    _vector(index, "target_ids", target_ids, torch.int64)
    if target_ids.numel() != total + n:
        raise ValueError(f"target_ids must have {total + n} entries")
    tokens, accepted = _drafts_out(n, max_drafts, target_ids.device)
    _call("b2p_verify_drafts_greedy", index, target_ids.data_ptr(), draft_tokens.data_ptr(),
          cu_drafts.data_ptr(), n, total, max_drafts, tokens.data_ptr(), max_drafts + 1,
          accepted.data_ptr(), _err_flag(index, err_flag))
    return tokens, accepted


def _check_pages(key_cache: torch.Tensor, value_cache: torch.Tensor, block_size: int,
                 key_scales: torch.Tensor | None, value_scales: torch.Tensor | None
                 ) -> tuple[int, torch.Size]:
    """(device index, pool shape) of a valid pool of any dtype."""
    if key_cache.dtype is FP8_DTYPE:
        if key_scales is None or value_scales is None:
            raise ValueError("an 8-bit pool needs its key_scales and value_scales")
        return _check_fp8_pool(key_cache, value_cache, key_scales, value_scales, block_size)
    _check_pool(key_cache, value_cache)
    dtype_code(key_cache.dtype)
    if key_scales is not None or value_scales is not None:
        raise ValueError("only an 8-bit pool has scales")
    if block_size <= 0 or key_cache.shape[1] % block_size:
        raise ValueError("the pool's slots must be a multiple of block_size")
    index = key_cache.get_device()
    _on(index, "value_cache", value_cache)
    return index, key_cache.shape


def copy_blocks(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    src_blocks: torch.Tensor,
    dst_blocks: torch.Tensor,
    block_size: int,
    key_scales: torch.Tensor | None = None,
    value_scales: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
) -> None:
    """K9: copy block src_blocks[i] to block dst_blocks[i] in every layer of K and V (and of the
    scales of an 8-bit pool). int32 CUDA vectors; a pair with a negative id is skipped. Targets
    must be distinct, and none of them a source of the same call."""
    index, (layers, slots, hkv, d) = _check_pages(key_cache, value_cache, block_size, key_scales,
                                                  value_scales)
    _vector(index, "src_blocks", src_blocks, torch.int32)
    _vector(index, "dst_blocks", dst_blocks, torch.int32)
    pairs = src_blocks.numel()
    if dst_blocks.numel() != pairs:
        raise ValueError("src_blocks and dst_blocks must have one entry per pair")
    _call("b2p_copy_blocks", index, key_cache.data_ptr(), value_cache.data_ptr(), _ptr(key_scales),
          _ptr(value_scales), src_blocks.data_ptr(), dst_blocks.data_ptr(), pairs, layers, slots,
          hkv, d, key_cache.element_size(), block_size, _err_flag(index, err_flag))


def compact_blocks(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    key_scales: torch.Tensor | None = None,
    value_scales: torch.Tensor | None = None,
    err_flag: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """K9: move the live blocks (those in the first ceil(context / block_size) entries of each
    row of block_tables) into the first blocks of the pool, in every layer, and rewrite
    block_tables in place. Returns (new_ids, num_live): int32 (num_blocks,), the new id of each
    live block and -1 for the others, and int32 (1,). Live blocks already in place stay; the
    j-th of the others, in ascending order, goes to the j-th free block. A block that no row names
    counts as free: pass every table that is in use."""
    index, (layers, slots, hkv, d) = _check_pages(key_cache, value_cache, block_size, key_scales,
                                                  value_scales)
    n = context_lens.numel()
    width = _check_tables(index, n, block_tables, context_lens)
    dev, blocks = key_cache.device, slots // block_size
    size = _lib.load().b2p_compact_blocks_workspace_size(blocks)
    workspace = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=dev)
    new_ids = torch.empty_strided((blocks,), (1,), dtype=torch.int32, device=dev)
    num_live = torch.empty_strided((1,), (1,), dtype=torch.int32, device=dev)
    _call("b2p_compact_blocks", index, key_cache.data_ptr(), value_cache.data_ptr(),
          _ptr(key_scales), _ptr(value_scales), block_tables.data_ptr(), width, width, context_lens.data_ptr(), n, layers, slots, hkv, d,
          key_cache.element_size(), block_size, new_ids.data_ptr(), num_live.data_ptr(),
          workspace.data_ptr(), size, _err_flag(index, err_flag))
    return new_ids, num_live
