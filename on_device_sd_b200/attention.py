"""The attention side of a decoding step over a paged key-value cache: the cache write (with head norms and rotary
embedding in the same launch) and the attention of new tokens, single ones (draft step) or spans (verify step).

The cache tensors are the reference's, [num_blocks, block_size, kv_heads, head_dim] (demo/src/memory/paged_kv_cache.py:228),
and stay the caller's.  All calls run on the current stream of their tensors' device, never synchronise and can be
captured into CUDA graphs.  `status`, where given, is an int32 tensor of one element on the same device that the kernels
OR DEV_* bits into (include/b200moe.h); the caller zeroes and reads it."""
from __future__ import annotations

from contextlib import nullcontext
from ctypes import byref, c_int64
from typing import Dict, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import PagedAttentionArgs, StoreKvArgs, check
from .context import _stream, dtype_tag

_WORKSPACE: Dict[Tuple, int] = {}


def _on(device: torch.device):
    """The library launches on the current device; switch only where the tensors live elsewhere."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _need(t: torch.Tensor, name: str, device: torch.device, dtype: Optional[torch.dtype], dims: int) -> None:
    if t.device != device or not t.is_cuda:
        raise ValueError(f"{name} must live on {device}, got {t.device} (this package has no CPU path)")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")


def _index(t: torch.Tensor, name: str, device: torch.device, length: int) -> int:
    """Checks an index vector and returns 1 for int64, 0 for int32."""
    _need(t, name, device, None, 1)
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be int64 or int32, got {t.dtype}")
    if t.shape[0] != length or (length > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be contiguous of length {length}, got {tuple(t.shape)}")
    return 1 if t.dtype == torch.int64 else 0


def _status_ptr(status: Optional[torch.Tensor], device: torch.device) -> Optional[int]:
    if status is None:
        return None
    if status.device != device or status.dtype != torch.int32 or status.numel() != 1:
        raise ValueError(f"status must be an int32 tensor of one element on {device}")
    return status.data_ptr()


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, device: torch.device, dtype: torch.dtype, kv_heads: Optional[int], head_dim: int):
    _need(k_cache, "k_cache", device, dtype, 4)
    _need(v_cache, "v_cache", device, dtype, 4)
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("k_cache and v_cache must have the same shape and strides")
    if k_cache.stride(3) != 1 or k_cache.shape[3] != head_dim or (kv_heads is not None and k_cache.shape[2] != kv_heads):
        raise ValueError(f"the caches must be [blocks, block_size, {'kv_heads' if kv_heads is None else kv_heads}, {head_dim}] with contiguous heads, "
                         f"got {tuple(k_cache.shape)}")
    if k_cache.shape[1] == 0:
        raise ValueError("the caches need a block size of at least one slot")
    return k_cache.shape[0], k_cache.shape[1]


def rotary_table(head_dim: int, max_position: int, base: float = 1e6, device: Optional[torch.device] = None) -> torch.Tensor:
    """The fp32 angle table [max_position, head_dim] that rope_store_kvcache takes: cos of the position's head_dim/2 angles,
    then sin.  Angles are formed in fp64, where a far position times a frequency still has all its digits."""
    inv = base ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), dim=-1).float().to(device or "cpu")


def _store(query, key, value, positions, cos_sin, k_cache, v_cache, slot_mapping, q_norm_weight, k_norm_weight, eps, out, status):
    dev, dt = key.device, key.dtype
    tag = dtype_tag(dt)
    _need(key, "key", dev, dt, 3)
    T, hk, D = key.shape
    _need(value, "value", dev, dt, 3)
    if value.shape != key.shape:
        raise ValueError(f"key and value must have the same shape, got {tuple(key.shape)} and {tuple(value.shape)}")
    blocks, page = _cache(k_cache, v_cache, dev, dt, hk, D)
    slots64 = _index(slot_mapping, "slot_mapping", dev, T)
    if key.stride(2) != 1 or value.stride(2) != 1:
        raise ValueError("heads must be contiguous")
    ks, vs, cs = key.stride(), value.stride(), k_cache.stride()
    hq, qs, os_, q_ptr, o_ptr = 0, (0, 0), (0, 0), None, None
    if query is not None:
        _need(query, "query", dev, dt, 3)
        hq = query.shape[1]
        if query.shape[0] != T or query.shape[2] != D or query.stride(2) != 1:
            raise ValueError(f"query must be [{T}, heads, {D}] with contiguous heads, got {tuple(query.shape)}")
        if out is None:
            out = torch.empty(T, hq, D, dtype=dt, device=dev)
        else:
            _need(out, "out", dev, dt, 3)
            if out.shape != query.shape or out.stride(2) != 1:
                raise ValueError(f"out must be {tuple(query.shape)} with contiguous heads")
        qs, os_, q_ptr, o_ptr = query.stride(), out.stride(), query.data_ptr(), out.data_ptr()
    pos_ptr = table_ptr = None
    pos64 = limit = 0
    if cos_sin is not None:
        _need(cos_sin, "cos_sin", dev, torch.float32, 2)
        if cos_sin.shape[1] != D or not cos_sin.is_contiguous():
            raise ValueError(f"cos_sin must be a contiguous [positions, {D}], got {tuple(cos_sin.shape)}")
        pos64 = _index(positions, "positions", dev, T)
        pos_ptr, table_ptr, limit = positions.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0]
    weights = []
    for name, w in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
        if w is not None:
            _need(w, name, dev, dt, 1)
            if w.shape[0] != D or w.stride(0) != 1:
                raise ValueError(f"{name} must be a contiguous [{D}]")
        weights.append(None if w is None else w.data_ptr())
    args = StoreKvArgs(q_ptr, key.data_ptr(), value.data_ptr(), o_ptr, k_cache.data_ptr(), v_cache.data_ptr(), pos_ptr, slot_mapping.data_ptr(),
                       table_ptr, weights[0], weights[1], _status_ptr(status, dev),
                       qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], cs[0], cs[1], cs[2],
                       T, hq, hk, D, blocks, page, limit, tag, pos64, slots64, eps, 0)
    with _on(dev):
        check(None, _lib.load().b200moe_store_kv(byref(args), _stream(dev)))
    return out


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                  status: Optional[torch.Tensor] = None) -> None:
    """key, value [T, kv_heads, D] -> rows slot_mapping[t] of the caches; slot -1 stores nothing (the reference's function of
    this name, demo/src/layers/attention.py:56-79).  The slots of one call are distinct."""
    _store(None, key, value, None, None, k_cache, v_cache, slot_mapping, None, None, 0.0, None, status)


def rope_store_kvcache(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                       k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, *, q_norm_weight: Optional[torch.Tensor] = None,
                       k_norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, out: Optional[torch.Tensor] = None,
                       status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What the reference's attention layer does between the projection and the attention, in one launch: per-head RMS norm
    of queries and keys (where weights are given), rotary embedding at `positions`, keys and values into the cache.

    query [T, heads, D], key and value [T, kv_heads, D] may be views of one projection row; cos_sin is rotary_table's.
    Returns the rotated queries [T, heads, D] (`out` when given, which may be `query` itself).  fp32 inside, each
    output rounded once."""
    if query is None or cos_sin is None or positions is None:
        raise ValueError("rope_store_kvcache needs query, positions and cos_sin (store_kvcache stores keys and values alone)")
    return _store(query, key, value, positions, cos_sin, k_cache, v_cache, slot_mapping, q_norm_weight, k_norm_weight, eps, out, status)


def paged_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor, *,
                    query_start: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False,
                    status: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of new tokens over their sequences' cached keys and values (theirs included), causal within a span.

    query [T, heads, D]; block_tables int32 [B, max_blocks]; context_lens int32 [B].  Without query_start there is one token
    per sequence (T == B, the draft step); with it (int32 [B+1]) sequence b owns rows query_start[b]:query_start[b+1] and
    its last row sees all context_lens[b] keys (the verify step).  max_query_len, the longest span, picks the row tile; any
    value gives right results.  scale defaults to D ** -0.5.

    Returns out [T, heads, D] (with return_lse also the fp32 log-sum-exp [T, heads]).  A row that sees no key gives zeros
    and -inf; rows behind query_start[B] are not written (nor initialised unless `out` was given)."""
    dev, dt = query.device, query.dtype
    tag = dtype_tag(dt)
    _need(query, "query", dev, dt, 3)
    T, hq, D = query.shape
    blocks, page = _cache(k_cache, v_cache, dev, dt, None, D)
    hk = k_cache.shape[2]
    _need(block_tables, "block_tables", dev, torch.int32, 2)
    _need(context_lens, "context_lens", dev, torch.int32, 1)
    B, width = block_tables.shape
    if context_lens.shape[0] != B or (B > 1 and context_lens.stride(0) != 1) or (width > 1 and block_tables.stride(1) != 1):
        raise ValueError("block_tables [B, max_blocks] and context_lens [B] must be contiguous along their last dimension and agree in B")
    if query.stride(2) != 1:
        raise ValueError("heads must be contiguous")
    start_ptr, span = None, 1
    if query_start is not None:
        _need(query_start, "query_start", dev, torch.int32, 1)
        if query_start.shape[0] != B + 1 or query_start.stride(0) != 1:
            raise ValueError(f"query_start must be a contiguous [{B + 1}]")
        start_ptr = query_start.data_ptr()
        span = T if max_query_len is None else int(max_query_len)
        if span < 0:
            raise ValueError("max_query_len must not be negative")
    elif T != B:
        raise ValueError(f"without query_start there is one token per sequence, got {T} tokens for {B} sequences")
    if out is None:
        out = torch.empty(T, hq, D, dtype=dt, device=dev)
    else:
        _need(out, "out", dev, dt, 3)
        if out.shape != query.shape or out.stride(2) != 1:
            raise ValueError(f"out must be {tuple(query.shape)} with contiguous heads")
    lse = torch.empty(T, hq, dtype=torch.float32, device=dev) if return_lse else None
    lib = _lib.load()
    with _on(dev):
        # the workspace belongs to this call: calls on several streams and captured graphs do not share one
        key = (tag, hq, hk, D, span, width * page, dev.index)
        need = _WORKSPACE.get(key)
        if need is None:
            n = c_int64(0)
            check(None, lib.b200moe_paged_attention_workspace(tag, hq, hk, D, span, width * page, byref(n)))
            if len(_WORKSPACE) > 4096:
                _WORKSPACE.clear()
            need = _WORKSPACE[key] = n.value
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        qs, os_, cs = query.stride(), out.stride(), k_cache.stride()
        args = PagedAttentionArgs(query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(),
                                  start_ptr, out.data_ptr(), None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(),
                                  _status_ptr(status, dev), need, qs[0], qs[1], os_[0], os_[1], cs[0], cs[1], cs[2], block_tables.stride(0),
                                  T, B, hq, hk, D, blocks, page, width, span, tag, D ** -0.5 if scale is None else scale, 0)
        check(None, lib.b200moe_paged_attention(byref(args), _stream(dev)))
    return (out, lse) if return_lse else out
