"""RMS norm of query and key heads with the position rotation, and the paged K/V write (one HIP launch).

For target and draft models whose attention norms each query and key head
before the rotation.  The reference leaves this to its platform's kernels
(the rotation it writes itself, of gathered keys, is
diffspec/compact_kv.py:68-101).  One pass reads the heads of the fused
projection and writes the rotated queries, the rotated keys (to a tensor, to
the pages that ``prefix_attention`` reads, or both) and, for a draft's raw
cache (``capture.capture_raw_kv_rows``), the normed keys before rotation.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["qk_norm_rope"]

STATUS_BAD_POSITION = 1
STATUS_BAD_SLOT = 2


def _heads(t: torch.Tensor, tokens: int, heads: int | None, head_dim: int | None, name: str) -> None:
    if t.ndim != 3 or t.shape[0] != tokens or (heads is not None and t.shape[1:] != (heads, head_dim)):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] like the tensor it belongs to")
    if t.stride(2) != 1:
        raise ValueError(f"{name} must be contiguous in head_dim")


def qk_norm_rope(
    query: torch.Tensor,
    key: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    *,
    eps: float,
    rotary_dim: int,
    is_neox_style: bool,
    query_out: torch.Tensor | None = None,
    key_out: torch.Tensor | None = None,
    normed_key: torch.Tensor | None = None,
    value: torch.Tensor | None = None,
    key_cache: torch.Tensor | None = None,
    value_cache: torch.Tensor | None = None,
    slot_mapping: torch.Tensor | None = None,
    status: torch.Tensor | None = None,
    reuse: dict | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Norm, rotate and store the heads of ``tokens`` new tokens.

    ``query`` ``[tokens, Hq, D]`` and ``key`` ``[tokens, Hkv, D]`` (views of a
    fused projection are fine), weights ``[D]``, ``positions`` int32 or int64
    ``[tokens]``, ``cos_sin_cache`` ``[positions, >= rotary_dim]`` (cosines,
    then sines), in the heads' type or fp32 like the weights.  A ``rotary_dim``
    of 0 is the norm alone: the table is not read, whatever the positions.

    ``query_out`` is written (None: ``query`` itself, in place), and
    ``key_out`` (None: ``key`` itself when there is no paged cache, else the
    rotated keys go to the pages alone).  ``normed_key`` ``[tokens, Hkv, D]``
    gets the keys before rotation.  ``key_cache`` / ``value_cache``
    ``[blocks, block_size, Hkv, D]`` with ``slot_mapping`` (int32 or int64
    ``[tokens]``: page * block_size + place, distinct, negative for graph
    padding) and ``value`` ``[tokens, Hkv, D]`` get the rotated keys and the
    values.  ``status`` (an int32 device word the caller clears) receives
    ``STATUS_BAD_POSITION`` and ``STATUS_BAD_SLOT``; such a token, or its
    pages, are not written.  ``reuse`` (a dict the caller keeps) holds the
    validated descriptor of each layout; every address is taken from the
    call.  Returns the queries' and the keys' output (None where the pages
    alone got the keys).
    """
    if query_out is None:
        query_out = query
    if key_out is None and key_cache is None:
        key_out = key
    tensors = (query, key, q_weight, k_weight, positions, cos_sin_cache, query_out, key_out, normed_key, value,
               key_cache, value_cache, slot_mapping, status)
    layout = None
    if reuse is not None:
        layout = (*[None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors], eps,
                  rotary_dim, is_neox_style)
        hit = reuse.get(layout)
        if hit is not None:
            return _launch(hit[0], hit[1], tensors)
    if query.ndim != 3 or key.ndim != 3:
        raise ValueError("query and key must be [tokens, heads, head_dim]")
    tokens, hq, head_dim = query.shape
    hkv = key.shape[1]
    _heads(query, tokens, None, None, "query")
    _heads(key, tokens, hkv, head_dim, "key")
    _heads(query_out, tokens, hq, head_dim, "query_out")
    for name, t in (("key_out", key_out), ("normed_key", normed_key), ("value", value)):
        if t is not None:
            _heads(t, tokens, hkv, head_dim, name)
    paged = (value, key_cache, value_cache, slot_mapping)
    if any(t is not None for t in paged) and any(t is None for t in paged):
        raise ValueError("the paged write needs value, key_cache, value_cache and slot_mapping together")
    for t in (query, key, query_out, key_out, normed_key, value, key_cache, value_cache):
        if t is not None and t.dtype != query.dtype:
            raise ValueError("queries, keys, values and caches must share a dtype")
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t.shape != (head_dim,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [head_dim] tensor")
    if q_weight.dtype != k_weight.dtype or q_weight.dtype not in (query.dtype, torch.float32):
        raise ValueError("weights must both use the heads' dtype or both fp32")
    if cos_sin_cache.dtype not in (query.dtype, torch.float32):
        raise ValueError("cos/sin cache must use the heads' dtype or fp32")
    if rotary_dim < 0 or rotary_dim > head_dim or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and between zero and head_dim")
    if cos_sin_cache.ndim != 2 or cos_sin_cache.shape[1] < rotary_dim or cos_sin_cache.stride(1) != 1:
        raise ValueError("cos/sin cache must be [positions, >= rotary_dim] with unit last stride")
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32 or int64 [tokens] tensor")
    desc = _lib.QkNormRopeDesc()
    if key_cache is not None:
        if key_cache.ndim != 4 or key_cache.shape[2:] != (hkv, head_dim) or value_cache.shape != key_cache.shape:
            raise ValueError("key and value caches must both be [blocks, block_size, kv_heads, head_dim]")
        if key_cache.stride(3) != 1 or value_cache.stride(3) != 1:
            raise ValueError("key and value caches must be contiguous in head_dim")
        if slot_mapping.dtype not in (torch.int32, torch.int64) or slot_mapping.shape != (tokens,) or \
                not slot_mapping.is_contiguous():
            raise ValueError("slot_mapping must be a contiguous int32 or int64 [tokens] tensor")
        desc.kc_block_stride, desc.kc_token_stride, desc.kc_head_stride = key_cache.stride()[:3]
        desc.vc_block_stride, desc.vc_token_stride, desc.vc_head_stride = value_cache.stride()[:3]
        desc.num_blocks, desc.block_size = key_cache.shape[:2]
        desc.slots_int64 = 1 if slot_mapping.dtype == torch.int64 else 0
        desc.v_row_stride, desc.v_head_stride = value.stride(0), value.stride(1)
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 device word")
    device = _lib.require_gpu(*tensors)
    desc.dtype, desc.weight_dtype = _lib.dtype_code(query.dtype), _lib.dtype_code(q_weight.dtype)
    desc.cos_sin_dtype = _lib.dtype_code(cos_sin_cache.dtype)
    desc.q_row_stride, desc.q_head_stride = query.stride(0), query.stride(1)
    desc.k_row_stride, desc.k_head_stride = key.stride(0), key.stride(1)
    desc.qo_row_stride, desc.qo_head_stride = query_out.stride(0), query_out.stride(1)
    if key_out is not None:
        desc.ko_row_stride, desc.ko_head_stride = key_out.stride(0), key_out.stride(1)
    if normed_key is not None:
        desc.nk_row_stride, desc.nk_head_stride = normed_key.stride(0), normed_key.stride(1)
    desc.positions_int64 = 1 if positions.dtype == torch.int64 else 0
    desc.cs_stride, desc.cs_rows = cos_sin_cache.stride(0), cos_sin_cache.shape[0]
    desc.tokens, desc.num_q_heads, desc.num_kv_heads, desc.head_dim = tokens, hq, hkv, head_dim
    desc.rotary_dim, desc.is_neox_style, desc.eps = rotary_dim, 1 if is_neox_style else 0, float(eps)
    out = _launch(desc, device, tensors)
    if layout is not None:
        if len(reuse) >= 64:
            reuse.clear()
        reuse[layout] = (desc, device)
    return out


def _launch(desc, device, tensors):
    # Addresses go into a copy: another thread may be launching from the kept descriptor.
    desc = _lib.QkNormRopeDesc.from_buffer_copy(desc)
    (desc.query, desc.key, desc.q_weight, desc.k_weight, desc.positions, desc.cos_sin, desc.query_out, desc.key_out,
     desc.normed_key, desc.value, desc.key_cache, desc.value_cache, desc.slot_mapping, desc.status) = map(_lib.ptr,
                                                                                                         tensors)
    with _lib.on_device(device):
        _lib.check(_lib.load().ds_qk_norm_rope(_lib.stream_handle(device), ctypes.byref(desc)))
    return tensors[6], tensors[7]
