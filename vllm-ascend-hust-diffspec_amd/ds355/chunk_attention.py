"""Attention of a chunk of new tokens over a paged cache (three HIP launches).

The reference leaves the target model's attention to its platform and
captures query, softmax LSE and paged keys from it
(diffspec/ascend_patch.py:191-240, diffspec/runtime.py:841-878).  This is that
attention for prompts that enter in chunks: ragged rows of many query tokens,
each causal at its end and over a sliding window where the layer has one,
with rows that decode a single token beside them.  For a verified batch that
shares a long prefix there is ``prefix_attention``, which is also the faster
one for steps of single tokens only.  The LSE it writes is
what ``step.VerifierSnapshot``, ``kernels.paged_chunk_attention_scores`` and
``eviction.attention_mass`` take.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["chunk_workspace_bytes", "new_chunk_workspace", "chunk_attention"]

STATUS_BAD_ROW = 1
STATUS_LENGTH = 2
STATUS_BAD_PAGE = 4


def chunk_workspace_bytes(batch_rows: int, tokens: int, num_q_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """Bytes of the workspace on the current device for up to ``batch_rows`` rows and ``tokens`` query tokens."""
    return int(_lib.load().ds_chunk_attention_workspace_bytes(batch_rows, tokens, num_q_heads, num_kv_heads, head_dim))


def new_chunk_workspace(batch_rows: int, tokens: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                        device: torch.device | str) -> torch.Tensor:
    """A workspace (uint8); it keeps nothing between calls, and serves one launch at a time."""
    with _lib.on_device(torch.device(device)):
        size = chunk_workspace_bytes(batch_rows, tokens, num_q_heads, num_kv_heads, head_dim)
    if size <= 0:
        raise ValueError("workspace sizes must be positive, num_q_heads a multiple of num_kv_heads and head_dim "
                         "64, 128 or 256")
    return torch.empty(size, dtype=torch.uint8, device=device)


def chunk_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    output: torch.Tensor,
    lse: torch.Tensor | None,
    block_table: torch.Tensor,
    query_start: torch.Tensor,
    query_len: torch.Tensor,
    target_len: torch.Tensor,
    *,
    scale: float,
    workspace: torch.Tensor,
    window: int | None = None,
    batch_size: int | None = None,
    status: torch.Tensor | None = None,
    reuse: dict | None = None,
) -> torch.Tensor:
    """Attention of ragged query rows over paged keys and values, causal at each row's end.

    ``query`` / ``output`` ``[tokens, Hq, D]`` (bf16 or fp16, rows contiguous
    in D), ``key_cache`` / ``value_cache`` ``[blocks, block_size, Hkv, D]``,
    ``block_table`` int32 ``[rows, *]``; ``query_start`` / ``query_len`` /
    ``target_len`` int32 ``[rows]`` as in ``step.VerifierRows``: row b's
    query tokens are the last ``query_len[b]`` of its ``target_len[b]``
    tokens.  ``lse`` fp32 ``[tokens, Hq]`` (any strides) or None.
    ``window``: each query token sees itself and the ``window - 1`` keys
    before it (None: all).  A query token that sees no key gets a zero
    output and an LSE of -infinity; output and LSE rows of tokens that no
    row has (graph padding) are left as they were.  ``output`` may be
    ``query`` itself.  Rows at or beyond
    ``batch_size`` are padding.  Rows must not share query tokens.

    ``status`` (an int32 device word the caller clears) receives
    ``STATUS_BAD_ROW``, ``STATUS_LENGTH`` and ``STATUS_BAD_PAGE``
    (include/ds355.h).  ``reuse`` (a dict the caller keeps) holds the
    validated descriptor of each layout (shapes, strides, types, devices): a
    later call of the same layout skips the checks; every address is taken
    from the call.  Returns ``output``.
    """
    key = None
    if reuse is not None:
        tensors = (query, key_cache, value_cache, output, lse, block_table, query_start, query_len, target_len,
                   workspace, status)
        key = (*[None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors], window, batch_size)
        hit = reuse.get(key)
        if hit is not None:
            return _launch(hit[0], hit[1], query, key_cache, value_cache, output, lse, block_table, query_start,
                           query_len, target_len, scale, workspace, status)
    if query.ndim != 3 or output.shape != query.shape:
        raise ValueError("query and output must both be [tokens, query_heads, head_dim]")
    if key_cache.ndim != 4 or value_cache.shape != key_cache.shape:
        raise ValueError("key and value caches must both be [blocks, block_size, kv_heads, head_dim]")
    tokens, hq, head_dim = query.shape
    blocks, block_size, hkv, key_dim = key_cache.shape
    if key_dim != head_dim:
        raise ValueError("query and key head dimensions must match")
    if hkv == 0 or hq % hkv != 0:
        raise ValueError("query heads must be divisible by KV heads")
    for name, t in (("query", query), ("output", output), ("key cache", key_cache), ("value cache", value_cache)):
        if t.dtype != query.dtype:
            raise ValueError("query, output and KV caches must share a dtype")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous in head_dim")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (tokens, hq)):
        raise ValueError("lse must be fp32 [tokens, query_heads]")
    if window is not None and window < 1:
        raise ValueError("window must be positive, or None")
    rows = query_len.numel()
    for name, t in (("query_start", query_start), ("query_len", query_len), ("target_len", target_len)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor")
    if query_start.numel() != rows or target_len.numel() != rows:
        raise ValueError("query_start, query_len and target_len need one entry per row")
    if batch_size is not None:
        if not 0 <= batch_size <= rows:
            raise ValueError("batch_size must be between zero and the number of rows")
        rows = batch_size
    if block_table.dtype != torch.int32 or block_table.ndim != 2 or block_table.stride(1) != 1 or \
            block_table.shape[0] < rows:
        raise ValueError("block_table must be int32 [rows, blocks] with unit last stride")
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor (see new_chunk_workspace)")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 device word")
    device = _lib.require_gpu(query, key_cache, value_cache, output, lse, block_table, query_start, query_len,
                              target_len, workspace, status)
    desc = _lib.ChunkAttentionDesc()
    desc.dtype = _lib.dtype_code(query.dtype)
    desc.q_row_stride, desc.q_head_stride = query.stride(0), query.stride(1)
    desc.o_row_stride, desc.o_head_stride = output.stride(0), output.stride(1)
    if lse is not None:
        desc.lse_token_stride, desc.lse_head_stride = lse.stride(0), lse.stride(1)
    desc.k_block_stride, desc.k_token_stride, desc.k_head_stride = key_cache.stride()[:3]
    desc.v_block_stride, desc.v_token_stride, desc.v_head_stride = value_cache.stride()[:3]
    desc.bt_stride, desc.max_blocks = block_table.stride(0), _lib.count(block_table.shape[1])
    desc.num_blocks, desc.block_size = _lib.count(blocks), _lib.count(block_size)
    desc.rows, desc.tokens = _lib.count(rows), _lib.count(tokens)
    desc.num_q_heads, desc.num_kv_heads, desc.head_dim = (_lib.count(n) for n in (hq, hkv, head_dim))
    desc.window = 0 if window is None else min(int(window), 1 << 30)
    desc.workspace_bytes = workspace.numel()
    _launch(desc, device, query, key_cache, value_cache, output, lse, block_table, query_start, query_len, target_len,
            scale, workspace, status)
    if key is not None:
        if len(reuse) >= 64:
            reuse.clear()
        reuse[key] = (desc, device)
    return output


def _launch(desc, device, query, key_cache, value_cache, output, lse, block_table, query_start, query_len, target_len,
            scale, workspace, status):
    # Addresses go into a copy: another thread may be launching from the kept descriptor.
    desc = _lib.ChunkAttentionDesc.from_buffer_copy(desc)
    desc.query, desc.output, desc.lse = query.data_ptr(), output.data_ptr(), _lib.ptr(lse)
    desc.key_cache, desc.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    desc.block_table, desc.query_start = block_table.data_ptr(), query_start.data_ptr()
    desc.query_len, desc.target_len = query_len.data_ptr(), target_len.data_ptr()
    desc.workspace, desc.status = workspace.data_ptr(), _lib.ptr(status)
    desc.scale = float(scale)
    with _lib.on_device(device):
        _lib.check(_lib.load().ds_chunk_attention(_lib.stream_handle(device), ctypes.byref(desc)))
    return output
