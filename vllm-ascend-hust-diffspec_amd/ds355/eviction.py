"""A bounded target cache: the attention weight that cached keys receive, and eviction by it.

The reference bounds the context of the draft model (diffspec/runtime.py:1650-1681)
and leaves the target's cache to the serving engine.  ``attention_mass`` adds
up, from the LSE that ``chunk_attention`` or ``prefix_attention`` wrote, how
much weight each cached key got, and ``evict_tokens`` keeps the heaviest keys
of each KV head, in place.  The pages behind the kept slots go back with
``pages.PagePool.free``, and the attention of the next step reads the shorter
rows like any others.  Drafting by retrieval (``step.retrieval_step``) takes
slots for tokens: rows that draft so must be kept out of the eviction.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["mass_workspace_bytes", "new_mass_workspace", "attention_mass", "evict_workspace_bytes",
           "new_evict_workspace", "evict_tokens"]

STATUS_BAD_ROW = 1
STATUS_LENGTH = 2
STATUS_BAD_PAGE = 4
STATUS_BUDGET = 8
STATUS_SHARED_PAGE = 16


def mass_workspace_bytes() -> int:
    """Bytes of the workspace of ``attention_mass`` on the current device, whatever the sizes."""
    return int(_lib.load().ds_attention_mass_workspace_bytes())


def new_mass_workspace(device: torch.device | str) -> torch.Tensor:
    """A workspace (uint8) for ``attention_mass``; it keeps nothing between calls, and serves one launch at a time."""
    with _lib.on_device(torch.device(device)):
        return torch.empty(mass_workspace_bytes(), dtype=torch.uint8, device=device)


def evict_workspace_bytes(batch_rows: int, num_kv_heads: int, capacity: int) -> int:
    """Bytes of the workspace of ``evict_tokens`` for up to ``batch_rows`` rows of up to ``capacity`` slots."""
    return int(_lib.load().ds_evict_workspace_bytes(batch_rows, num_kv_heads, capacity))


def new_evict_workspace(batch_rows: int, num_kv_heads: int, capacity: int, device: torch.device | str) -> torch.Tensor:
    """A workspace (uint8) for ``evict_tokens``; it keeps nothing between calls, and serves one launch at a time."""
    size = evict_workspace_bytes(batch_rows, num_kv_heads, capacity)
    if size <= 0:
        raise ValueError("workspace sizes must be positive")
    return torch.empty(size, dtype=torch.uint8, device=device)


def _layout(*tensors):
    return [None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors]


def _keep(reuse, key, desc, device):
    if key is not None:
        if len(reuse) >= 64:
            reuse.clear()
        reuse[key] = (desc, device)


def _ints(rows, **tensors):
    for name, t in tensors.items():
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor")
        if t.numel() != rows:
            raise ValueError(f"{name} needs one entry per row")


def _rows(rows, batch_size):
    if batch_size is None:
        return rows
    if not 0 <= batch_size <= rows:
        raise ValueError("batch_size must be between zero and the number of rows")
    return batch_size


def _table(block_table, rows):
    if block_table.dtype != torch.int32 or block_table.ndim != 2 or block_table.stride(1) != 1 or \
            block_table.shape[0] < rows:
        raise ValueError("block_table must be int32 [rows, blocks] with unit last stride")


def _per_slot(t, name, dtype, rows, heads):
    if t.dtype != dtype or t.ndim != 3 or t.shape[0] < rows or t.shape[1] != heads or t.shape[2] < 1 or t.stride(2) != 1:
        kind = "fp32" if dtype == torch.float32 else "int32"
        raise ValueError(f"{name} must be {kind} [rows, kv_heads, capacity] with unit last stride")
    # Rows of heads or heads of rows, as a rule; places of other layouts are looked at one by one.
    (inner, count), (outer, others) = sorted(((t.stride(0), t.shape[0]), (t.stride(1), t.shape[1])))
    if (count == 1 or inner >= t.shape[2]) and (others == 1 or outer >= (count - 1) * inner + t.shape[2]):
        return
    places = sorted(i * inner + j * outer for i in range(count) for j in range(others))
    if any(y - x < t.shape[2] for x, y in zip(places, places[1:])):
        raise ValueError(f"{name}'s rows and heads overlap")


def _words(workspace, status, new):
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor (see {new})")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 device word")


def attention_mass(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    lse: torch.Tensor,
    mass: torch.Tensor,
    block_table: torch.Tensor,
    query_start: torch.Tensor,
    query_len: torch.Tensor,
    target_len: torch.Tensor,
    *,
    scale: float,
    workspace: torch.Tensor,
    previous: torch.Tensor | None = None,
    decay: float = 1.0,
    window: int | None = None,
    batch_size: int | None = None,
    status: torch.Tensor | None = None,
    reuse: dict | None = None,
) -> torch.Tensor:
    """The weight that each cached key of a row receives from the row's query tokens.

    ``mass[b, h, t] = decay * previous[b, h, t] + sum exp(scale * q . k_t - lse)``
    over row b's query tokens that see key t (as in ``chunk_attention``,
    whose rows, table, ``window`` and ``lse`` these are) and the query heads
    of KV head h, for t < ``target_len[b]``.  ``mass`` and ``previous`` are
    fp32 ``[rows, Hkv, capacity]``; ``previous`` may be ``mass`` itself (it
    is then added to in place), memory apart from it, or None for zeros.  Entries at or past a
    row's length, and rows without query tokens, are left as they were.
    Rows may name only the last tokens of each request, or only the accepted
    ones of a verified draft: ``query_len`` their number and ``target_len``
    the accepted length.  Rejected tokens then add nothing, and their slots
    hold no mass that the next tokens there would inherit.

    ``status`` receives ``STATUS_BAD_ROW``, ``STATUS_LENGTH`` and
    ``STATUS_BAD_PAGE`` (include/ds355.h); ``reuse`` as in
    ``chunk_attention``.  Returns ``mass``.
    """
    key = None
    if reuse is not None:
        key = (*_layout(query, key_cache, lse, mass, block_table, query_start, query_len, target_len, previous, workspace,
                        status), window, batch_size)
        hit = reuse.get(key)
        if hit is not None:
            return _launch_mass(hit[0], hit[1], query, key_cache, lse, mass, block_table, query_start, query_len,
                                target_len, scale, workspace, previous, decay, status)
    if query.ndim != 3 or key_cache.ndim != 4:
        raise ValueError("query must be [tokens, query_heads, head_dim] and the key cache [blocks, block_size, kv_heads, "
                         "head_dim]")
    tokens, hq, head_dim = query.shape
    blocks, block_size, hkv, key_dim = key_cache.shape
    if key_dim != head_dim:
        raise ValueError("query and key head dimensions must match")
    if hkv == 0 or hq % hkv != 0:
        raise ValueError("query heads must be divisible by KV heads")
    if key_cache.dtype != query.dtype:
        raise ValueError("query and key cache must share a dtype")
    for name, t in (("query", query), ("key cache", key_cache)):
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous in head_dim")
    if lse.dtype != torch.float32 or lse.shape != (tokens, hq):
        raise ValueError("lse must be fp32 [tokens, query_heads]")
    if window is not None and window < 1:
        raise ValueError("window must be positive, or None")
    rows = query_len.numel()
    _ints(rows, query_len=query_len, query_start=query_start, target_len=target_len)
    rows = _rows(rows, batch_size)
    _table(block_table, rows)
    _per_slot(mass, "mass", torch.float32, rows, hkv)
    if previous is not None:
        _per_slot(previous, "previous", torch.float32, rows, hkv)
        if previous.shape[2] != mass.shape[2]:
            raise ValueError("previous must have mass's capacity")
    _words(workspace, status, "new_mass_workspace")
    device = _lib.require_gpu(query, key_cache, lse, mass, block_table, query_start, query_len, target_len, previous,
                              workspace, status)
    desc = _lib.AttentionMassDesc()
    desc.dtype = _lib.dtype_code(query.dtype)
    desc.q_row_stride, desc.q_head_stride = query.stride(0), query.stride(1)
    desc.k_block_stride, desc.k_token_stride, desc.k_head_stride = key_cache.stride()[:3]
    desc.lse_token_stride, desc.lse_head_stride = lse.stride(0), lse.stride(1)
    if previous is not None:
        desc.previous_row_stride, desc.previous_head_stride = previous.stride(0), previous.stride(1)
    desc.mass_row_stride, desc.mass_head_stride, desc.capacity = mass.stride(0), mass.stride(1), _lib.count(mass.shape[2])
    desc.bt_stride, desc.max_blocks = block_table.stride(0), _lib.count(block_table.shape[1])
    desc.num_blocks, desc.block_size = _lib.count(blocks), _lib.count(block_size)
    desc.rows, desc.tokens = _lib.count(rows), _lib.count(tokens)
    desc.num_q_heads, desc.num_kv_heads, desc.head_dim = (_lib.count(n) for n in (hq, hkv, head_dim))
    desc.window = 0 if window is None else min(int(window), 1 << 30)
    desc.workspace_bytes = workspace.numel()
    _launch_mass(desc, device, query, key_cache, lse, mass, block_table, query_start, query_len, target_len, scale,
                 workspace, previous, decay, status)
    _keep(reuse, key, desc, device)
    return mass


def _launch_mass(desc, device, query, key_cache, lse, mass, block_table, query_start, query_len, target_len, scale,
                 workspace, previous, decay, status):
    # Addresses go into a copy: another thread may be launching from the kept descriptor.
    desc = _lib.AttentionMassDesc.from_buffer_copy(desc)
    desc.query, desc.key_cache, desc.lse = query.data_ptr(), key_cache.data_ptr(), lse.data_ptr()
    desc.mass, desc.previous = mass.data_ptr(), _lib.ptr(previous)
    desc.block_table, desc.query_start = block_table.data_ptr(), query_start.data_ptr()
    desc.query_len, desc.target_len = query_len.data_ptr(), target_len.data_ptr()
    desc.workspace, desc.status = workspace.data_ptr(), _lib.ptr(status)
    desc.scale, desc.decay = float(scale), float(decay)
    with _lib.on_device(device):
        _lib.check(_lib.load().ds_attention_mass(_lib.stream_handle(device), ctypes.byref(desc)))
    return mass


def evict_tokens(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    mass: torch.Tensor,
    positions: torch.Tensor,
    settled: torch.Tensor,
    block_table: torch.Tensor,
    target_len: torch.Tensor,
    keep_len: torch.Tensor,
    kept_len: torch.Tensor,
    *,
    workspace: torch.Tensor,
    sinks: int = 0,
    recent: int = 0,
    ref_counts: torch.Tensor | None = None,
    batch_size: int | None = None,
    status: torch.Tensor | None = None,
    reuse: dict | None = None,
) -> torch.Tensor:
    """Cuts each row of ``target_len[b]`` slots to its ``keep_len[b]`` best, head by head, in place.

    A KV head keeps the request's first ``sinks`` tokens and its newest
    ``recent`` ones, then the slots of largest ``mass`` (ties to the lowest
    slot, NaN below all numbers).  Kept slots below ``keep_len[b]`` stay; the
    others move, in order, to the slots that are given up there, with their
    keys, values, mass and positions.  ``kept_len`` (int32 ``[rows]``, apart
    from the other lengths) gets each row's new length.

    ``key_cache`` / ``value_cache`` ``[blocks, block_size, Hkv, D]`` (bf16,
    fp16 or fp32); ``mass`` fp32 and ``positions`` int32 ``[rows, Hkv,
    capacity]``; ``settled`` int32 ``[rows, 2]``: the slots whose
    ``positions`` are written, and the tokens evicted so far.  A new request
    starts with zeros in ``settled`` and ``mass``, and needs no positions;
    its tokens are appended behind its last slot.  A row is not cut back
    below its settled slots.  Layers have caches, mass, positions and settled
    of their own and share lengths and tables.

    Rows that cannot be cut are left as they are, with a bit of ``status``:
    ``STATUS_LENGTH`` (longer than the table or ``capacity``),
    ``STATUS_BAD_PAGE``, ``STATUS_BUDGET`` (``keep_len`` negative or below
    ``sinks + recent``) and, where ``ref_counts`` (a ``PagePool``'s) is
    given, ``STATUS_SHARED_PAGE`` (a page of the kept slots has other rows).
    ``reuse`` as in ``chunk_attention``.  Returns ``kept_len``.
    """
    key = None
    if reuse is not None:
        key = (*_layout(key_cache, value_cache, mass, positions, settled, block_table, target_len, keep_len, kept_len,
                        workspace, ref_counts, status), sinks, recent, batch_size)
        hit = reuse.get(key)
        if hit is not None:
            return _launch_evict(hit[0], hit[1], key_cache, value_cache, mass, positions, settled, block_table,
                                 target_len, keep_len, kept_len, workspace, ref_counts, status)
    if key_cache.ndim != 4 or value_cache.shape != key_cache.shape:
        raise ValueError("key and value caches must both be [blocks, block_size, kv_heads, head_dim]")
    if value_cache.dtype != key_cache.dtype:
        raise ValueError("key and value caches must share a dtype")
    for name, t in (("key cache", key_cache), ("value cache", value_cache)):
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous in head_dim")
    if sinks < 0 or recent < 0:
        raise ValueError("sinks and recent must not be negative")
    blocks, block_size, hkv, head_dim = key_cache.shape
    rows = target_len.numel()
    _ints(rows, target_len=target_len, keep_len=keep_len, kept_len=kept_len)
    if settled.dtype != torch.int32 or settled.shape != (rows, 2) or not settled.is_contiguous():
        raise ValueError("settled must be a contiguous int32 [rows, 2] tensor")
    rows = _rows(rows, batch_size)
    _table(block_table, rows)
    _per_slot(mass, "mass", torch.float32, rows, hkv)
    _per_slot(positions, "positions", torch.int32, rows, hkv)
    if positions.shape[2] != mass.shape[2]:
        raise ValueError("positions must have mass's capacity")
    if ref_counts is not None and (ref_counts.dtype != torch.int32 or ref_counts.shape != (blocks,)
                                   or not ref_counts.is_contiguous()):
        raise ValueError("ref_counts must be a contiguous int32 [num_pages] tensor")
    _words(workspace, status, "new_evict_workspace")
    device = _lib.require_gpu(key_cache, value_cache, mass, positions, settled, block_table, target_len, keep_len,
                              kept_len, workspace, ref_counts, status)
    desc = _lib.EvictDesc()
    desc.dtype = _lib.dtype_code(key_cache.dtype)
    desc.k_block_stride, desc.k_token_stride, desc.k_head_stride = key_cache.stride()[:3]
    desc.v_block_stride, desc.v_token_stride, desc.v_head_stride = value_cache.stride()[:3]
    desc.mass_row_stride, desc.mass_head_stride, desc.capacity = mass.stride(0), mass.stride(1), _lib.count(mass.shape[2])
    desc.positions_row_stride, desc.positions_head_stride = positions.stride(0), positions.stride(1)
    desc.bt_stride, desc.max_blocks = block_table.stride(0), _lib.count(block_table.shape[1])
    desc.num_blocks, desc.block_size = _lib.count(blocks), _lib.count(block_size)
    desc.rows, desc.num_kv_heads, desc.head_dim = _lib.count(rows), _lib.count(hkv), _lib.count(head_dim)
    desc.sinks, desc.recent = _lib.count(sinks), _lib.count(recent)
    desc.workspace_bytes = workspace.numel()
    _launch_evict(desc, device, key_cache, value_cache, mass, positions, settled, block_table, target_len, keep_len,
                  kept_len, workspace, ref_counts, status)
    _keep(reuse, key, desc, device)
    return kept_len


def _launch_evict(desc, device, key_cache, value_cache, mass, positions, settled, block_table, target_len, keep_len,
                  kept_len, workspace, ref_counts, status):
    desc = _lib.EvictDesc.from_buffer_copy(desc)
    desc.key_cache, desc.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    desc.mass, desc.positions, desc.settled = mass.data_ptr(), positions.data_ptr(), settled.data_ptr()
    desc.block_table, desc.ref_counts = block_table.data_ptr(), _lib.ptr(ref_counts)
    desc.target_len, desc.keep_len, desc.kept_len = target_len.data_ptr(), keep_len.data_ptr(), kept_len.data_ptr()
    desc.workspace, desc.status = workspace.data_ptr(), _lib.ptr(status)
    with _lib.on_device(device):
        _lib.check(_lib.load().ds_evict(_lib.stream_handle(device), ctypes.byref(desc)))
    return kept_len
