"""Launches over a paged cache relation (``Graph.paged``): attention, the
upkeep of the cache, reading it back and the choice of pages
(csrc/tgx_paged.hip, csrc/tgx_paged_scaled.hip, csrc/tgx_pages.hip,
csrc/tgx_pages_scaled.hip), and the same on Torch operations for host tensors.

The page tables and lengths are read by the kernels at every launch, so none
of these copies them to the host or synchronises; outputs and workspaces are
allocated by Torch on the current stream of the operands' device.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native
from ._dual import carries_tangent
from .blockscaled import CODES, BlockScaled, encode, scale_of

# Element types of the paged kernels (TGX_DTYPE_*).
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def rows_on_16_bytes(t: torch.Tensor) -> bool:
    """Every row of `t` (its last dimension, dense) starts a multiple of 16
    bytes from the tensor's start."""
    vec, shape, strides = 16 // t.element_size(), t.shape, t.stride()
    if shape[-1] > 1 and strides[-1] != 1:
        return False
    for n, s in zip(shape[:-1], strides):
        if n > 1 and s % vec:
            return False
    return True


def _on_16_bytes(t: torch.Tensor) -> torch.Tensor:
    if not rows_on_16_bytes(t):
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def heads_of(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
    """(key heads, query heads on each) of attention fields of matching
    shapes, else None: q [n, heads, group, D] on k [m, heads, 1, D], or
    q [n, heads, D] on k [m, heads, D], or q [n, group, D] on k [m, 1, D]."""
    if k.shape != v.shape or q.ndim != k.ndim or q.ndim not in (3, 4) or \
            q.shape[-1] != k.shape[-1]:
        return None
    if q.ndim == 4:
        if k.shape[1] != q.shape[1] or k.shape[2] != 1:
            return None
        return q.shape[1], q.shape[2]
    if k.shape[1] == q.shape[1]:
        return q.shape[1], 1
    return (1, q.shape[1]) if k.shape[1] == 1 else None


def wants_derivative(q, k, v) -> bool:
    """Whether attention of these has to carry gradients or a tangent."""
    return ((q.requires_grad or k.requires_grad or v.requires_grad) and
            torch.is_grad_enabled()) or carries_tangent(q, _carrier(k), _carrier(v))


def _carrier(t) -> torch.Tensor:
    """The tensor of a field that could carry a tangent."""
    return t.scales if isinstance(t, BlockScaled) else t


def cache_kind(k, v):
    """(code, block) of key and value fields, (0, 1) of tensors; None where
    one is in 8 bits and the other is not, or in another form."""
    if not isinstance(k, BlockScaled) and not isinstance(v, BlockScaled):
        return 0, 1
    if not isinstance(k, BlockScaled) or not isinstance(v, BlockScaled) or \
            (k.dtype, k.block, k.tables) != (v.dtype, v.block, v.tables):
        return None
    return CODES[k.dtype], k.block


def cache_rows_ok(k, v) -> bool:
    """Whether a launch can read these key and value fields in place."""
    if isinstance(k, BlockScaled):
        # (Codes are read by eights, or sixteens where the rows allow it.)
        return k.eights and v.eights and (k.codes.data_ptr() | v.codes.data_ptr()) % 8 == 0
    return rows_on_16_bytes(k) and rows_on_16_bytes(v)


def tiles_take(q, k, v) -> bool:
    """Whether the matrix tiles take a launch, as csrc/tgx_paged.hip chooses them; the
    rows kernel takes every other."""
    if q.dtype == torch.float32 or q.shape[-1] not in (32, 64, 128):
        return False
    # (Codes by sixteens; those that lie on 8 bytes only go to the rows kernel.)
    return not isinstance(k, BlockScaled) or all(
        rows_on_16_bytes(c.codes) and c.codes.data_ptr() % 16 == 0 for c in (k, v))


def csr_takes(D: int) -> bool:
    """Whether the CSR attention kernels take heads of this width."""
    return D % 8 == 0 and 8 <= D <= 512 and (D // 8) & (D // 8 - 1) == 0


def _view(state, k=None, v=None):
    """The native tgx_paged_view of a launch, None where tgx_paged_attn covers it."""
    scaled = isinstance(k, BlockScaled)
    if not scaled and state.window is None:
        return None
    return _native.PagedView(
        state.window or 0, state.sinks, CODES[k.dtype] if scaled else 0,
        k.block if scaled else 1, k.scales.data_ptr() or None if scaled else None,
        v.scales.data_ptr() or None if scaled else None)


def attention_workspace(graph, k, v, heads: int, group: int, D: int, code: int) -> int | None:
    """Workspace bytes of an attention launch, None where no launch covers the
    sizes; asked once a relation and shape."""
    state = graph.paged_state
    key = ("attention-workspace", heads, group, D, code, cache_kind(k, v))
    need = state.checked.get(key)
    if need is None:
        bytes_ = ctypes.c_size_t()
        view = _view(state, k, v)
        with torch.cuda.device(graph.device):
            if view is None:
                takes = _native.covered("tgx_paged_attn_workspace", state.native(), heads, group,
                                        D, code, ctypes.byref(bytes_))
            else:
                takes = _native.covered("tgx_paged_attn_view_workspace", state.native(),
                                        ctypes.byref(view), heads, group, D, code,
                                        ctypes.byref(bytes_))
        need = state.checked[key] = bytes_.value if takes else -1
    return None if need < 0 else need


def bind_attention(graph, q, k, v, scale: float, heads: int, group: int):
    """The attention launch with its native arguments bound: a zero-argument
    callable that returns a new output."""
    state = graph.paged_state
    for t in (q, k, v):
        if t.device != graph.device:
            raise ValueError(f"operand on {t.device} for a graph on {graph.device}")
    q, view = _on_16_bytes(q), _view(state, k, v)
    fields = (k, v)
    if isinstance(k, BlockScaled):
        # (Another call's of the same layout may lie elsewhere.)
        k, v = (c.codes if c.codes.data_ptr() % 8 == 0 else c.codes.clone() for c in (k, v))
    else:
        k, v = fields = (_on_16_bytes(k), _on_16_bytes(v))
    tables = state.table_heads
    D = q.shape[-1]
    by_head = lambda t: t.stride(1) if heads > 1 else 0
    # A row of a relation with a table per head is (token, table head).  (The
    # stride of a dimension of one element may be any.)
    by_row = lambda t: t.stride(0) if t.shape[0] > 1 else 0
    strides = (ctypes.c_int64 * 9)(
        by_row(q), by_head(q), q.stride(-2) if group > 1 else 0,
        by_row(k) * tables, by_row(k) if tables > 1 else 0, by_head(k),
        by_row(v) * tables, by_row(v) if tables > 1 else 0, by_head(v))
    code = DTYPES[q.dtype]
    need = attention_workspace(graph, *fields, heads, group, D, code)
    if need is None:
        raise NotImplementedError("paged attention: too many sequences, heads and queries for one "
                                  "launch")
    shape, dtype, device = q.shape, q.dtype, q.device
    tensors = (q.data_ptr(), k.data_ptr() if k.numel() else None,
               v.data_ptr() if v.numel() else None)
    name, relation = "tgx_paged_attn", ()
    if view is not None:
        name, relation = "tgx_paged_attn_view", (ctypes.byref(view),)

    def launch(keep=(q, _carrier(fields[0]), _carrier(fields[1])), rows=(k, v)):
        if carries_tangent(*keep):
            raise NotImplementedError("paged attention has no forward-mode derivative")
        out = torch.empty(shape, dtype=dtype, device=device)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _native.launch(out, name, state.native(), *relation, *tensors, strides, scale,
                       out.data_ptr(), heads, group, D, code,
                       work.data_ptr() if need else None, need)
        return out

    if not q.numel():
        return lambda: torch.empty(shape, dtype=dtype, device=device)

    return launch


# ---------------------------------------------------------------------------
# append

def _on_torch_operations(name: str, t: torch.Tensor) -> bool:
    """Whether operands of t's device and type run on Torch operations, which
    strict mode refuses on the GPU."""
    if not t.is_cuda:
        return True
    if t.dtype in DTYPES:
        return False
    from .message_passing import config

    if config.strict:
        raise RuntimeError(f"{name}: no HIP kernel covers {t.dtype} and tiga.config.strict is set")
    return True


def plan_append(key_cache, key, value_cache, value, page_sums):
    """What append keeps for operands of some types, shapes and strides: for caches
    in 8 bits the native arguments but for addresses, else True."""
    if not isinstance(key_cache, BlockScaled):
        return True
    k, v, (_, heads, D) = key_cache.codes, value_cache.codes, key.shape
    strides = (ctypes.c_int64 * 8)(_step(k, 0), _step(k, 1), _step(key, 0), _step(key, 1),
                                   _step(v, 0), _step(v, 1), _step(value, 0), _step(value, 1))
    return strides, rows_on_16_bytes(key) and rows_on_16_bytes(value), heads, D, \
        DTYPES[key.dtype], CODES[k.dtype], key_cache.block


def append(graph, key_cache, key, value_cache, value, page_sums, plan) -> None:
    state = graph.paged_state
    if plan is not True:
        _append_scaled(state, key_cache, key, value_cache, value, page_sums, plan)
        return
    if _on_torch_operations("append", key_cache):
        _append_torch(state, key_cache, key, value_cache, value, page_sums)
        return
    if carries_tangent(key_cache, key, value_cache, value, page_sums):
        raise NotImplementedError("append has no forward-mode derivative: detach its operands")
    rows, heads, D = key.shape
    if D > 1:
        key = key if key.stride(2) == 1 else key.contiguous()
        value = value if value.stride(2) == 1 else value.contiguous()
    if rows * heads * D == 0 or key_cache.shape[0] == 0:
        return
    strides = (ctypes.c_int64 * 8)(*key_cache.stride()[:2], *key.stride()[:2],
                                   *value_cache.stride()[:2], *value.stride()[:2])
    _native.launch(key_cache, "tgx_paged_append", state.native(), key_cache.data_ptr(),
                   key.data_ptr(), value_cache.data_ptr(), value.data_ptr(), strides,
                   _native.ptr(page_sums), heads, D, DTYPES[key.dtype])
    torch.autograd.graph.increment_version(
        (key_cache, value_cache) if page_sums is None else (key_cache, value_cache, page_sums))


def _append_torch(state, key_cache, key, value_cache, value, page_sums) -> None:
    queries, size = state.queries, state.page_size
    if state.page_table.numel() == 0 or state.num_pages == 0:
        return
    length = state.clamped_lengths()
    position = length[:, None] - queries + torch.arange(queries, device=length.device)
    page = position.clamp(min=0) // size
    ids = state.page_table.long().gather(1, page)
    there = (position >= 0) & (ids >= 0) & (ids < state.num_pages)
    slots = (ids * size + position.clamp(min=0) % size)[there]
    rows = there.reshape(-1)
    key_cache[slots] = key[rows]
    value_cache[slots] = value[rows]
    if page_sums is None:
        return
    first = (length - queries).clamp(min=0) // size
    touched = first[:, None] + torch.arange((queries - 1) // size + 2, device=length.device)
    held = (length[:, None] - touched * size).clamp(min=0, max=size)
    ids = state.page_table.long().gather(1, touched.clamp(max=state.page_table.shape[1] - 1))
    there = (held > 0) & (ids >= 0) & (ids < state.num_pages)
    ids, held = ids[there], held[there]
    rows = key_cache.view(state.num_pages, size, *key_cache.shape[1:])[ids].float()
    inside = torch.arange(size, device=length.device) < held[:, None]
    page_sums[ids] = torch.where(inside[..., None, None], rows, 0.0).sum(1)


# ---------------------------------------------------------------------------
# Caches in 8 bits

def _scaled_on_torch_operations(name: str, width: int, caches) -> bool:
    """Whether caches of this width run on Torch operations, which strict
    mode refuses on the GPU."""
    if not caches[0].codes.is_cuda:
        return True
    if width % 8 == 0 and 0 < width <= 512 and cache_rows_ok(*caches):
        return False
    from .message_passing import config

    if config.strict:
        raise RuntimeError(f"{name}: no HIP kernel covers 8-bit rows of {width} values (multiples "
                           "of 8 up to 512, on 8 bytes) and tiga.config.strict is set")
    return True


def _step(t: torch.Tensor, dim: int) -> int:
    """A stride; 0 for a dimension of one element, whose stride may be any."""
    return t.stride(dim) if t.shape[dim] > 1 else 0


def _append_scaled(state, key_cache, key, value_cache, value, page_sums, plan) -> None:
    if carries_tangent(key, value, page_sums, key_cache.scales, value_cache.scales):
        raise NotImplementedError("append has no forward-mode derivative: detach its operands")
    strides, dense, heads, D, dtype, code, block = plan
    on_torch = _scaled_on_torch_operations("append", D, (key_cache, value_cache))
    k, v = key_cache.codes, value_cache.codes
    if key.numel() and k.numel() and (
            k.data_ptr() == v.data_ptr() or
            key_cache.scales.data_ptr() == value_cache.scales.data_ptr()):
        raise ValueError("key_cache and value_cache must not share their codes or scales: each "
                         "is written by its own rows")
    if on_torch:
        for cache, new in ((key_cache, key), (value_cache, value)):
            _append_scaled_torch(state, cache, new)
        if page_sums is not None:
            _sum_scaled_torch(state, key_cache, page_sums)
        return
    if key.numel() == 0 or k.numel() == 0:
        return
    at = key.data_ptr(), value.data_ptr()
    if not dense or (at[0] | at[1]) % 16:
        key, value = _on_16_bytes(key), _on_16_bytes(value)
        strides = plan_append(key_cache, key, value_cache, value, page_sums)[0]
        at = key.data_ptr(), value.data_ptr()
    _native.launch(key, "tgx_paged_append_scaled", state.native(), k.data_ptr(),
                   key_cache.scales.data_ptr(), at[0], v.data_ptr(),
                   value_cache.scales.data_ptr(), at[1], strides,
                   None if page_sums is None else page_sums.data_ptr(), heads, D, dtype, code,
                   block)
    written = (k, key_cache.scales, v, value_cache.scales)
    torch.autograd.graph.increment_version(
        written if page_sums is None else (*written, page_sums))


def _positions(state, first, count: int, size: int):
    """(slots, named) [sequences, count, size] of the positions of `count` runs of
    `size` from run first[b] of each sequence on; named: cached, on a page that
    exists."""
    at = (first[:, None] + torch.arange(count, device=first.device)) * size
    at = at[..., None] + torch.arange(size, device=first.device)
    page = (at // state.page_size).clamp(max=state.page_table.shape[1] - 1)
    ids = state.page_table.long().gather(1, page.flatten(1)).view(at.shape)
    named = (at < state.clamped_lengths()[:, None, None]) & (ids >= 0) & (ids < state.num_pages)
    return torch.where(named, ids * state.page_size + at % state.page_size, 0), named, at


def _append_scaled_torch(state, cache, new) -> None:
    if state.page_table.numel() == 0 or state.num_pages == 0 or new.numel() == 0:
        return
    queries, block, dtype = state.queries, cache.block, cache.dtype
    length = state.clamped_lengths()
    fresh = (length - queries).clamp(min=0)
    slots, named, at = _positions(state, fresh // block, (queries - 1) // block + 2, block)
    row = at - length[:, None, None] + queries + \
        torch.arange(length.numel(), device=length.device)[:, None, None] * queries
    is_new = named & (at >= fresh[:, None, None])
    x = torch.where(is_new[..., None, None], new[torch.where(is_new, row, 0)].float(), 0.0)
    # (amax of a NaN is a NaN.)
    scale = scale_of(x.abs().amax((2, 4)), dtype)                  # [sequences, blocks, heads]
    blocks = slots[:, :, 0] // block
    held = cache.scales[blocks]
    begun = (named[:, :, 0] & ~is_new[:, :, 0])[..., None]
    # (By magnitude: a scale from elsewhere may be negative.  Either one's NaN stays.)
    stays = begun & ((scale <= held.abs()) | held.isnan())
    scale = torch.where(stays, held, scale)
    raw = cache.codes.view(torch.int8)
    older = raw[slots]
    got = encode(x / scale[:, :, None, :, None], dtype).view(torch.int8)
    # Older codes of a scale that stays, or by a NaN, stay as they are; others are rounded
    # again (and a NaN among them stays one).
    # As on the kernels: int8 products rounded once, e4m3's to fp32 first (both exact where
    # the older scale is a power of two).
    wide = torch.float64 if dtype == torch.int8 else torch.float32
    moved = older.view(dtype).to(wide) * (held / scale).to(wide)[:, :, None, :, None]
    moved = torch.where(moved.isnan(), older, encode(moved, dtype).view(torch.int8))
    again = (begun & (held != scale) & ~scale.isnan())[:, :, None, :, None]
    got = torch.where(is_new[..., None, None], got, torch.where(again, moved, older))
    raw[slots[named]] = got[named]
    touched = is_new.any(-1)
    cache.scales[blocks[touched]] = scale[touched]


def _sum_scaled_torch(state, cache, page_sums) -> None:
    if state.page_table.numel() == 0 or state.num_pages == 0:
        return
    size = state.page_size
    fresh = (state.clamped_lengths() - state.queries).clamp(min=0)
    slots, named, at = _positions(state, fresh // size, (state.queries - 1) // size + 2, size)
    rows = cache.codes.view(torch.int8)[slots].view(cache.dtype).float() * \
        cache.scales[slots // cache.block][..., None]
    total = torch.where(named[..., None, None], rows, 0.0).sum(2)
    touched = (named & (at >= fresh[:, None, None])).any(-1)
    page_sums[(slots[:, :, 0] // size)[touched]] = total[touched]


def plan_read(graph, key_cache, value_cache, dtype):
    """The native arguments of a read but for addresses."""
    k, v, (heads, D) = key_cache.codes, value_cache.codes, key_cache.shape[1:]
    strides = (ctypes.c_int64 * 4)(_step(k, 0), _step(k, 1), _step(v, 0), _step(v, 1))
    return strides, (graph.schema.num_dst, heads, D), heads, D, DTYPES[dtype], CODES[k.dtype], \
        key_cache.block


def read(graph, key_cache, value_cache, dtype, plan) -> tuple[torch.Tensor, torch.Tensor]:
    state = graph.paged_state
    if carries_tangent(key_cache.scales, value_cache.scales):
        raise NotImplementedError("read has no forward-mode derivative: detach the scales")
    strides, shape, heads, D, out_type, code, block = plan
    if _scaled_on_torch_operations("read", D, (key_cache, value_cache)):
        return tuple(_read_torch(state, c, dtype) for c in (key_cache, value_cache))
    k, v = key_cache.codes, value_cache.codes
    key = torch.empty(shape, dtype=dtype, device=k.device)
    value = torch.empty(shape, dtype=dtype, device=k.device)
    if key.numel():
        _native.launch(key, "tgx_paged_read", state.native(), k.data_ptr() or None,
                       key_cache.scales.data_ptr() or None, v.data_ptr() or None,
                       value_cache.scales.data_ptr() or None, strides, key.data_ptr(),
                       value.data_ptr(), heads, D, out_type, code, block)
    return key, value


def _read_torch(state, cache, dtype) -> torch.Tensor:
    heads, D = cache.shape[1:]
    rows = state.page_table.shape[0] * state.queries
    if state.page_table.numel() == 0 or state.num_pages == 0:
        return torch.zeros(rows, heads, D, dtype=dtype, device=state.lengths.device)
    length = state.clamped_lengths()
    at = length[:, None] - state.queries + torch.arange(state.queries, device=length.device)
    ids = state.page_table.long().gather(1, at.clamp(min=0) // state.page_size)
    named = (at >= 0) & (ids >= 0) & (ids < state.num_pages)
    slots = torch.where(named, ids * state.page_size + at % state.page_size, 0).flatten()
    got = cache.codes.view(torch.int8)[slots].view(cache.dtype).float() * \
        cache.scales[slots // cache.block][..., None]
    return torch.where(named.flatten()[:, None, None], got, 0.0).to(dtype)


# ---------------------------------------------------------------------------
# select

def select(graph, query, page_sums, count: int, table, lengths) -> None:
    """Write the chosen pages of every (row, key head) to `table`
    [rows, heads, count] and the positions they hold to `lengths` [rows]."""
    state = graph.paged_state
    query, page_sums = query.detach(), page_sums.detach()
    if _on_torch_operations("select_pages", query):
        _select_torch(state, query, page_sums, count, table, lengths)
        return
    if query.shape[-1] > 1 and query.stride(-1) != 1:
        query = query.contiguous()
    rows, heads, group, D = query.shape
    if rows == 0:
        return
    relation = state.native()
    need = state.checked.get(("select-workspace", heads, count))
    if need is None:
        bytes_ = ctypes.c_size_t()
        _native.call("tgx_select_pages_workspace", relation, heads, count, ctypes.byref(bytes_))
        need = state.checked["select-workspace", heads, count] = bytes_.value
    work = torch.empty(need, dtype=torch.uint8, device=query.device)
    strides = (ctypes.c_int64 * 3)(*query.stride()[:3])
    _native.launch(query, "tgx_select_pages", relation, query.data_ptr(), strides,
                   page_sums.data_ptr() if page_sums.numel() else None, heads, group, D,
                   DTYPES[query.dtype], count, table.data_ptr(), lengths.data_ptr(),
                   work.data_ptr(), need)
    torch.autograd.graph.increment_version((table, lengths))


def _select_torch(state, query, page_sums, count, table, lengths) -> None:
    size = state.page_size
    limit = state.limits().reshape(-1)
    pages = (limit + size - 1) // size
    kept = pages.clamp(max=count)
    lengths.copy_(torch.where(limit > 0, (kept - 1) * size + limit - (pages - 1) * size, 0))
    table.fill_(-1)
    summed = query.double().sum(2)
    for row in range(query.shape[0]):
        n = int(pages[row])
        if n == 0:
            continue
        ids = state.page_table[row // state.queries, :n].long()
        ok = (ids[:-1] >= 0) & (ids[:-1] < state.num_pages)
        score = torch.full((query.shape[1], n - 1), -torch.inf, dtype=torch.float64,
                           device=query.device)
        if bool(ok.any()):
            got = (page_sums[ids[:-1][ok]].double() * summed[row]).sum(-1).T
            score[:, ok] = torch.where(torch.isnan(got), -torch.inf, got)
        want = int(kept[row]) - 1
        best = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :want]
        chosen = torch.cat([best.sort(-1).values,
                            best.new_full((best.shape[0], 1), n - 1)], -1)
        table[row, :, :want + 1] = ids[chosen].to(table.dtype)


# ---------------------------------------------------------------------------
# The relation's edges

def csr(state):
    """(row_ptr, col_idx), int64, of the relation as its table and lengths
    stand: row ((sequence * queries + token) * table heads + head), column
    slot * table heads + head, in order of position."""
    device = state.page_table.device
    heads, size = state.table_heads, state.page_size
    table = state.page_table.long()
    if table.ndim == 2:
        table = table[:, None]
    limit = state.limits()                                        # [sequences, queries]
    position = torch.arange(table.shape[2] * size, device=device)
    ids = table[:, :, position // size]                           # [sequences, heads, positions]
    there = (ids >= 0) & (ids < state.num_pages)
    column = (ids * size + position % size) * heads + torch.arange(heads, device=device)[:, None]
    # [sequences, queries, heads, positions]
    edge = there[:, None] & state.sees(position, limit[:, :, None, None])
    row_ptr = torch.zeros(limit.numel() * heads + 1, dtype=torch.int64, device=device)
    torch.cumsum(edge.sum(-1).reshape(-1), 0, out=row_ptr[1:])
    return row_ptr, column[:, None].expand(edge.shape)[edge]
