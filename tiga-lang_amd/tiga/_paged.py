"""Launches over a paged cache relation (``Graph.paged``): attention, the
upkeep of the cache and the choice of pages (csrc/tgx_paged.hip,
csrc/tgx_pages.hip), and the same on Torch operations for host tensors.

The page tables and lengths are read by the kernels at every launch, so none
of these copies them to the host or synchronises; outputs and workspaces are
allocated by Torch on the current stream of the operands' device.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native
from ._dual import carries_tangent

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
            torch.is_grad_enabled()) or carries_tangent(q, k, v)


def csr_takes(D: int) -> bool:
    """Whether the CSR attention kernels take heads of this width."""
    return D % 8 == 0 and 8 <= D <= 512 and (D // 8) & (D // 8 - 1) == 0


def attention_workspace(graph, heads: int, group: int, D: int, code: int) -> int | None:
    """Workspace bytes of an attention launch, None where no launch covers the
    sizes; asked once a relation and shape."""
    state = graph.paged_state
    key = ("attention-workspace", heads, group, D, code)
    need = state.checked.get(key)
    if need is None:
        bytes_ = ctypes.c_size_t()
        with torch.cuda.device(graph.device):
            takes = _native.covered("tgx_paged_attn_workspace", state.native(), heads, group, D,
                                    code, ctypes.byref(bytes_))
        need = state.checked[key] = bytes_.value if takes else -1
    return None if need < 0 else need


def bind_attention(graph, q, k, v, scale: float, heads: int, group: int):
    """The attention launch with its native arguments bound: a zero-argument
    callable that returns a new output."""
    state = graph.paged_state
    for t in (q, k, v):
        if t.device != graph.device:
            raise ValueError(f"operand on {t.device} for a graph on {graph.device}")
    q, k, v = (_on_16_bytes(t) for t in (q, k, v))
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
    need = attention_workspace(graph, heads, group, D, code)
    if need is None:
        raise NotImplementedError("paged attention: too many sequences, heads and queries for one "
                                  "launch")
    shape, dtype, device = q.shape, q.dtype, q.device
    tensors = (q.data_ptr(), k.data_ptr() if k.numel() else None,
               v.data_ptr() if v.numel() else None)

    def launch(keep=(q, k, v)):
        if carries_tangent(*keep):
            raise NotImplementedError("paged attention has no forward-mode derivative")
        out = torch.empty(shape, dtype=dtype, device=device)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _native.launch(out, "tgx_paged_attn", state.native(), *tensors, strides, scale,
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


def append(graph, key_cache, key, value_cache, value, page_sums) -> None:
    state = graph.paged_state
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
    edge = there[:, None] & (position < limit[:, :, None, None])  # [.., queries, heads, ..]
    row_ptr = torch.zeros(limit.numel() * heads + 1, dtype=torch.int64, device=device)
    torch.cumsum(edge.sum(-1).reshape(-1), 0, out=row_ptr[1:])
    return row_ptr, column[:, None].expand(edge.shape)[edge]
