"""Relations that look back over a window and a few first tokens, on host tensors
against the definition; their task lists; and what they refuse."""

import ctypes

import numpy as np
import pytest
import torch

import tiga as tg
from tiga import _native

import scaled_reference as want


class Attention(tg.MessagePassing):
    reducer = tg.online_softmax()

    def edge(self, src, dst, edge, scale):
        return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)


def edges(lengths, window, sinks):
    """The relation as a set of rows, each its columns in order."""
    out, start = [], 0
    for n in lengths:
        out += [[start + int(j) for j in want.seen(i + 1, window, sinks)] for i in range(n)]
        start += n
    return out


def packed(lengths, dtype=torch.int64):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=dtype)


@pytest.mark.parametrize("lengths", [[7], [0, 5, 1, 12, 0], [], [0]])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 2), (2, 9), (100, 0), (1, 1)])
def test_the_edges_are_the_last_and_the_first(lengths, window, sinks):
    g = tg.Graph.cu_seqlens(packed(lengths), window=window, sinks=sinks)
    rows = edges(lengths, window, sinks)
    degrees = [len(r) for r in rows]
    assert g.num_edges == sum(degrees)
    assert g.degree_bounds() == ((min(degrees), max(degrees)) if degrees else (0, 0))
    assert g.degree_histogram() == tuple(np.bincount(degrees, minlength=1)) if degrees else True
    row_ptr, col = g.resolve_csr()
    assert [col[a:b].tolist() for a, b in zip(row_ptr[:-1], row_ptr[1:])] == rows
    assert col.dtype == row_ptr.dtype == torch.int64
    assert g.num_edges == sum(degrees) and g.transpose().num_edges == sum(degrees)
    if len(lengths) == 1:
        t = tg.Graph.triangular(lengths[0], window=window, sinks=sinks)
        assert t.num_edges == g.num_edges and t.is_dense
        assert all(torch.equal(a, b) for a, b in zip(t.resolve_csr(), (row_ptr, col)))


def test_relations_joined_keep_their_window():
    a = tg.Graph.cu_seqlens(packed([4, 3]), window=2, sinks=1)
    b = tg.Graph.triangular(5, window=2, sinks=1)
    g = tg.Graph.cat([a, b])
    assert g.is_varlen and g.num_edges == a.num_edges + b.num_edges
    assert torch.equal(g.resolve_csr()[1],
                       tg.Graph.cu_seqlens(packed([4, 3, 5]), window=2, sinks=1).resolve_csr()[1])
    other = tg.Graph.cat([a, tg.Graph.triangular(5, window=3, sinks=1)])
    assert not other.is_varlen
    assert other.num_edges == a.num_edges + tg.Graph.triangular(5, window=3, sinks=1).num_edges
    assert a.planning_key() != tg.Graph.cu_seqlens(packed([4, 3])).planning_key()
    assert a.planning_key() != tg.Graph.cu_seqlens(packed([4, 3]), window=2).planning_key()


@pytest.mark.parametrize("heads,group,D", [(2, 3, 8), (1, 1, 4)])
def test_attention_and_its_gradients_on_the_host(heads, group, D):
    rng = np.random.default_rng(1)
    lengths, window, sinks = [0, 9, 1, 14], 4, 2
    n = sum(lengths)
    q, d = rng.standard_normal((2, n, heads, group, D))
    k, v = rng.standard_normal((2, n, heads, D))
    t = [torch.tensor(x, requires_grad=True) for x in (q, k[:, :, None], v[:, :, None])]
    out = Attention()(graph=tg.Graph.cu_seqlens(packed(lengths), window=window, sinks=sinks),
                      src={"key": t[1], "value": t[2]}, dst={"query": t[0]}, scale=0.4)
    got = [out, *torch.autograd.grad(out, t, torch.tensor(d))]
    exp, _ = want.window_attention(lengths, q, k, v, 0.4, window, sinks, d)
    for a, b in zip(got, exp):
        assert np.abs(a.detach().numpy().reshape(b.shape) - b).max() <= 1e-12


def test_the_reference_gradients_are_the_differences():
    """The oracle's own gradients against central differences of its output."""
    rng = np.random.default_rng(2)
    q, d = rng.standard_normal((2, 6, 1, 2, 3))
    k, v = rng.standard_normal((2, 6, 1, 3))
    res, _ = want.window_attention([6], q, k, v, 0.7, 3, 1, d)
    f = lambda: (want.window_attention([6], q, k, v, 0.7, 3, 1)[0] * d).sum()
    for x, grad in ((q, res[1]), (k, res[2]), (v, res[3])):
        for at in [tuple(rng.integers(s) for s in x.shape) for _ in range(5)]:
            kept, h = x[at], 1e-5
            x[at] = kept + h
            up = f()
            x[at] = kept - h
            down = f()
            x[at] = kept
            assert abs((up - down) / (2 * h) - grad[at]) <= 1e-8


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 2), (2, 9), (100, 0)])
@pytest.mark.parametrize("queries", [1, 3])
def test_paged_relations(window, sinks, queries):
    """The window counts from each asking token; pages in between may name nothing."""
    size, pages = 4, 9
    table = torch.tensor([[3, 0, 7], [5, -1, 8], [1, 2, 6]], dtype=torch.int32)
    lengths = torch.tensor([1, 12, 11], dtype=torch.int32)
    g = tg.Graph.paged(table, lengths, page_size=size, num_pages=pages, queries=queries,
                       window=window, sinks=sinks)
    row_ptr, col = g.resolve_csr()
    for b in range(3):
        for t in range(queries):
            n = max(int(lengths[b]) - (queries - 1 - t), 0)
            exp = [int(table[b, j // size]) * size + j % size for j in want.seen(n, window, sinks)
                   if table[b, j // size] >= 0]
            r = b * queries + t
            assert col[row_ptr[r]:row_ptr[r + 1]].tolist() == exp
    assert g.num_edges == col.numel()
    plain = tg.Graph.paged(table, lengths, page_size=size, num_pages=pages, queries=queries)
    assert g.planning_key() != plain.planning_key()
    # append is the same with a window and without.
    x = torch.randn(3 * queries, 1, 2)
    caches = [torch.zeros(pages * size, 1, 2) for _ in range(4)]
    g.append(caches[0], x, caches[1], x)
    plain.append(caches[2], x, caches[3], x)
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_what_is_refused():
    cu = packed([4])
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    paged = lambda **kw: tg.Graph.paged(table, lengths, page_size=4, num_pages=1, **kw)
    for make in (lambda **kw: tg.Graph.cu_seqlens(cu, **kw), paged,
                 lambda **kw: tg.Graph.triangular(4, **kw)):
        for kw in (dict(window=0), dict(window=-1), dict(window=1.5), dict(window=True),
                   dict(window=2**31), dict(sinks=1), dict(window=2, sinks=-1),
                   dict(window=2, sinks="1")):
            with pytest.raises(ValueError):
                make(**kw)
    with pytest.raises(ValueError, match="causal"):
        tg.Graph.cu_seqlens(cu, causal=False, window=2)
    with pytest.raises(ValueError, match="window"):
        paged(window=2).select_pages(torch.zeros(1, 1, 1, 8), torch.zeros(1, 1, 8), 1)

    class Pruned(Attention):
        reducer = tg.online_softmax(block_prune_threshold=0.5)

    x = torch.randn(4, 1, 8)
    with pytest.raises(NotImplementedError):
        Pruned()(graph=tg.Graph.triangular(4, window=2), src={"key": x, "value": x},
                 dst={"query": x}, scale=1.0)


def tasks_of(lengths, heads, group, window, sinks, kind):
    cu = packed(lengths).to(torch.int32).numpy()
    n, slots = ctypes.c_int64(), ctypes.c_int64()
    args = (cu.ctypes.data, len(lengths), heads, group, window, sinks, kind)
    _native.call("tgx_window_tasks", *args, None, ctypes.byref(n), ctypes.byref(slots))
    out = np.zeros((n.value, 4 if kind == 0 else 8), dtype=np.int32)
    _native.call("tgx_window_tasks", *args, out.ctypes.data, ctypes.byref(n), ctypes.byref(slots))
    return (out if kind == 2 else out[out[:, 0] >= 0]), slots.value, n.value


@pytest.mark.parametrize("lengths,heads,group,window,sinks", [
    ([1], 1, 1, 1, 0), ([300, 0, 64, 65], 2, 3, 50, 4), ([5000], 2, 4, 100, 70),
    ([2000, 700], 1, 5, 1, 130), ([900], 1, 128, 10**9, 10**9), ([], 2, 1, 4, 0), ([0, 0], 1, 1, 3, 3)])
def test_tasks_cover_every_pair_once(lengths, heads, group, window, sinks):
    rows, _, count = tasks_of(lengths, heads, group, window, sinks, 0)
    assert count % 8 == 0
    exp = {(b, r, h) for b, n in enumerate(lengths) for h in range(heads)
           for r in range(0, n * group, 128)}
    assert len(rows) == len(exp) and {tuple(r[:3]) for r in rows} == exp
    keys, slots, _ = tasks_of(lengths, heads, group, window, sinks, 1)
    joins, _, _ = tasks_of(lengths, heads, group, window, sinks, 2)
    by_tile = {}
    for b, k0, h, first, blocks, slot, *_ in keys.tolist():
        by_tile.setdefault((b, k0, h), []).append((first, blocks, slot))
    assert set(by_tile) == {(b, k, h) for b, n in enumerate(lengths) for h in range(heads)
                            for k in range(0, n, 64)}
    joined = {tuple(j[:3]): (j[3], j[4]) for j in joins.tolist()}
    used = []
    for (b, k0, h), parts in by_tile.items():
        parts.sort()
        # Whole runs of row blocks, from the tile's first query to the last that sees it.
        assert parts[0][0] == k0 * group // 64
        assert all(a + n == c for (a, n, _), (c, _, _) in zip(parts, parts[1:]))
        end = parts[-1][0] + parts[-1][1]
        n = lengths[b]
        last = n - 1 if k0 < sinks else min(n - 1, k0 + 63 + window - 1)
        assert (end - 1) * 64 < (last + 1) * group <= end * 64
        if len(parts) == 1:
            assert parts[0][2] == -1 and (b, k0, h) not in joined
        else:
            first, count = joined[b, k0, h]
            assert [s for _, _, s in parts] == list(range(first, first + count))
            used += [s for _, _, s in parts]
    assert sorted(used) == list(range(slots))


def test_native_entries_refuse_what_they_do_not_take():
    cu = np.array([0, 4], dtype=np.int32)
    n, slots = ctypes.c_int64(), ctypes.c_int64()
    task = lambda cu=cu.ctypes.data, heads=1, group=1, window=1, sinks=0, kind=0: _native.call(
        "tgx_window_tasks", cu, 1, heads, group, window, sinks, kind, None, ctypes.byref(n),
        ctypes.byref(slots))
    task()
    back = np.array([4, 0], dtype=np.int32)
    for kw in (dict(cu=None), dict(cu=back.ctypes.data), dict(heads=0), dict(group=0),
               dict(group=129), dict(window=0), dict(sinks=-1), dict(kind=3)):
        with pytest.raises(RuntimeError):
            task(**kw)
    one, seven = 0x1000, (ctypes.c_int64 * 7)(*[64] * 7)
    fwd = lambda q=one, s=seven, window=1, D=64, dtype=0, group=1, n=4: _native.call(
        "tgx_window_attn_fwd", one, one, 8, q, one, one, s, 1.0, window, 0, one, one, one, n, 1, group,
        D, dtype, None)
    for kw in (dict(q=None), dict(q=one + 8), dict(s=None), dict(s=(ctypes.c_int64 * 7)(*[4] * 7)),
               dict(window=0), dict(group=0), dict(group=129), dict(n=-1), dict(n=2**31)):
        with pytest.raises(RuntimeError):
            fwd(**kw)
    for kw in (dict(D=96), dict(dtype=2), dict(s=(ctypes.c_int64 * 7)(*[2**24] * 7))):
        with pytest.raises(NotImplementedError):
            fwd(**kw)
    need = ctypes.c_size_t()
    _native.call("tgx_window_attn_bwd_workspace", 4, 3, 1, 1, 64, ctypes.byref(need))
    bwd = lambda work=one, size=need.value, dq=one: _native.call(
        "tgx_window_attn_bwd", one, one, 8, one, 8, one, 1, 3, one, one, one, seven, one, one, one,
        one, 1.0, 1, 0, dq, one, one, 4, 1, 1, 64, 0, work, size, None)
    for kw in (dict(work=None), dict(size=need.value - 1), dict(dq=None), dict(dq=one + 8)):
        with pytest.raises(RuntimeError):
            bwd(**kw)


@pytest.mark.parametrize("lengths,heads,group,window,sinks", [
    ([131072], 8, 4, 128, 1024), ([32768], 8, 4, 256, 4096), ([131072], 8, 8, 1024, 8192),
    ([20000] * 6, 4, 16, 64, 20000), ([300] * 500, 32, 1, 1, 64), ([1000000], 1, 1, 64, 64)])
def test_partial_sums_are_bounded(lengths, heads, group, window, sinks):
    """The backward's workspace does not grow with sinks times tokens: of all the work a
    piece has at least 1 / 2048, and a tile that is cut more than two pieces' work."""
    keys, slots, _ = tasks_of(lengths, heads, group, window, sinks, 1)
    joins, same, _ = tasks_of(lengths, heads, group, window, sinks, 2)
    assert same == slots == joins[:, 4].sum() and slots <= 1.5 * 2048
    need = ctypes.c_size_t()
    n = sum(lengths)
    _native.call("tgx_window_attn_bwd_workspace", n, slots, heads, group, 128, ctypes.byref(need))
    assert need.value <= 4 * n * heads * group + 256 + 1.5 * 2048 * 2 * 64 * 128 * 4
    # Nothing is longer than the longest tile without sinks, or two pieces.
    total = int(keys[:, 4].sum())
    piece = max(-(-(window + 63) * group // 64), 16, -(-total // 2048))
    assert keys[:, 4].max() <= max(2 * piece, -(-(window + 63) * group // 64) + 1)


def test_a_forward_alone_prepares_no_backward(monkeypatch):
    """Without gradients, also of inputs that want them elsewhere, a call forms no lists of
    key tiles and has no second part of the output written.  (Launches are recorded only.)"""
    from tiga import _ops

    calls = []
    monkeypatch.setattr(_native, "launch", lambda t, name, *args: calls.append((name, args)))
    rng = np.random.default_rng(4)
    mk = lambda *s: torch.tensor(rng.standard_normal(s)).to(torch.bfloat16).requires_grad_(True)
    q, k, v = mk(70, 2, 3, 32), mk(70, 2, 1, 32), mk(70, 2, 1, 32)
    g = tg.Graph.cu_seqlens(packed([40, 30]), window=5, sinks=1)
    run = lambda q: _ops.window_attention(q, k, v, 0.2, 2, 3, g)
    plan = lambda: g._native_cache["window-plan", 2, 3, 32]
    rest = lambda: calls[-1][1][11]
    with torch.no_grad():
        assert not run(q).requires_grad
    assert calls[-1][0] == "tgx_window_attn_fwd" and rest() is None
    assert plan().backward is None and ("window", 1, 2, 3) not in g._native_cache
    out = run(q.detach())                        # (the keys and values want gradients)
    assert rest() and plan().backward is not None
    grads = torch.autograd.grad(out, (k, v), torch.ones_like(out))
    assert [c[0] for c in calls[-2:]] == ["tgx_window_attn_fwd", "tgx_window_attn_bwd"]
    assert calls[-1][1][13] == calls[-2][1][11]
    assert [x.shape for x in grads] == [k.shape, v.shape]
    with torch.no_grad():
        run(q)
    assert rest() is None
    with torch.inference_mode():
        run(q)
    assert rest() is None


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_lists_too_long_for_a_launch_are_refused_before_they_are_formed(kind):
    cu = np.array([0, 2 ** 20, 2 ** 30], dtype=np.int32)
    n, slots = ctypes.c_int64(), ctypes.c_int64()
    for blocks, heads in ((1, 2 ** 30), (1, 2 ** 11), (2, 1)):
        if blocks == 2 and kind == 0:
            continue
        with pytest.raises(RuntimeError, match="too many tasks"):
            _native.call("tgx_window_tasks", cu.ctypes.data, blocks, heads, 1, 64, 1, kind, None,
                         ctypes.byref(n), ctypes.byref(slots))
