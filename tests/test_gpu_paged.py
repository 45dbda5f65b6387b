"""Paged attention, append and page selection on the HIP kernels against the
formulas in float64: lengths of nothing, of one and across tiles and pieces,
pages that are not there, values nobody may see, strides, live tables,
captured launches, streams and gradients."""

import numpy as np
import pytest
import torch

import tiga as tg
from tiga import _native

import paged_reference as want

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Attention(tg.MessagePassing):
    reducer = tg.online_softmax()

    def edge(self, src, dst, edge, scale):
        return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)


@pytest.fixture(autouse=True)
def _strict():
    tg.config.strict = True
    yield
    tg.config.strict = False


f64 = lambda t: t.detach().double().cpu().numpy()


def relation(rng, lengths, size, spare=2, width=None, missing=0):
    """(table, lengths, num_pages): shuffled pages, -1 where nothing is named;
    `missing` of the named pages are pages that do not exist."""
    used = [-(-max(n, 0) // size) for n in lengths]
    width = width or max(max(used), 1) + 1
    num_pages = sum(used) + spare
    order = rng.permutation(num_pages)
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        n = min(n, width)
        table[b, :n] = order[at:at + n]
        at += n
    for _ in range(missing):
        b = int(rng.integers(len(lengths)))
        if used[b]:
            table[b, rng.integers(min(used[b], width))] = rng.choice([-5, num_pages, 2 ** 31 - 1])
    return table, np.asarray(lengths, dtype=np.int32), num_pages


def bound(dtype, q, k, v, exp, scale, keys):
    """What rounding can do to an attention output: half a step of the output;
    half a step of each weight (16-bit weights multiply V; the denominator
    rounds the same weights); in fp32 the score's D products (the relative
    error of a weight is the score's absolute one) and the additions over a
    lane's share of the keys."""
    half = torch.finfo(dtype).eps / 2
    f32 = 2.0 ** -24
    D = q.shape[-1]
    vmax = np.abs(v).max()
    score = scale * np.sqrt((q ** 2).sum(-1).max() * (k ** 2).sum(-1).max())
    weight = 2 * ((D + 8) * f32 * (score + 1) + (keys / 16 + 64) * f32)
    if dtype != torch.float32:
        weight += 2 * half
    return half * np.abs(exp) + weight * vmax + np.finfo(np.float32).tiny


def check(lengths, size, heads, group, D, dtype, queries=1, seed=0, missing=0, width=None,
          poison=True, interleave=False):
    print(f"paged {dtype} D={D} heads={heads} group={group} queries={queries} size={size} "
          f"lengths={lengths[:6]} missing={missing}", flush=True)
    rng = np.random.default_rng(seed)
    table, length, num_pages = relation(rng, lengths, size, width=width, missing=missing)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(length, device=DEV),
                       page_size=size, num_pages=num_pages, queries=queries)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(dtype)
    slots = num_pages * size
    q = mk(len(lengths) * queries, heads, group, D)
    if interleave:      # keys and values of a slot next to each other
        kv = mk(slots, 2, heads, D)
        k, v = kv[:, 0], kv[:, 1]
    else:
        k, v = mk(slots, heads, D), mk(slots, heads, D)
    scale = D ** -0.5
    exp = want.attention(table, length, size, num_pages, queries, f64(q), f64(k), f64(v), scale)
    ek, ev = f64(k), f64(v)
    if poison:
        # Slots that no row sees hold NaN and Inf.
        seen = np.zeros(slots, dtype=bool)
        for b in range(len(lengths)):
            n = want.length_of(length, b, table.shape[1], size)
            at, named = want.slots(table[b], n, size, num_pages)
            seen[at[named]] = True
        hidden = torch.tensor(~seen, device=DEV)
        k[hidden] = float("nan")
        v[hidden] = float("inf")
    kernel = Attention()
    out = kernel(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]}, dst={"query": q},
                 scale=scale)
    assert kernel.last_variant.pattern == "paged-attention"
    assert out.shape == q.shape and out.dtype == dtype
    err = np.abs(f64(out) - exp)
    lim = bound(dtype, f64(q), ek, ev, exp, scale, max(lengths))
    assert (err <= lim).all(), f"error {err.max():.3e}, {(err / lim).max():.2f} of the bound"
    return kernel, g, q, k, v, out


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("queries", [1, 3])
def test_lengths_around_tiles_and_pages(dtype, D, queries):
    check(EDGES, 16, 2, 4, D, TYPES[dtype], queries=queries)


@pytest.mark.parametrize("D", [8, 24, 40, 80, 96, 192, 256, 320, 512])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_other_widths(D, dtype):
    check([0, 1, 70, 333], 16, 2, 2, D, TYPES[dtype])


@pytest.mark.parametrize("size", [1, 3, 8, 24, 48, 100, 256])
def test_page_sizes_that_end_inside_a_tile(size):
    check([5, 64, 131, 700], size, 2, 4, 64, torch.float16, queries=2, seed=size)


@pytest.mark.parametrize("heads,group,queries", [
    (1, 1, 1), (3, 1, 1), (8, 4, 1), (1, 16, 1), (1, 17, 1), (2, 32, 1), (2, 5, 4), (2, 7, 5),
    (1, 3, 40), (2, 71, 1)])
def test_head_groups_and_queries(heads, group, queries):
    check([0, 1, 30, 64, 200], 16, heads, group, 64, torch.bfloat16, queries=queries)
    check([0, 1, 30, 64, 200], 16, heads, group, 128, torch.float16, queries=queries)


@pytest.mark.parametrize("lengths", [[20000], [9000, 1, 0, 300, 4111], [3000] * 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_long_lengths_in_pieces(lengths, dtype):
    check(lengths, 16, 2, 4, 64 if len(lengths) > 9 else 128, TYPES[dtype], queries=2)


def test_many_sequences():
    rng = np.random.default_rng(5)
    check([int(n) for n in rng.integers(0, 40, size=700)], 8, 1, 2, 32, torch.float16)


@pytest.mark.parametrize("dtype", TYPES)
def test_launches_that_are_not_split(dtype):
    """Short tables of many sequences, and as many workgroups of one piece as the
    GPU holds."""
    rng = np.random.default_rng(15)
    check([int(n) for n in rng.integers(0, 1000, size=150)], 16, 2, 2, 64, TYPES[dtype])
    if dtype != "f32":
        check([400, 20], 16, 8, 16, 128, TYPES[dtype], queries=300)


@pytest.mark.parametrize("dtype", TYPES)
def test_pages_that_are_not_there(dtype):
    check([40, 64, 300, 1000], 16, 2, 3, 64, TYPES[dtype], queries=2, missing=12)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_lengths_outside_the_table_are_clamped(dtype):

    rng = np.random.default_rng(0)
    table = rng.permutation(20).reshape(5, 4).astype(np.int32)
    lengths = np.array([-3, 70, 64, 2 ** 31 - 1, -2 ** 31], dtype=np.int32)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=20, queries=2)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(TYPES[dtype])
    q, k, v = mk(10, 2, 64), mk(320, 2, 64), mk(320, 2, 64)
    out = Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.125)
    exp = want.attention(table, lengths, 16, 20, 2, f64(q)[:, :, None], f64(k), f64(v), 0.125)
    lim = bound(TYPES[dtype], f64(q), f64(k), f64(v), exp[:, :, 0], 0.125, 64)
    assert (np.abs(f64(out) - exp[:, :, 0]) <= lim).all()


def test_keys_and_values_of_a_slot_next_to_each_other():
    check([0, 77, 1000], 16, 4, 2, 64, torch.bfloat16, interleave=True)
    check([0, 77, 1000], 16, 4, 2, 64, torch.float32, interleave=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_newer_tokens_never_reach_older_rows(dtype):
    """A NaN or Inf in the newest tokens' keys and values belongs to the rows
    that see them, and to no other."""
    rng = np.random.default_rng(1)
    table, lengths, pages = relation(rng, [70, 6, 64, 131, 3], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages, queries=4)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(TYPES[dtype])
    q, k, v = mk(20, 2, 3, 64), mk(pages * 16, 2, 64), mk(pages * 16, 2, 64)
    clean = [f64(x) for x in (q, k, v)]
    exp = want.attention(table, lengths, 16, pages, 4, *clean, 0.125)
    for b, n in enumerate(lengths):
        slot = int(table[b, (n - 1) // 16]) * 16 + int(n - 1) % 16
        v[slot] = float("nan") if b % 2 else float("inf")
        k[slot, 0] = float("nan")
    out = Attention()(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]},
                      dst={"query": q}, scale=0.125)
    got = f64(out).reshape(5, 4, 2, 3, 64)
    exp = exp.reshape(got.shape)
    lim = bound(TYPES[dtype], *clean, exp, 0.125, 131)
    assert (np.abs(got - exp)[:, :3] <= lim[:, :3]).all()
    assert not np.isfinite(got[:, 3]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries,group", [(1, 4), (6, 4), (12, 4), (30, 4)])
def test_values_that_are_infinite_where_they_are_seen(dtype, queries, group):
    """Inf, -Inf and NaN of a seen value come out as the formula has them."""
    rng = np.random.default_rng(14)
    table, lengths, pages = relation(rng, [100, 300], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages, queries=queries)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(TYPES[dtype])
    q, k, v = mk(2 * queries, 2, group, 64), mk(pages * 16, 2, 64), mk(pages * 16, 2, 64)
    for pos, d, x in ((3, 5, np.inf), (50, 9, -np.inf), (60, 11, np.nan), (40, 13, np.inf),
                      (41, 13, -np.inf)):
        for b in range(2):
            v[int(table[b, pos // 16]) * 16 + pos % 16, :, d] = x
    out = Attention()(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]},
                      dst={"query": q}, scale=0.125)
    with np.errstate(invalid="ignore"):
        exp = want.attention(table, lengths, 16, pages, queries, f64(q), f64(k), f64(v), 0.125)
    got = f64(out)
    assert np.array_equal(np.isnan(got), np.isnan(exp))
    assert np.array_equal(np.isposinf(got), np.isposinf(exp))
    assert np.array_equal(np.isneginf(got), np.isneginf(exp))
    fin = np.isfinite(exp)
    lim = bound(TYPES[dtype], f64(q), f64(k), np.nan_to_num(f64(v), posinf=0, neginf=0), exp,
                0.125, 300)
    assert (np.abs(got - exp)[fin] <= lim[fin]).all()


@pytest.mark.parametrize("scale", [0.0, -0.25, 30.0])
def test_scales(scale):
    rng = np.random.default_rng(2)
    table, lengths, pages = relation(rng, [200, 65], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages)
    for dtype in TYPES.values():
        mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(dtype)
        q, k, v = mk(2, 2, 64), mk(pages * 16, 2, 64), mk(pages * 16, 2, 64)
        out = Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=scale)
        exp = want.attention(table, lengths, 16, pages, 1, f64(q)[:, :, None], f64(k), f64(v),
                             scale)[:, :, 0]
        lim = bound(dtype, f64(q), f64(k), f64(v), exp, abs(scale), 200)
        assert (np.abs(f64(out) - exp) <= lim).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_table_per_head(dtype):
    """Rows of (sequence, token, head), sources of (slot, head), and key heads
    inside a table head."""
    rng = np.random.default_rng(16)
    B, T, P, size, pages, queries, heads, group, D = 3, 4, 6, 16, 30, 2, 2, 3, 64
    table = rng.integers(-1, pages, size=(B, T, P)).astype(np.int32)
    lengths = np.array([90, 1, 33], dtype=np.int32)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=size, num_pages=pages, queries=queries)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(TYPES[dtype])
    q = mk(B * queries * T, heads, group, D)
    k, v = mk(pages * size * T, heads, 1, D), mk(pages * size * T, heads, 1, D)
    out = Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.125)
    by = lambda t: f64(t).reshape(pages * size, T, heads, D)
    exp = want.attention(table, lengths, size, pages, queries, f64(q), by(k), by(v), 0.125)
    lim = bound(TYPES[dtype], f64(q), f64(k), f64(v), exp, 0.125, 90)
    assert (np.abs(f64(out) - exp) <= lim).all()


def test_field_shapes_without_a_group_dimension():
    rng = np.random.default_rng(3)
    table, lengths, pages = relation(rng, [33, 100], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(torch.float16)
    q, k, v = mk(2, 6, 64), mk(pages * 16, 1, 64), mk(pages * 16, 1, 64)
    out = Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.125)
    wide = Attention()(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]},
                       dst={"query": q[:, None]}, scale=0.125)
    assert torch.equal(out, wide[:, 0])
    # Queries that are strided, and on no 16 bytes.
    odd = torch.zeros(2, 6, 65, device=DEV, dtype=torch.float16)[..., 1:]
    odd.copy_(q)
    assert torch.equal(Attention()(graph=g, src={"key": k, "value": v}, dst={"query": odd},
                                   scale=0.125), out)


def test_a_misaligned_cache_is_copied_or_goes_through_the_snapshot():
    rng = np.random.default_rng(4)
    table, lengths, pages = relation(rng, [33, 100], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(torch.float16)
    q, k, v = mk(2, 2, 64), mk(pages * 16, 2, 64), mk(pages * 16, 2, 64)
    kernel = Attention()
    call = lambda k, v: kernel(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.125)
    out = call(k, v)

    def shifted(t, row):
        flat = torch.zeros(t.shape[0] * row + 1, device=DEV, dtype=t.dtype)
        view = torch.as_strided(flat, t.shape, (row, 64, 1), 1)
        return view.copy_(t)

    assert torch.equal(call(shifted(k, 128), shifted(v, 128)), out)   # the start is odd
    assert kernel.last_variant.pattern == "paged-attention"
    through = call(shifted(k, 131), shifted(v, 131))                  # every row is
    assert kernel.last_variant.pattern == "dot-product"
    lim = bound(torch.float16, f64(q), f64(k), f64(v), f64(out), 0.125, 100)
    assert (np.abs(f64(through) - f64(out)) <= 2 * lim).all()


def test_prepared_and_captured_launches_follow_the_live_tables():
    rng = np.random.default_rng(6)
    full = [900, 50, 17]
    table, _, pages = relation(rng, full, 16)
    live = torch.tensor([1, 1, 1], dtype=torch.int32, device=DEV)
    ids = torch.tensor(table, device=DEV)
    g = tg.Graph.paged(ids, live, page_size=16, num_pages=pages)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(torch.bfloat16)
    q, k, v = mk(3, 2, 4, 64), mk(pages * 16, 2, 64), mk(pages * 16, 2, 64)
    kernel = Attention()
    launch = kernel.prepare(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]},
                            dst={"query": q}, scale=0.125)
    other = Attention().prepare(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]},
                                dst={"query": q}, scale=0.25)
    graphs, outs = [], []
    for run in (launch, other):
        run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    for step in ([1, 1, 1], [900, 0, 16], [899, 50, 17], [2, 49, 3], [640, 33, 1]):
        live.copy_(torch.tensor(step, dtype=torch.int32))
        ids[0, 0], ids[1, 0] = ids[1, 0].clone(), ids[0, 0].clone()
        q.mul_(-1)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        host = ids.cpu().numpy()
        for out, run, scale in zip(outs, (launch, other), (0.125, 0.25)):
            exp = want.attention(host, step, 16, pages, 1, f64(q), f64(k), f64(v), scale)
            lim = bound(torch.bfloat16, f64(q), f64(k), f64(v), exp, scale, 900)
            assert (np.abs(f64(out) - exp) <= lim).all()
            assert torch.equal(run(), out)


def test_two_streams_at_once():
    calls = []
    for seed, lengths in ((7, [5000, 3]), (8, [64, 2000, 700])):
        _, g, q, k, v, out = check(lengths, 16, 2, 4, 64, torch.float16, seed=seed)
        calls.append((g, q, k, v, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(5):
        for i, ((g, q, k, v, _), s) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(s):
                got[i].append(Attention()(graph=g, dst={"query": q}, scale=64 ** -0.5,
                                          src={"key": k[:, :, None], "value": v[:, :, None]}))
    torch.cuda.synchronize()
    for outs, call in zip(got, calls):
        assert all(torch.equal(o, call[-1]) for o in outs)


@pytest.mark.parametrize("D", [64, 24])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_of_shared_heads(D, dtype):
    tg.config.strict = False
    rng = np.random.default_rng(9)
    table, lengths, pages = relation(rng, [0, 20, 70], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages, queries=2)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(
        TYPES[dtype]).requires_grad_(True)
    q, k, v = mk(6, 2, 3, D), mk(pages * 16, 2, 1, D), mk(pages * 16, 2, 1, D)
    dout = torch.tensor(rng.standard_normal((6, 2, 3, D)), device=DEV).to(TYPES[dtype])
    out = Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.2)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    host = [t.detach().double().cpu().requires_grad_(True) for t in (q, k, v)]
    ref = Attention()(graph=tg.Graph.paged(torch.tensor(table), torch.tensor(lengths),
                                           page_size=16, num_pages=pages, queries=2),
                      src={"key": host[1], "value": host[2]}, dst={"query": host[0]}, scale=0.2)
    exp = torch.autograd.grad(ref, host, dout.double().cpu())
    # The CSR attention's own tolerances (1e-5 of the largest value in 32 bits; 16-bit
    # output gradients and outputs round by half a step each, some four of them in a sum).
    tol = 1e-5 if dtype == "f32" else 4 * torch.finfo(TYPES[dtype]).eps
    assert float((out.double().cpu() - ref).abs().max()) <= tol * float(ref.abs().max())
    for got, e in zip(grads, exp):
        assert float((got.double().cpu() - e).abs().max()) <= tol * float(e.abs().max())


def test_other_edge_functions_run_on_the_snapshot():
    class Sum(tg.MessagePassing):
        reducer = tg.sum()

        def edge(self, src, dst, edge):
            return src.x

    rng = np.random.default_rng(10)
    table, lengths, pages = relation(rng, [0, 20, 70], 16)
    live = torch.tensor(lengths, device=DEV)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), live, page_size=16, num_pages=pages)
    x = torch.randn(pages * 16, 8, device=DEV)
    kernel = Sum()
    for _ in range(2):
        out = kernel(graph=g, src={"x": x}, dst={})
        assert kernel.last_variant.pattern == "weighted-sum"
        for b in range(3):
            at, _ = want.slots(table[b], int(live[b]), 16, pages)
            exp = f64(x)[at].sum(0)
            assert np.abs(f64(out[b]) - exp).max() <= 80 * 2 ** -24 * 70 * float(x.abs().max())
        live -= torch.tensor([0, 5, 7], dtype=torch.int32, device=DEV)


def test_a_cache_whose_offsets_pass_32_bits():
    """The last pages of a cache of 9 GB, attended to, appended to and selected."""
    heads, D, size = 8, 256, 16
    pages = 72000          # 72000 * 16 * 8 * 256 * 2 bytes = 4.7 GB each
    k = torch.empty(pages * size, heads, D, device=DEV, dtype=torch.float16)
    v = torch.empty_like(k)
    rng = np.random.default_rng(12)
    for width in (256, 64):     # (64: the first columns, on the matrix tiles)
        ids = np.arange(pages - 12, pages)[rng.permutation(12)].reshape(2, 6)
        table = torch.tensor(ids, dtype=torch.int32, device=DEV)
        lengths = torch.tensor([90, 33], dtype=torch.int32, device=DEV)
        g = tg.Graph.paged(table, lengths, page_size=size, num_pages=pages)
        mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).half()
        kc, vc = k[..., :width], v[..., :width]
        lo = (pages - 12) * size
        kc[lo:], vc[lo:] = mk(12 * size, heads, width), mk(12 * size, heads, width)
        new_k, new_v = mk(2, heads, width), mk(2, heads, width)
        sums = torch.zeros(pages, heads, width, device=DEV)
        small = [f64(kc[lo:]), f64(new_k), f64(vc[lo:]), f64(new_v), f64(sums[-12:])]
        exp = want.append(ids - (pages - 12), [90, 33], size, 12, 1, *small)
        g.append(kc, new_k, vc, new_v, page_sums=sums)
        assert np.array_equal(f64(kc[lo:]), exp[0]) and np.array_equal(f64(vc[lo:]), exp[1])
        assert np.abs(f64(sums[-12:]) - exp[2]).max() <= 16 * 2 ** -24 * 16 * 6
        q = mk(2, heads, 2, width)
        out = Attention()(graph=g, src={"key": kc[:, :, None], "value": vc[:, :, None]},
                          dst={"query": q}, scale=width ** -0.5)
        ref = want.attention(ids - (pages - 12), [90, 33], size, 12, 1, f64(q), exp[0], exp[1],
                             width ** -0.5)
        lim = bound(torch.float16, f64(q), exp[0], exp[1], ref, width ** -0.5, 90)
        assert (np.abs(f64(out) - ref) <= lim).all()
        chosen = g.select_pages(q, sums, 3)
        pick, held = want.select(ids, [90, 33], size, pages, 1, f64(q),
                                 _Offset(f64(sums[-12:]), pages - 12), 3)
        assert np.array_equal(chosen.page_table.cpu().numpy(), pick)
        assert np.array_equal(chosen.lengths.cpu().numpy(), held)


class _Offset:
    """An array whose first row has index `start`."""

    def __init__(self, rows, start):
        self.rows, self.start = rows, start

    def __getitem__(self, at):
        return self.rows[at[0] - self.start, at[1]]


def test_under_inference_mode():
    with torch.inference_mode():
        table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
        g = tg.Graph.paged(table, torch.tensor([17], dtype=torch.int32, device=DEV), page_size=16,
                           num_pages=2)
        kc = torch.zeros(32, 1, 64, device=DEV, dtype=torch.bfloat16)
        new = torch.ones(1, 1, 64, device=DEV, dtype=torch.bfloat16)
        sums = torch.zeros(2, 1, 64, device=DEV)
        q, k = tg.nn.norm_rotary(new, new, torch.tensor([16], device=DEV),
                                 torch.ones(32, device=DEV), query_weight=new[0, 0])
        g.append(kc, k, kc.clone(), new, page_sums=sums)
        chosen = g.select_pages(q, sums, 1)
        assert chosen.page_table.tolist() == [[[0]]] and chosen.lengths.tolist() == [1]
        out = Attention()(graph=chosen, src={"key": kc, "value": kc}, dst={"query": q}, scale=1.0)
        assert torch.equal(out, kc[:1])


def test_empty_relations():
    for B, P, pages in ((0, 3, 4), (3, 0, 4), (3, 2, 0)):
        table = torch.zeros(B, P, dtype=torch.int32, device=DEV)
        g = tg.Graph.paged(table, torch.full((B,), 9, dtype=torch.int32, device=DEV),
                           page_size=16, num_pages=pages, queries=2)
        q = torch.randn(2 * B, 2, 64, device=DEV, dtype=torch.float16)
        k = torch.randn(pages * 16, 2, 64, device=DEV, dtype=torch.float16)
        out = Attention()(graph=g, src={"key": k, "value": k}, dst={"query": q}, scale=1.0)
        assert out.shape == q.shape and not out.any()
        sums = torch.zeros(pages, 2, 64, device=DEV)
        new = torch.ones(2 * B, 2, 64, device=DEV, dtype=torch.float16)
        g.append(k, new, k.clone(), new, page_sums=sums)
        chosen = g.select_pages(q, sums, 3)
        assert chosen.page_table.shape == (2 * B, 2, 3)
        if P == 0:
            assert bool((chosen.page_table == -1).all()) and not chosen.lengths.any()


# ---------------------------------------------------------------------------
# append

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 2, 17, 70])
@pytest.mark.parametrize("D", [64, 20])
def test_append(dtype, queries, D):
    print(f"append {dtype} queries={queries} D={D}", flush=True)
    rng = np.random.default_rng(queries)
    table, lengths, pages = relation(rng, [1, 0, 16, 17, 90, 200, 71], 16, missing=2)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages, queries=queries)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(TYPES[dtype])
    slots, rows = pages * 16, 7 * queries
    cache = mk(slots, 2, 3, D)
    kc, vc = cache[:, 0], cache[:, 1]
    qkv = mk(rows, 8, D)
    k, v = qkv[:, 2:5], qkv[:, 5:]
    sums = torch.randn(pages, 3, D, device=DEV)
    plain = torch.zeros_like(sums)
    exp = want.append(table, lengths, 16, pages, queries, f64(kc), f64(k), f64(vc), f64(v),
                      f64(sums))
    before = kc._version
    g.append(kc, k, vc, v, page_sums=sums)
    assert kc._version > before
    assert np.array_equal(f64(kc), exp[0]) and np.array_equal(f64(vc), exp[1])
    # 16 additions in 32 bits of values of at most 6.
    assert np.abs(f64(sums) - exp[2]).max() <= 16 * 2 ** -24 * 16 * 6
    kc2 = mk(slots, 3, D)
    g.append(kc2, k, vc, v)
    g.append(kc2, k, vc, v, page_sums=plain)
    g.append(kc2, k, vc, v, page_sums=sums)
    touched = plain.abs().sum((1, 2)) != 0
    assert torch.equal(plain[touched], sums[touched])


def test_taking_tokens_back_keeps_the_sums_right():
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([0], dtype=torch.int32, device=DEV)
    g = tg.Graph.paged(table, lengths, page_size=4, num_pages=3)
    kc, vc = torch.zeros(2, 12, 1, 8, device=DEV, dtype=torch.float16)
    sums = torch.zeros(3, 1, 8, device=DEV)
    for length, value in ((1, 1.0), (2, 2.0), (3, 4.0), (2, 8.0), (3, 16.0)):
        lengths.fill_(length)
        new = torch.full((1, 1, 8), value, device=DEV, dtype=torch.float16)
        g.append(kc, new, vc, new, page_sums=sums)
    assert sums[2].unique().tolist() == [25.0]     # 1 + 8 + 16


# ---------------------------------------------------------------------------
# select

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,size,count,queries", [
    ([0, 1, 16, 17, 100, 500], 16, 4, 1),
    ([0, 1, 16, 17, 100, 500], 16, 1, 3),
    ([40, 7, 300], 4, 64, 2),
    ([9000, 300], 4, 33, 1),
    ([4111], 1, 700, 1),
])
def test_select_pages(dtype, lengths, size, count, queries):
    print(f"select {dtype} {lengths} size={size} count={count}", flush=True)
    rng = np.random.default_rng(count)
    table, length, pages = relation(rng, lengths, size, missing=2)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(length, device=DEV),
                       page_size=size, num_pages=pages, queries=queries)
    for heads, group, D in ((2, 3, 64), (3, 1, 128), (1, 5, 20)):
        q = torch.tensor(rng.standard_normal((len(lengths) * queries, heads, group, D)),
                         device=DEV).to(TYPES[dtype])
        sums = rng.standard_normal((pages, heads, D)).astype(np.float32)
        # Equal scores, NaN and Inf among them.
        for _ in range(pages // 3):
            sums[rng.integers(pages)] = sums[rng.integers(pages)]
        sums[rng.integers(pages), 0, 0] = np.nan
        sums[rng.integers(pages), 0, 0] = np.inf
        sums[rng.integers(pages)] = 0.0
        chosen = g.select_pages(q, torch.tensor(sums, device=DEV), count)
        exp_table, exp_lengths = want.select(table, length, size, pages, queries, f64(q),
                                             sums.astype(np.float64), count)
        assert np.array_equal(chosen.lengths.cpu().numpy(), exp_lengths)
        assert np.array_equal(chosen.page_table.cpu().numpy(), exp_table)


def test_select_pages_where_all_scores_are_equal():
    g = tg.Graph.paged(torch.arange(600, dtype=torch.int32, device=DEV)[None],
                       torch.tensor([1197], dtype=torch.int32, device=DEV), page_size=2,
                       num_pages=600)
    q = torch.zeros(1, 1, 1, 64, device=DEV, dtype=torch.bfloat16)
    chosen = g.select_pages(q, torch.randn(600, 1, 64, device=DEV), 300)
    assert chosen.page_table[0, 0].tolist() == [*range(299), 598]
    assert chosen.lengths.tolist() == [599]


# ---------------------------------------------------------------------------
# Together, as a program answers token by token

@pytest.mark.parametrize("captured", [False, True])
def test_a_decode_loop(captured):
    """norm_rotary, append, select_pages and attention of six steps, the lengths
    and tables advanced on the device, against the formulas."""
    rng = np.random.default_rng(11)
    B, H, G, D, size, count = 3, 2, 4, 64, 4, 3
    start, steps = np.array([0, 3, 17]), 6
    table = rng.permutation(3 * 8).reshape(3, 8).astype(np.int32)
    pages, scale, dtype = 24, D ** -0.5, torch.float16
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(dtype)
    lengths = torch.tensor(start, dtype=torch.int32, device=DEV)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), lengths, page_size=size, num_pages=pages)
    kc, vc = mk(pages * size, H, D), mk(pages * size, H, D)
    sums = kc.view(pages, size, H, D).float().sum(1)
    freqs = torch.tensor(1000.0 ** (-np.arange(D // 2) / (D // 2)), device=DEV).float()
    wq, wk = (1 + 0.1 * torch.randn(2, D, device=DEV)).to(dtype)
    qkv = torch.zeros(B, H * G + 2 * H, D, device=DEV, dtype=dtype)
    attention, chosen = Attention(), None
    flat = lambda t: t.view(-1, 1, D)

    def step():
        nonlocal chosen
        lengths.add_(1)
        q, k = tg.nn.norm_rotary(qkv[:, :H * G], qkv[:, H * G:H * G + H], lengths - 1, freqs,
                                 query_weight=wq, key_weight=wk)
        g.append(kc, k, vc, qkv[:, H * G + H:], page_sums=sums)
        chosen = g.select_pages(q.view(B, H, G, D), sums, count, out=chosen)
        out = attention(graph=chosen, src={"key": flat(kc), "value": flat(vc)},
                        dst={"query": q.view(B * H, G, D)}, scale=scale)
        return q, k, out.view(B, H, G, D)

    inputs = [mk(*qkv.shape) for _ in range(steps)]
    graph = None
    if captured:
        state = [t.clone() for t in (lengths, kc, vc, sums)]
        step()      # (allocates `chosen`, loads kernels)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
        for t, s in zip((lengths, kc, vc, sums), state):
            t.copy_(s)
    host_k, host_v, n = f64(kc), f64(vc), start.copy()
    host_sums = f64(sums)
    for x in inputs:
        qkv.copy_(x)
        if captured:
            graph.replay()
        else:
            result = step()
        q, k, out = result
        torch.cuda.synchronize()
        n += 1
        angle = want.angles((n - 1)[:, None], freqs.cpu().numpy(), (D // 2,))
        for got, part, w in ((q, x[:, :H * G], wq), (k, x[:, H * G:H * G + H], wk)):
            exp = want.norm_rotary(f64(part), f64(w), angle, 1e-6, True, False)
            # Rounded once from 32 bits: half a step, and some 40 roundings of 2^-24.
            assert (np.abs(f64(got) - exp) <= np.abs(exp) * 2.0 ** -11 +
                    40 * 2.0 ** -24 * np.abs(exp).max()).all()
        # From what was stored on: every later stage on its own inputs.
        host_k, host_v, host_sums = want.append(table, n, size, pages, 1, host_k, f64(k), host_v,
                                                f64(x[:, H * G + H:]), host_sums)
        assert np.array_equal(f64(kc), host_k) and np.array_equal(f64(vc), host_v)
        assert np.abs(f64(sums) - host_sums).max() <= 4 * 2 ** -24 * 4 * 6
        qh = f64(q).reshape(B, H, G, D)
        exp_table, exp_len = want.select(table, n, size, pages, 1, qh, f64(sums), count)
        assert np.array_equal(chosen.page_table.cpu().numpy(), exp_table)
        assert np.array_equal(chosen.lengths.cpu().numpy(), exp_len)
        exp = want.attention(exp_table, exp_len, size, pages, 1, qh.reshape(B * H, 1, G, D),
                             host_k[:, :, None], host_v[:, :, None], scale).reshape(B, H, G, D)
        assert (np.abs(f64(out) - exp) <= bound(dtype, qh, host_k, host_v, exp, scale, 12)).all()


# ---------------------------------------------------------------------------
# The C entries' refusals: on the host, before any launch

def test_c_entries_refuse_what_does_not_fit():
    import ctypes

    t = torch.zeros(4, 4, dtype=torch.int32, device=DEV)
    x = torch.zeros(64, 2, 64, dtype=torch.float16, device=DEV)
    p = _native.Paged(t.data_ptr(), 4, 0, t.data_ptr(), 4, 1, 4, 16, 4, 1)
    strides = (ctypes.c_int64 * 9)(128, 64, 64, 128, 0, 64, 128, 0, 64)
    size = ctypes.c_size_t()
    args = lambda D=64, dtype=1, q=x.data_ptr(), ws=None, n=0: (
        ctypes.byref(p), q, x.data_ptr(), x.data_ptr(), strides, 1.0, x.data_ptr(), 2, 1, D,
        dtype, ws, n, _native.stream_of(x))
    with pytest.raises(NotImplementedError, match="head width"):
        _native.call("tgx_paged_attn", *args(D=12))
    with pytest.raises(RuntimeError, match="unknown dtype"):
        _native.call("tgx_paged_attn", *args(dtype=7))
    with pytest.raises(RuntimeError, match="16 bytes"):
        _native.call("tgx_paged_attn", *args(q=x.data_ptr() + 2))
    with pytest.raises(RuntimeError, match="null operand"):
        _native.call("tgx_paged_attn", *args(q=None))
    p.pages_per_seq = 4000
    p.page_size = 16
    _native.call("tgx_paged_attn_workspace", ctypes.byref(p), 2, 1, 64, 1, ctypes.byref(size))
    assert size.value > 0
    with pytest.raises(RuntimeError, match="workspace"):
        _native.call("tgx_paged_attn", *args())
    p.queries = 0
    with pytest.raises(RuntimeError, match="negative or zero"):
        _native.call("tgx_paged_attn", *args())


def test_gradients_tell_what_ran():
    """Under `strict` a width without CSR kernels is refused when gradients are
    wanted; the record names the CSR kernels, or Torch, where they ran."""
    rng = np.random.default_rng(24)
    table, lengths, pages = relation(rng, [20, 70], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages)
    for D in (64, 24):
        q = torch.randn(2, 2, 3, D, device=DEV).half()
        k, v = torch.randn(2, pages * 16, 2, 1, D, device=DEV).half()
        kernel = Attention()
        call = lambda q: kernel(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.2)
        plain = call(q)
        assert kernel.last_variant.entry_points == ("tgx_paged_attn",)
        leaf = q.clone().requires_grad_(True)
        if D == 24:
            with pytest.raises(RuntimeError, match="strict"):
                call(leaf)
            tg.config.strict = False
            out = call(leaf)
            assert kernel.last_variant.backend == "torch-eager"
            assert not kernel.last_variant.entry_points
            with pytest.raises(NotImplementedError, match="prepared"):
                kernel.prepare(graph=g, src={"key": k, "value": v}, dst={"query": leaf}, scale=0.2)
            tg.config.strict = True
        else:
            out = call(leaf)
            assert kernel.last_variant.entry_points == ("tgx_dot_attn_fwd", "tgx_dot_attn_bwd")
            run = kernel.prepare(graph=g, src={"key": k, "value": v}, dst={"query": leaf},
                                 scale=0.2)
            assert run.variant.pattern == "dot-product"
            assert torch.equal(run(), out) and run().requires_grad
        assert out.requires_grad
        # (A step of 16 bits between two ways of rounding the same sums.)
        assert (out - plain).abs().max() <= 2.0 ** -9 * plain.abs().max()
        with torch.no_grad():
            assert torch.equal(call(leaf), plain)
        assert kernel.last_variant.entry_points == ("tgx_paged_attn",)
        assert torch.equal(call(q), plain)


def test_gradients_where_nobody_sees_a_key():
    """Zeros, without an error under `strict`: how many keys there are is data."""
    lengths = torch.zeros(2, dtype=torch.int32, device=DEV)
    g = tg.Graph.paged(torch.zeros(2, 3, dtype=torch.int32, device=DEV), lengths, page_size=16,
                       num_pages=1)
    leaves = [torch.randn(n, 2, m, 64, device=DEV).half().requires_grad_(True)
              for n, m in ((2, 3), (16, 1), (16, 1))]
    out = Attention()(graph=g, src={"key": leaves[1], "value": leaves[2]},
                      dst={"query": leaves[0]}, scale=0.2)
    assert out.shape == leaves[0].shape and not out.any()
    for grad in torch.autograd.grad(out.sum(), leaves):
        assert not grad.any()


def dual(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("D", [64, 24])
def test_forward_mode_never_loses_a_tangent(D):
    """Refused like the other attention kernels where a kernel would run; carried
    by Torch operations where they do, which `strict` refuses."""
    unpack = torch.autograd.forward_ad.unpack_dual
    rng = np.random.default_rng(23)
    table, lengths, pages = relation(rng, [0, 20, 70], 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(lengths, device=DEV),
                       page_size=16, num_pages=pages, queries=2)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).float()
    args = [mk(6, 2, 3, D), mk(pages * 16, 2, 1, D), mk(pages * 16, 2, 1, D)]
    kernel = Attention()
    call = lambda q, k, v: kernel(graph=g, src={"key": k, "value": v}, dst={"query": q},
                                  scale=0.2)
    call(*args)     # (a warm launch is no way around)
    for i in range(3):
        with torch.autograd.forward_ad.dual_level():
            duals = [dual(t) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(NotImplementedError if D == 64 else RuntimeError):
                call(*duals)
            if D == 24:
                tg.config.strict = False
                got = unpack(call(*duals)).tangent
                assert got is not None and kernel.last_variant.backend == "torch-eager"
        if D == 24:
            up, down = ([t + h if j == i else t for j, t in enumerate(x.double().cpu()
                         for x in args)] for h in (1e-5, -1e-5))
            host = tg.Graph.paged(torch.tensor(table), torch.tensor(lengths), page_size=16,
                                  num_pages=pages, queries=2)
            f = lambda q, k, v: Attention()(graph=host, src={"key": k, "value": v},
                                            dst={"query": q}, scale=0.2)
            exp = (f(*up) - f(*down)) / 2e-5
            # (As in the gradients' test: 1e-5 of the largest value in 32 bits.)
            assert (got.double().cpu() - exp).abs().max() <= 1e-5 * max(1.0, exp.abs().max())
            tg.config.strict = True


def test_append_refuses_forward_mode():
    """The caches would lose the tangent."""
    g = tg.Graph.paged(torch.arange(4, dtype=torch.int32, device=DEV)[None],
                       torch.tensor([9], dtype=torch.int32, device=DEV), page_size=16, num_pages=4)
    args = [torch.zeros(n, 2, 8, device=DEV) for n in (64, 1, 64, 1)]
    sums = torch.zeros(4, 2, 8, device=DEV)
    for i in range(4):
        with torch.autograd.forward_ad.dual_level():
            duals = [dual(t) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(NotImplementedError, match="detach"):
                g.append(*duals, page_sums=sums)
    g.append(*args, page_sums=sums)


def test_strict_refuses_torch_operations_on_the_gpu():
    g = tg.Graph.paged(torch.arange(4, dtype=torch.int32, device=DEV)[None],
                       torch.tensor([40], dtype=torch.int32, device=DEV), page_size=16,
                       num_pages=4)
    mk = lambda n: torch.randn(n, 2, 8, device=DEV, dtype=torch.float64)
    kc, k, vc, v, sums = mk(64), mk(1), mk(64), mk(1), torch.randn(4, 2, 8, device=DEV)
    before = kc.clone()
    with pytest.raises(RuntimeError, match="strict"):
        g.append(kc, k, vc, v)
    assert torch.equal(kc, before)
    with pytest.raises(RuntimeError, match="strict"):
        g.select_pages(k, sums, 2)
    tg.config.strict = False
    g.append(kc, k, vc, v)
    assert torch.equal(kc[39], k[0]) and torch.equal(vc[39], v[0])
    chosen = g.select_pages(k, sums, 2)
    exp, held = want.select(np.arange(4)[None], [40], 16, 4, 1, f64(k)[:, :, None], f64(sums), 2)
    assert np.array_equal(chosen.page_table.cpu().numpy(), exp)
    assert np.array_equal(chosen.lengths.cpu().numpy(), held)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("queries", [1, 5, 12, 30])
@pytest.mark.parametrize("gap", [17.0, 18.0, 20.0])
def test_small_weights_of_many_keys_add_up(gap, queries, D):
    """One key far above the rest whose value is 0: the output is the rest's
    weights, each of them below half a step of fp16 relative to the largest."""
    n = 200
    g = tg.Graph.paged(torch.arange(13, dtype=torch.int32, device=DEV)[None],
                       torch.tensor([n], dtype=torch.int32, device=DEV), page_size=16,
                       num_pages=13, queries=queries)
    for dtype in (torch.float16, torch.bfloat16):
        q = torch.zeros(queries, 1, 4, D, device=DEV, dtype=dtype)
        k, v = torch.zeros(2, 208, 1, 1, D, device=DEV, dtype=dtype)
        q[..., 0] = 1.0
        k[0, ..., 0] = gap
        v[1:] = 32768.0
        out = f64(Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=1.0))
        seen = (n - np.arange(queries - 1, -1, -1))[:, None, None, None] - 1
        exp = 32768.0 * seen * np.exp(-gap) / (1 + seen * np.exp(-gap))
        # Half a step of the output and as much for the weights: e^-20 = 2^-28.9 in parts
        # that are off by 2^-39 at most, 2^-10.1 of it; a step where it is smallest.
        step = 2.0 ** (-10 if dtype == torch.float16 else -8)
        assert (np.abs(out - exp) <= 1.5 * step * exp).all(), (out / exp).min()


def test_small_weights_of_a_long_sequence_add_up():
    """131072 keys, one of them far above the rest, for sequences enough that
    each is one piece."""
    n, B = 131072, 600
    table = torch.arange(n // 64, dtype=torch.int32, device=DEV).expand(B, -1)
    g = tg.Graph.paged(table, torch.full((B,), n, dtype=torch.int32, device=DEV), page_size=64,
                       num_pages=n // 64)
    q = torch.zeros(B, 1, 1, 32, device=DEV, dtype=torch.float16)
    k, v = torch.zeros(2, n, 1, 1, 32, device=DEV, dtype=torch.float16)
    q[..., 0] = 1.0
    v.fill_(1.0)
    for gap in (17.40625, 18.0):
        for first in (1.0, 0.0, -1.0):
            k[0, ..., 0], v[0] = gap, first
            out = f64(Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q},
                                  scale=1.0))
            rest = (n - 1) * np.exp(-gap)
            exp = (first + rest) / (1 + rest)
            # A step of the output, and of each weight 2^-11.
            assert np.abs(out - exp).max() <= 2.0 ** -10 * abs(exp) + 2.0 ** -11 * rest


def tight(lengths, size, heads, group, D, dtype, queries=1, seed=21):
    """An attention against the formula, by each row's own weights."""
    print(f"tight {dtype} D={D} heads={heads} group={group} queries={queries} "
          f"lengths={lengths[:6]}", flush=True)
    rng = np.random.default_rng(seed)
    table, length, pages = relation(rng, lengths, size)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(length, device=DEV),
                       page_size=size, num_pages=pages, queries=queries)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(TYPES[dtype])
    q = mk(len(lengths) * queries, heads, group, D)
    k, v = mk(pages * size, heads, D), mk(pages * size, heads, D)
    out = Attention()(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]},
                      dst={"query": q}, scale=D ** -0.5)
    args = (table, length, size, pages, queries, f64(q), f64(k), f64(v), D ** -0.5)
    tiles = dtype != "f32" and D in (32, 64, 128)
    err = np.abs(f64(out) - want.attention(*args))
    lim = want.attention_bound(*args, dtype, tiles)
    assert (err <= lim).all(), f"{(err / lim).max():.2f} of the bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries,group", [(4, 4), (5, 4), (12, 5), (17, 4), (40, 4)])
def test_accuracy_does_not_depend_on_how_many_ask(queries, group, dtype):
    for D in (64, 128):
        tight([700, 90, 33], 16, 2, group, D, dtype, queries=queries)


@pytest.mark.parametrize("queries", [1, 6, 12, 30])
def test_infinite_values_of_small_weights(queries):
    """An Inf of a key whose weight is below fp16's numbers is an Inf."""
    g = tg.Graph.paged(torch.arange(13, dtype=torch.int32, device=DEV)[None],
                       torch.tensor([200], dtype=torch.int32, device=DEV), page_size=16,
                       num_pages=13, queries=queries)
    q = torch.zeros(queries, 1, 4, 64, device=DEV, dtype=torch.float16)
    k, v = torch.zeros(2, 208, 1, 1, 64, device=DEV, dtype=torch.float16)
    q[..., 0], k[0, ..., 0] = 1.0, 40.0
    v[100, ..., 5], v[101, ..., 7] = float("inf"), float("-inf")
    out = f64(Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=1.0))
    assert np.isposinf(out[..., 5]).all() and np.isneginf(out[..., 7]).all()
    assert np.isfinite(np.delete(out, (5, 7), axis=-1)).all()


def test_more_queries_than_a_launch_has_workgroups():
    """17 * 2^20 queries of one key head: tiles of 128 of them."""
    queries, group = 1 << 20, 17
    g = tg.Graph.paged(torch.arange(13, dtype=torch.int32, device=DEV)[None],
                       torch.tensor([40], dtype=torch.int32, device=DEV), page_size=16,
                       num_pages=13, queries=queries)
    q = torch.randn(1, 1, group, 32, device=DEV).half().expand(queries, -1, -1, -1)
    k, v = torch.randn(2, 208, 1, 1, 32, device=DEV).half()
    kernel = Attention()
    out = kernel(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.2)
    assert kernel.last_variant.pattern == "paged-attention"
    assert not out[:-40].any()
    few = tg.Graph.paged(g.page_table, g.lengths, page_size=16, num_pages=13, queries=40)
    same = Attention()(graph=few, src={"key": k, "value": v}, dst={"query": q[:40]}, scale=0.2)
    assert torch.equal(out[-40:], same)


def test_a_cache_of_one_slot_whose_stride_is_odd():
    """The stride of a dimension of one element moves nothing."""
    g = tg.Graph.paged(torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                       torch.ones(1, dtype=torch.int32, device=DEV), page_size=1, num_pages=1)
    k = torch.randn(3, 129, device=DEV).half()[:, :128].view(3, 2, 64)[:1]
    q = torch.randn(1, 2, 64, device=DEV).half()
    out = Attention()(graph=g, src={"key": k, "value": k}, dst={"query": q}, scale=1.0)
    assert torch.equal(out, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,D", [([20000], 128), ([9000, 1, 0, 300, 4111], 64),
                                       ([3000] * 12, 128), ([5000], 32), ([2000, 77], 80)])
def test_long_lengths_to_the_last_rounding(lengths, D, dtype):
    tight(lengths, 16, 2, 4, D, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,group,queries,D", [
    ([20001], 1, 4, 1, 128), ([1, 0, 640, 9001], 2, 4, 3, 64), ([3000] * 40, 2, 1, 1, 32),
    ([2100, 5], 1, 8, 4, 128), ([2100, 5], 1, 8, 7, 64), ([2100, 5, 130], 1, 8, 20, 128),
    ([777, 3000], 2, 3, 1, 96)])
def test_every_key_counts_once(lengths, heads, group, queries, D, dtype):
    """All scores equal: a row is the mean of the values it sees.  Column d holds
    a one for every D-th key of a window, so n times the row is the number of
    those it sees: at most 64, off by at most 64 * 2^-8 = 1/4 and never by one."""
    print(f"count {dtype} {lengths[:4]} queries={queries} D={D}", flush=True)
    rng = np.random.default_rng(22)
    table, length, pages = relation(rng, lengths, 16)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(length, device=DEV),
                       page_size=16, num_pages=pages, queries=queries)
    q = torch.zeros(len(lengths) * queries, heads, group, D, device=DEV, dtype=TYPES[dtype])
    k = torch.randn(pages * 16, heads, 1, D, device=DEV).to(TYPES[dtype])
    kernel = Attention()
    for start in range(0, max(lengths), 64 * D):
        v = np.zeros((pages * 16, D))
        exp = np.zeros((len(lengths), queries, D))
        for b, n in enumerate(lengths):
            at, _ = want.slots(table[b], n, 16, pages)
            for j in range(start, min(n, start + 64 * D)):
                v[at[j], j % D] = 1.0
                exp[b, max(j - (n - queries), 0):, j % D] += 1.0
        values = torch.tensor(v, device=DEV).to(TYPES[dtype])[:, None, None].expand(
            -1, heads, 1, D).contiguous()
        out = kernel(graph=g, src={"key": k, "value": values}, dst={"query": q}, scale=1.0)
        seen = np.maximum(np.asarray(lengths)[:, None] - np.arange(queries - 1, -1, -1), 0)
        got = f64(out).reshape(len(lengths), queries, heads * group, D)
        got = got * seen[:, :, None, None]
        assert np.array_equal(np.rint(got), np.broadcast_to(exp[:, :, None], got.shape))
