"""Attention of packed sequences over a window on the HIP tiles, forward and backward,
against the formulas in float64."""

import numpy as np
import pytest
import torch

import tiga as tg

import scaled_reference as want

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# Results below the type's normal numbers, and P and dS below them, round in absolute
# steps: of the smallest number, and of each of what is added up.
TINY = {"bf16": 2.0 ** -133, "f16": 2.0 ** -25}


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


def packed(lengths, dtype=torch.int32):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=dtype, device=DEV)


def inputs(rng, lengths, heads, group, D, dtype):
    n = sum(lengths)
    mk = lambda *s: torch.tensor(rng.standard_normal(s), device=DEV).to(TYPES[dtype])
    return mk(n, heads, group, D), mk(n, heads, 1, D), mk(n, heads, 1, D), mk(n, heads, group, D)


def run(graph, q, k, v, d, scale):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    kernel = Attention()
    out = kernel(graph=graph, src={"key": leaves[1], "value": leaves[2]}, dst={"query": leaves[0]},
                 scale=scale)
    assert kernel.last_variant.pattern == "window-attention"
    return [out, *torch.autograd.grad(out, leaves, d)]


def bounded(got, lengths, q, k, v, d, scale, window, sinks, dtype, rows=None):
    """`rows`: what of (out, dq, dk, dv) has to hold, all of it without."""
    one = lambda t: f64(t)[:, :, 0]
    exp, lim = want.window_attention(lengths, f64(q), one(k), one(v), scale, window, sinks, f64(d),
                                     HALF[dtype])
    for i, (a, b, e) in enumerate(zip(got, exp, lim)):
        assert a.dtype == TYPES[dtype]
        a = f64(a).reshape(b.shape)
        e = e + TINY[dtype] * (4 + max(lengths, default=0) * q.shape[2] * 8)
        if rows is not None:
            a, b, e = a[rows[i]], b[rows[i]], e[rows[i]]
        err = np.abs(a - b)
        assert (err <= e).all(), (f"result {i}: error {np.nanmax(err):.3e}, "
                                  f"{np.nanmax(err / e):.2f} of the bound")


def check(lengths, heads, group, D, dtype, window, sinks, seed=0, scale=None):
    print(f"{dtype} D={D} heads={heads} group={group} window={window} sinks={sinks} "
          f"lengths={lengths[:6]}", flush=True)
    rng = np.random.default_rng(seed)
    q, k, v, d = inputs(rng, lengths, heads, group, D, dtype)
    g = tg.Graph.cu_seqlens(packed(lengths), window=window, sinks=sinks)
    scale = D ** -0.5 if scale is None else scale
    got = run(g, q, k, v, d, scale)
    bounded(got, lengths, q, k, v, d, scale, window, sinks, dtype)
    return g, q, k, v, d, got


EDGES = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (17, 0), (64, 4), (65, 64), (100, 130)])
def test_lengths_around_tiles(dtype, D, window, sinks):
    check(EDGES, 2, 1, D, dtype, window, sinks)


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 3), (1, 4), (2, 5), (1, 8), (1, 17),
                                         (1, 64), (1, 128)])
@pytest.mark.parametrize("window,sinks", [(20, 0), (70, 3)])
def test_head_groups(heads, group, window, sinks):
    check([1, 90, 0, 150], heads, group, 64, "bf16", window, sinks)
    check([1, 90, 0, 150], heads, group, 128, "f16", window, sinks)


@pytest.mark.parametrize("window,sinks", [(100, 0), (100, 5), (300, 70), (1000, 1), (2**31 - 1, 0),
                                          (5, 2**31 - 1)])
def test_long_sequences(window, sinks):
    check([1700, 5, 900], 1, 2, 64, "f16", window, sinks)
    check([1500], 2, 1, 128, "bf16", window, sinks)


def test_first_tokens_in_many_pieces():
    """A tile of first tokens whose rows are cut into pieces and joined."""
    g, *_ = check([2500], 1, 4, 64, "bf16", 40, 66)
    assert g._window_tasks(1, 1, 4)[3] > 4
    check([2500], 1, 4, 32, "f16", 10, 1)


@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0])
def test_scales(scale):
    check([100, 70], 1, 3, 64, "bf16", 50, 2, scale=scale)
    check([100, 70], 1, 3, 32, "f16", 50, 2, scale=scale)


def test_triangular_and_field_shapes():
    rng = np.random.default_rng(2)
    q, k, v, d = inputs(rng, [200], 3, 1, 64, "bf16")
    g = tg.Graph.triangular(200, device="cuda", window=30, sinks=2)
    whole = run(g, q, k, v, d, 0.125)
    bounded(whole, [200], q, k, v, d, 0.125, 30, 2, "bf16")
    flat = run(g, q[:, :, 0], k[:, :, 0], v[:, :, 0], d[:, :, 0], 0.125)
    assert all(torch.equal(a.flatten(), b.flatten()) for a, b in zip(whole, flat))
    # One key head under several query heads.
    q, k, v, d = inputs(rng, [200], 1, 3, 64, "bf16")
    a = run(g, q, k, v, d, 0.125)
    b = run(g, q[:, 0], k[:, 0], v[:, 0], d[:, 0], 0.125)
    assert all(torch.equal(x.flatten(), y.flatten()) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_window_past_everything_is_causal_attention(dtype):
    """Within the bounds of both: the dense tiles over the same relation."""
    rng = np.random.default_rng(3)
    lengths = [300, 64, 1]
    q, k, v, d = inputs(rng, lengths, 2, 1, 64, dtype)
    got = run(tg.Graph.cu_seqlens(packed(lengths), window=300), q, k, v, d, 0.125)
    leaves = [t[:, :, 0].detach().requires_grad_(True) for t in (q, k, v)]
    out = Attention()(graph=tg.Graph.cu_seqlens(packed(lengths)),
                      src={"key": leaves[1], "value": leaves[2]}, dst={"query": leaves[0]},
                      scale=0.125)
    other = [out, *torch.autograd.grad(out, leaves, d[:, :, 0])]
    for res in (got, other):
        bounded(res, lengths, q, k, v, d, 0.125, 300, 0, dtype)


def test_strides_and_starts():
    """Fields of one projection, heads before tokens, starts on no 16 bytes, an expanded
    gradient."""
    rng = np.random.default_rng(4)
    lengths, window, sinks = [150, 20], 40, 3
    n, heads, group, D = 170, 2, 3, 64
    q, k, v, d = inputs(rng, lengths, heads, group, D, "f16")
    g = tg.Graph.cu_seqlens(packed(lengths), window=window, sinks=sinks)
    exp = run(g, q, k, v, d, 0.125)
    row = torch.zeros(n, heads, group + 2, D, dtype=q.dtype, device=DEV)
    row[:, :, :group], row[:, :, group:group + 1], row[:, :, group + 1:] = q, k, v
    views = [
        (row[:, :, :group], row[:, :, group:group + 1], row[:, :, group + 1:]),
        tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)),
        tuple(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in (q, k, v)),
        tuple(t.mT.contiguous().mT for t in (q, k, v)),
    ]
    for fields in views:
        got = run(g, *fields, d, 0.125)
        assert all(torch.equal(a, b) for a, b in zip(exp, got))
    same = d[:1, :1, :1, :1].expand(d.shape)
    assert all(torch.equal(a, b) for a, b in zip(run(g, q, k, v, same, 0.125),
                                                 run(g, q, k, v, same.contiguous(), 0.125)))
    # Shared keys and values of all tokens' heads: an expanded field.
    shared = k[:, :1].expand(n, heads, 1, D)
    a = run(g, q, shared, shared, d, 0.125)
    b = run(g, q, shared.contiguous(), shared.contiguous(), d, 0.125)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,group", [(64, 1), (128, 3)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_what_is_not_seen_never_arrives(dtype, D, group, bad):
    """A key, value, query or output gradient of no number reaches the rows and keys that
    its pairs reach, and no others."""
    rng = np.random.default_rng(5)
    lengths, window, sinks, heads = [300, 90], 70, 2, 2
    n, at = 390, 140                 # in the first sequence, seen by 140 .. 209
    g = tg.Graph.cu_seqlens(packed(lengths), window=window, sinks=sinks)
    q, k, v, d = inputs(rng, lengths, heads, group, D, dtype)
    tokens = np.arange(n)
    by = (tokens >= at) & (tokens < at + window)          # rows that see key `at`
    of = ((tokens <= at) & (tokens > at - window)) | (tokens < sinks)   # keys that row `at` sees
    # Keys that a row which sees key `at` sees, within its sequence.
    near = (((tokens > at - window) & (tokens < at + window)) | (tokens < sinks))
    scale = D ** -0.5
    for i, rows_off, keys_off in ((0, tokens == at, of), (1, by, near), (2, by, near),
                                  (3, None, None)):
        x = [t.clone() for t in (q, k, v, d)]
        x[i][at] = bad
        got = run(g, *x, scale)
        if i == 3:                   # the output is the same; dq of the row, dk and dv of its keys
            ok = [slice(None), tokens != at, ~of, ~of]
        else:
            ok = [~rows_off, ~rows_off, ~keys_off, ~keys_off]
        bounded(got, lengths, q, k, v, d, scale, window, sinks, dtype, ok)
        if i != 3:
            assert not torch.isfinite(got[0][torch.tensor(rows_off, device=DEV)]).all()


def test_the_same_bits_every_time():
    g, q, k, v, d, got = check([900, 300], 2, 4, 64, "bf16", 100, 5)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, run(g, q, k, v, d, 64 ** -0.5)))


def test_forward_without_gradients_and_second_derivatives():
    rng = np.random.default_rng(6)
    q, k, v, d = inputs(rng, [100], 1, 2, 64, "bf16")
    g = tg.Graph.cu_seqlens(packed([100]), window=30)
    with torch.no_grad():
        out = Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.1)
    assert torch.equal(out, run(g, q, k, v, d, 0.1)[0]) and not out.requires_grad
    with torch.inference_mode():
        assert torch.equal(out, Attention()(graph=g, src={"key": k, "value": v},
                                            dst={"query": q}, scale=0.1))
    leaf = q.clone().requires_grad_(True)
    out = Attention()(graph=g, src={"key": k, "value": v}, dst={"query": leaf}, scale=0.1)
    (grad,) = torch.autograd.grad(out, leaf, d, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, d)
        with pytest.raises(NotImplementedError):
            Attention()(graph=g, src={"key": k, "value": v}, dst={"query": dual}, scale=0.1)
    # Only some of the gradients.
    leaf = v.clone().requires_grad_(True)
    out = Attention()(graph=g, src={"key": k, "value": leaf}, dst={"query": q}, scale=0.1)
    assert torch.equal(torch.autograd.grad(out, leaf, d)[0], run(g, q, k, v, d, 0.1)[3])


def test_captured_training_steps():
    """Forward and backward in one captured graph, replayed between eager steps."""
    rng = np.random.default_rng(7)
    lengths = [260, 1, 90]
    g = tg.Graph.cu_seqlens(packed(lengths), window=50, sinks=2)
    q, k, v, d = inputs(rng, lengths, 2, 2, 64, "bf16")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(g, q, k, v, d, 0.125)
    torch.cuda.current_stream().wait_stream(stream)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        outs = run(g, q, k, v, d, 0.125)
    for i in range(4):
        for t in (q, k, v, d):
            t.copy_(torch.randn(t.shape, device=DEV))
        captured.replay()
        torch.cuda.synchronize()
        eager = run(g, q, k, v, d, 0.125)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_other_shapes_go_through_the_edges():
    """Widths and types that no tile takes, refused when strict."""
    rng = np.random.default_rng(8)
    n, window, sinks = 60, 9, 2
    g = tg.Graph.cu_seqlens(packed([60]), window=window, sinks=sinks)
    q, d = rng.standard_normal((2, n, 1, 2, 40))
    k, v = rng.standard_normal((2, n, 1, 40))
    t = lambda x: torch.tensor(x, device=DEV, dtype=torch.float32)
    call = lambda: Attention()(graph=g, src={"key": t(k)[:, :, None], "value": t(v)[:, :, None]},
                               dst={"query": t(q)}, scale=0.2)
    with pytest.raises(RuntimeError, match="strict"):
        call()
    tg.config.strict = False
    exp, lim = want.window_attention([n], q, k, v, 0.2, window, sinks, half=2.0 ** -24)
    assert (np.abs(f64(call()) - exp) <= 4 * lim + 1e-6 * np.abs(exp)).all()


def test_prompt_then_steps():
    """A prompt through the tiles, its keys and values into a cache, and the next token
    over the same window of it: the last row of a prompt that is one token longer."""
    rng = np.random.default_rng(9)
    heads, group, D, window, sinks, n, size = 2, 4, 64, 50, 3, 200, 16
    q, k, v, d = inputs(rng, [n], heads, group, D, "bf16")
    whole = tg.Graph.cu_seqlens(packed([n]), window=window, sinks=sinks)
    pages = -(-n // size)
    table = torch.tensor(rng.permutation(pages)[None], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    kc, vc = (torch.zeros(pages * size, heads, D, dtype=q.dtype, device=DEV) for _ in range(2))
    make = lambda queries: tg.Graph.paged(table, lengths, page_size=size, num_pages=pages,
                                          queries=queries, window=window, sinks=sinks)
    make(n).append(kc, k[:, :, 0], vc, v[:, :, 0])
    call = lambda g, q, k, v: Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q},
                                          scale=0.125)
    full = call(whole, q, k, v)
    _, lim = want.window_attention([n], f64(q), f64(k)[:, :, 0], f64(v)[:, :, 0], 0.125, window,
                                   sinks, half=HALF["bf16"])
    for queries in (1, 7, n):
        step = call(make(queries), q[-queries:], kc[:, :, None], vc[:, :, None])
        assert (np.abs(f64(step) - f64(full[-queries:])) <= 2 * lim[-queries:]).all()


def test_leaves_without_gradients_pay_for_no_backward():
    """Under no_grad the output is the same and nothing else of its size is kept, also for
    inputs that require gradients; a step with gradients on the same relation follows."""
    rng = np.random.default_rng(10)
    lengths = [4000]
    q, k, v, d = inputs(rng, lengths, 4, 4, 128, "bf16")
    leaf = q.clone().requires_grad_(True)
    g = tg.Graph.cu_seqlens(packed(lengths), window=30, sinks=2)
    call = lambda: Attention()(graph=g, src={"key": k, "value": v}, dst={"query": leaf}, scale=0.1)
    with torch.no_grad():
        call()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = call()
        grown = torch.cuda.max_memory_allocated() - before
    size = out.numel() * out.element_size()
    assert not out.requires_grad and size <= grown < 1.5 * size
    got = run(g, q, k, v, d, 0.1)
    assert torch.equal(got[0], out)
    assert all(torch.equal(a, b) for a, b in zip(got, run(
        tg.Graph.cu_seqlens(packed(lengths), window=30, sinks=2), q, k, v, d, 0.1)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_row_sums_take_the_output_to_twice_16_bits(dtype, D):
    """The root mean square error of dQ and dK at a window of 2, in that of the exact ones
    rounded once.  There delta's error weighs most: the kernels' roundings (weights, dS
    and the result, each to 16 bits), applied in float64 to such inputs, give 1.5 for
    every type and width with delta from both parts of the output, 2.2 with the first part
    alone, 2.7 with another row's second part and 3.6 with its sign turned."""
    rng = np.random.default_rng(11)
    lengths, heads, group = [500, 100], 2, 2
    q, k, v, d = inputs(rng, lengths, heads, group, D, dtype)
    g = tg.Graph.cu_seqlens(packed(lengths), window=2)
    got = run(g, q, k, v, d, D ** -0.5)
    one = lambda t: f64(t)[:, :, 0]
    exp, _ = want.window_attention(lengths, f64(q), one(k), one(v), D ** -0.5, 2, 0, f64(d),
                                   HALF[dtype])
    for i in (1, 2):
        once = torch.tensor(exp[i]).to(TYPES[dtype]).double().numpy()
        rms = lambda x: np.sqrt(np.square(x - exp[i]).mean())
        assert rms(f64(got[i]).reshape(exp[i].shape)) < 1.8 * rms(once)


@pytest.mark.parametrize("heads,group", [(1, 128), (128, 1)])
def test_offsets_past_32_bits(heads, group):
    """Queries, or keys and values too, of more than 2^31 elements: the first and the last
    sequence have the bits that they have alone."""
    D, lengths, window = 128, [300, 131000, 500], 16
    n = sum(lengths)
    assert n * heads * group * D > 2 ** 31
    gen = torch.Generator(device=DEV).manual_seed(12)
    mk = lambda *s: torch.randn(s, device=DEV, dtype=torch.bfloat16, generator=gen)
    q, d = mk(n, heads, group, D), mk(n, heads, group, D)
    k, v = mk(n, heads, 1, D), mk(n, heads, 1, D)
    got = run(tg.Graph.cu_seqlens(packed(lengths), window=window), q, k, v, d, 0.1)
    for first, length in ((0, 300), (131300, 500)):
        rows = slice(first, first + length)
        alone = run(tg.Graph.cu_seqlens(packed([length]), window=window), q[rows], k[rows], v[rows],
                    d[rows], 0.1)
        assert all(torch.equal(a[rows], b) for a, b in zip(got, alone))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,group", [(32, 2), (64, 1), (128, 3)])
def test_a_key_of_minus_infinity(dtype, D, group):
    """A seen key with -Inf in a column where all queries are positive has a score of -Inf
    and no weight: all is as with a key far down, but for 0 * -Inf in that column of dQ, in
    tiles that are masked and in those that are not."""
    rng = np.random.default_rng(13)
    lengths, window, sinks, heads, at, column = [400, 90], 170, 2, 2, 140, 5
    g = tg.Graph.cu_seqlens(packed(lengths), window=window, sinks=sinks)
    q, k, v, d = inputs(rng, lengths, heads, group, D, dtype)
    q[..., column] = q[..., column].abs() + 1
    low = k.clone()
    k[at, ..., column], low[at, ..., column] = -np.inf, -3e4     # (3e4 D^-1/2 > 2000)
    got, exp = run(g, q, k, v, d, D ** -0.5), run(g, q, low, v, d, D ** -0.5)
    sees = slice(at, at + window)
    assert got[1][sees, ..., column].isnan().all()
    got[1][sees, ..., column] = exp[1][sees, ..., column]
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, exp))


def test_small_fp16_weights_are_not_lost():
    """Keys of weight e^-18.4, 2^-26.6 of the first one's and below fp16's smallest
    number: what the rows have of their values, and they of the rows' gradients."""
    rng = np.random.default_rng(14)
    n, D = 30000, 32
    part = lambda *s: rng.uniform(0.5, 1.5, s)
    q, k = np.zeros((n, 1, 1, D)), np.zeros((n, 1, 1, D))
    v, d = part(n, 1, 1, D), part(n, 1, 1, D)
    q[..., 0], k[1:, ..., 0], v[0] = 1, -18.40625, 0
    t = [torch.tensor(x, device=DEV).to(torch.float16) for x in (q, k, v, d)]
    got = run(tg.Graph.triangular(n, device="cuda", window=n), *t, 1.0)
    weight = np.exp(-18.40625)
    total = 1 + weight * np.arange(n)
    values, grads = f64(t[2])[:, 0, 0], f64(t[3])[:, 0, 0]
    out = weight * np.cumsum(values, 0) / total[:, None]
    dv = weight * np.cumsum((grads / total[:, None])[::-1], 0)[::-1]
    # Half a step of a weight and of the result (or of the smallest number), fp32 sums 32
    # keys at a time, and scores of 27 in 32 bits.
    rel = 2 * HALF["f16"] + 2 * 2.0 ** -24 * (n / 32 + 64) + 2.0 ** -18
    assert (np.abs(f64(got[0])[:, 0, 0] - out) <= rel * out + 2.0 ** -25).all()
    assert (np.abs(f64(got[3])[1:, 0, 0] - dv[1:]) <= rel * dv[1:] + 2.0 ** -25).all()
    assert out[-1].min() > 100 * 2.0 ** -25 and dv[1].min() > 100 * 2.0 ** -25


@pytest.mark.parametrize("dtype", TYPES)
def test_sinks_past_everything_are_causal_attention(dtype):
    """All tokens as sinks: every key tile is cut into pieces, whose size goes by all the
    work; over a window of all tokens none is.  The products are the same."""
    rng = np.random.default_rng(15)
    n, heads, group, D = 6000, 4, 4, 64
    q, k, v, d = inputs(rng, [n], heads, group, D, dtype)
    cut, whole = (tg.Graph.cu_seqlens(packed([n]), window=w, sinks=s) for w, s in ((1, n), (n, 0)))
    got, exp = (run(g, q, k, v, d, 0.125) for g in (cut, whole))
    assert 1000 < cut._window_tasks(1, heads, group)[3] <= 1.5 * 2048
    assert whole._window_tasks(1, heads, group)[3] == 0
    assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
    for a, b in zip(got[2:], exp[2:]):
        a, b = a.float(), b.float()
        # fp32 sums of up to 24000 products in another order, each of them less than the
        # largest sum: then a rounding of each.
        lim = 2 * HALF[dtype] * b.abs() + 2 * 2.0 ** -24 * n * group * b.abs().max()
        assert ((a - b).abs() <= lim).all()
