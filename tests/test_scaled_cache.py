"""tiga.BlockScaled, append to it and read from it, and attention over it, on host
tensors against the formulas in float64; and what they refuse."""

import ctypes

import numpy as np
import pytest
import torch

import tiga as tg
from tiga import _native

import scaled_reference as want

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
SIZE, PAGES, BLOCK = 8, 12, 4
TABLE = torch.tensor([[3, 0, 7], [5, -1, 9], [1, 2, 12], [4, 6, 8]], dtype=torch.int32)
# (empty, ending on a page, behind a page that is not there, more than the table holds)
LENGTHS = torch.tensor([0, 16, 21, 40], dtype=torch.int32)


class Attention(tg.MessagePassing):
    reducer = tg.online_softmax()

    def edge(self, src, dst, edge, scale):
        return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)


class Sum(tg.MessagePassing):
    reducer = tg.sum()

    def edge(self, src, dst, edge):
        return src.x


def graph(queries=1, lengths=LENGTHS, **more):
    return tg.Graph.paged(TABLE, lengths, page_size=SIZE, num_pages=PAGES, queries=queries, **more)


def cache(rng, code, heads=2, D=8, slots=PAGES * SIZE, block=BLOCK):
    """A cache whose codes are what an append would have left, and codes as numbers."""
    scales = 2.0 ** rng.integers(-9, 3, size=(slots // block, heads))
    x = rng.uniform(-want.LARGEST[code], want.LARGEST[code], (slots, heads, D))
    codes = want.rounded(x, code)
    return tg.BlockScaled(torch.tensor(codes, dtype=torch.float32).to(CODES[code]),
                          torch.tensor(scales, dtype=torch.float32), block=block), codes, scales


f64 = lambda t: t.detach().double().numpy()


@pytest.mark.parametrize("code", CODES)
def test_dequantize_and_views(code):
    rng = np.random.default_rng(0)
    c, codes, scales = cache(rng, code)
    exp = want.values(codes, scales, BLOCK)
    assert np.array_equal(f64(c.dequantize()), exp)
    assert np.array_equal(f64(c.dequantize(torch.float64)), exp)
    assert c.dequantize(torch.bfloat16).dtype == torch.bfloat16
    assert np.array_equal(f64(c.grouped().dequantize()), exp[:, :, None])
    assert np.array_equal(f64(c.per_head().dequantize()), exp.reshape(-1, 1, 8))
    assert c.per_head().codes.data_ptr() == c.codes.data_ptr()
    assert c.shape == (96, 2, 8) and c.ndim == 3 and c.dtype == CODES[code]
    assert code[-4:] in repr(c).replace("float8_e4m3fn", "e4m3") and "block=4" in repr(c)
    empty = tg.BlockScaled.zeros(16, 2, 8, block=8, dtype=CODES[code])
    assert not empty.dequantize().any() and empty.scales.shape == (2, 2)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("queries", [1, 3, 11, 30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_append_and_read_match_the_formula(code, queries, dtype):
    rng = np.random.default_rng(queries)
    lengths = torch.tensor([1, 16, 21, 40], dtype=torch.int32)
    g = graph(queries, lengths)
    (kc, kn, ks), (vc, vn, vs) = cache(rng, code), cache(rng, code)
    big = np.exp(rng.standard_normal((4 * queries, 2, 1)) * 3)
    k, v = (torch.tensor(rng.standard_normal((4 * queries, 2, 8)) * big).to(dtype)
            for _ in range(2))
    k[0] = 0
    sums = torch.full((PAGES, 2, 8), 7.0)
    g.append(kc, k, vc, v, page_sums=sums)
    args = (TABLE.numpy(), lengths.numpy(), SIZE, PAGES, queries)
    for c, n, s, x in ((kc, kn, ks, k), (vc, vn, vs, v)):
        codes, scales = want.append(*args, n, s, f64(x), code, BLOCK)
        assert np.array_equal(f64(c.codes.float()), codes)
        assert np.array_equal(f64(c.scales), scales)
    rows = want.values(f64(kc.codes.float()), f64(kc.scales), BLOCK)
    exp = want.page_sums(*args, rows, np.full((PAGES, 2, 8), 7.0))
    # Sums of at most 8 values in fp32: 8 roundings of 2^-24 of at most 8 * max.
    assert np.abs(sums.numpy() - exp).max() <= 64 * 2.0 ** -24 * np.abs(exp).max()
    got = g.read(kc, vc, dtype=torch.float32)
    assert np.array_equal(f64(got[0]), want.read(*args, rows))
    assert torch.equal(g.read(kc, vc)[0], got[0].to(torch.bfloat16))
    assert np.array_equal(f64(got[1]), want.read(
        *args, want.values(f64(vc.codes.float()), f64(vc.scales), BLOCK)))


@pytest.mark.parametrize("code", CODES)
def test_the_scale_is_the_smallest_power_of_two(code):
    """Magnitudes at, just below and just above M 2^e, the smallest and the largest."""
    top = want.LARGEST[code]
    amax = [0.0, 2.0 ** -149, 2.0 ** -126, 1.0, top, np.nextafter(np.float32(top), np.float32(999)),
            np.nextafter(np.float32(top), np.float32(0)), top * 2.0 ** -130, 2.0 ** 127,
            np.finfo(np.float32).max]
    g = tg.Graph.paged(torch.arange(len(amax), dtype=torch.int32)[:, None],
                       torch.ones(len(amax), dtype=torch.int32), page_size=1, num_pages=len(amax))
    c = tg.BlockScaled.zeros(len(amax), 1, 8, block=1, dtype=CODES[code])
    x = torch.tensor(np.array(amax, dtype=np.float32))[:, None, None].repeat(1, 1, 8)
    x[:, :, 1:] *= -0.75
    g.append(c, x, tg.BlockScaled.zeros(len(amax), 1, 8, block=1, dtype=CODES[code]), x)
    codes, scales = want.append(
        np.arange(len(amax))[:, None], np.ones(len(amax)), 1, len(amax), 1,
        np.zeros((len(amax), 1, 8)), np.zeros((len(amax), 1)), f64(x), code, 1)
    assert np.array_equal(f64(c.scales), scales)
    assert np.array_equal(f64(c.codes.float()), codes)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_codes_cannot_hold_makes_the_block_nan(code, bad):
    """The block and head that a NaN or an infinity goes to reads back as NaN until it
    is begun again; its neighbours are as they were."""
    rng = np.random.default_rng(3)
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    lengths = torch.tensor([6], dtype=torch.int32)
    g = tg.Graph.paged(table, lengths, page_size=SIZE, num_pages=2, queries=6)
    kc, vc = (tg.BlockScaled.zeros(16, 2, 8, block=BLOCK, dtype=CODES[code]) for _ in range(2))
    k = torch.tensor(rng.standard_normal((6, 2, 8)), dtype=torch.float32)
    k[5, 1, 3] = bad
    g.append(kc, k, vc, k.abs().nan_to_num(0, 0, 0))
    rows = kc.dequantize()
    assert rows[4:6, 1].isnan().all() and not rows[:4].isnan().any() and \
        not rows[4:6, 0].isnan().any() and not vc.dequantize().isnan().any()
    # One token more of the same block, then the block begun again.
    one = tg.Graph.paged(table, lengths, page_size=SIZE, num_pages=2)
    lengths += 1
    fine = torch.ones(1, 2, 8)
    one.append(kc, fine, vc, fine)
    assert kc.dequantize()[4:7, 1].isnan().all() and not kc.dequantize()[4:7, 0].isnan().any()
    lengths.fill_(5)
    one.append(kc, fine, vc, fine)
    assert torch.equal(kc.dequantize()[4], fine[0])


def test_tokens_taken_back_and_written_again():
    """A block whose scale stays keeps its older codes; one that is begun again forgets."""
    table, lengths = torch.tensor([[1, 0]], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    g = tg.Graph.paged(table, lengths, page_size=SIZE, num_pages=2, queries=3)
    one = tg.Graph.paged(table, lengths, page_size=SIZE, num_pages=2)
    kc, vc = (tg.BlockScaled.zeros(16, 1, 8, block=SIZE, dtype=torch.int8) for _ in range(2))
    x = torch.full((3, 1, 8), 100.0)
    g.append(kc, x, vc, x)
    lengths += 1
    one.append(kc, x[:1] * 64, vc, x[:1])                  # rounds the first three again
    assert torch.equal(kc.dequantize()[8:12, 0, 0], torch.tensor([128., 128., 128., 6400.]))
    assert torch.equal(vc.dequantize()[8:12, 0, 0], torch.full((4,), 100.0))
    one.append(kc, x[:1], vc, x[:1])                       # the same position again
    assert torch.equal(kc.dequantize()[8:12, 0, 0], torch.tensor([128., 128., 128., 128.]))
    lengths.fill_(1)
    one.append(kc, x[:1], vc, x[:1])
    assert float(kc.scales[1, 0]) == 1.0 and float(kc.dequantize()[8, 0, 0]) == 100.0


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (5, 2), (1, 0), (100, 3)])
def test_attention_over_the_cache(code, window, sinks):
    rng = np.random.default_rng(5)
    (kc, kn, ks), (vc, vn, vs) = cache(rng, code), cache(rng, code)
    q = rng.standard_normal((12, 2, 3, 8))
    g = graph(3, window=window, sinks=sinks)
    out = Attention()(graph=g, src={"key": kc.grouped(), "value": vc.grouped()},
                      dst={"query": torch.tensor(q)}, scale=0.01)
    exp, _ = want.paged_attention(TABLE.numpy(), LENGTHS.numpy(), SIZE, PAGES, 3, q,
                                  want.values(kn, ks, BLOCK), want.values(vn, vs, BLOCK), 0.01,
                                  window, sinks)
    assert out.dtype == torch.float64
    # 64-bit sums of at most 24 products: far below 1e-12 of values up to 448 * 4.
    assert np.abs(out.numpy() - exp).max() <= 1e-12 * 448 * 4
    half = Attention()(graph=g, src={"key": kc.grouped(), "value": vc.grouped()},
                       dst={"query": torch.tensor(q).to(torch.float16)}, scale=0.01)
    assert half.dtype == torch.float16
    # Another edge function sees the values.
    got = Sum()(graph=g, src={"x": kc}, dst={})
    assert torch.equal(got, Sum()(graph=g, src={"x": kc.dequantize()}, dst={}))
    assert torch.equal(Attention().reference(
        graph=g, src={"key": kc.grouped(), "value": vc.grouped()},
        dst={"query": torch.tensor(q)}, scale=0.01), out)


def test_queries_and_scales_have_gradients():
    rng = np.random.default_rng(6)
    (kc, _, _), (vc, _, _) = cache(rng, "int8"), cache(rng, "int8")
    kc.scales.mul_(2 ** -7).requires_grad_(True)
    q = torch.tensor(rng.standard_normal((4, 2, 3, 8)), requires_grad=True)
    call = lambda q: Attention()(graph=graph(), src={"key": kc.grouped(), "value": vc.grouped()},
                                 dst={"query": q}, scale=0.1)
    call(q).square().sum().backward()
    dense = Attention()(graph=graph(), src={"key": kc.dequantize(torch.float64)[:, :, None],
                                            "value": vc.dequantize(torch.float64)[:, :, None]},
                        dst={"query": q}, scale=0.1)
    want_q, want_s = torch.autograd.grad(dense.square().sum(), (q, kc.scales))
    assert torch.allclose(q.grad, want_q, rtol=1e-12, atol=1e-12)
    assert torch.allclose(kc.scales.grad, want_s, rtol=1e-6) and want_s.abs().max() > 0
    with pytest.raises(NotImplementedError, match="no gradient"):
        graph().read(kc, vc)


def test_what_is_refused():
    codes, scales = torch.zeros(16, 2, 8, dtype=torch.int8), torch.zeros(4, 2)
    for bad, error in ((dict(codes=codes.float()), TypeError), (dict(scales=scales.double()), TypeError),
                       (dict(codes=codes[:15]), ValueError), (dict(scales=scales[:3]), ValueError),
                       (dict(block=0), ValueError), (dict(block=True), ValueError),
                       (dict(tables=0), ValueError), (dict(block=8), ValueError),
                       (dict(codes=codes[0]), ValueError), (dict(codes=[1]), TypeError),
                       (dict(codes=codes.mT.contiguous().mT), ValueError),
                       (dict(codes=codes[:, :, None].expand(-1, -1, 2, -1)), ValueError)):
        with pytest.raises(error):
            tg.BlockScaled(**{**dict(codes=codes, scales=scales, block=4), **bad})
    with pytest.raises(TypeError):
        tg.BlockScaled.zeros(16, 2, 8, block=4, dtype=torch.float32)
    with pytest.raises(ValueError):
        tg.BlockScaled.zeros(15, 2, 8, block=4)
    g = graph()
    kc, vc = (tg.BlockScaled.zeros(PAGES * SIZE, 2, 8, block=4) for _ in range(2))
    x = torch.zeros(4, 2, 8)
    other = tg.BlockScaled.zeros(PAGES * SIZE, 2, 8, block=4, dtype=torch.int8)
    odd = tg.BlockScaled.zeros(PAGES * SIZE, 2, 8, block=6)
    for args in ((kc, x, other, x), (kc, x, vc, x.half()), (kc, x.double(), vc, x.double()),
                 (kc, x, vc.dequantize(), x), (vc.dequantize(), x, vc, x)):
        with pytest.raises(TypeError):
            g.append(*args)
    for args in ((odd, x, odd, x), (kc.grouped(), x, vc.grouped(), x), (kc, x[:3], vc, x[:3]),
                 (kc.per_head(), x, vc.per_head(), x)):
        with pytest.raises(ValueError):
            g.append(*args)
    with pytest.raises(NotImplementedError, match="no gradient"):
        g.append(kc, x.clone().requires_grad_(), vc, x)
    for args, kw, error in (((kc, other), {}, TypeError), ((kc, vc.dequantize()), {}, TypeError),
                            ((kc, vc), dict(dtype=torch.float64), TypeError),
                            ((odd, odd), {}, ValueError),
                            ((tg.BlockScaled.zeros(8, 2, 8, block=4),) * 2, {}, ValueError)):
        with pytest.raises(error):
            g.read(*args, **kw)
    with pytest.raises(TypeError, match="paged"):
        tg.Graph.regular(4, 2).read(kc, vc)
    with pytest.raises(TypeError, match="paged relation"):
        Sum()(graph=tg.Graph.regular(PAGES * SIZE, 2), src={"x": kc}, dst={})
    with pytest.raises(TypeError, match="paged relation"):
        Attention()(graph=g, src={"key": kc.grouped(), "value": vc.grouped()},
                    dst={"query": kc.grouped()}, scale=1.0)
    with pytest.raises(ValueError, match="leading dimension"):
        Sum()(graph=g, src={"x": tg.BlockScaled.zeros(8, 2, 8, block=4)}, dst={})


def test_append_refuses_one_cache_for_keys_and_values():
    """(Each would form the other's older codes again.)"""
    g, x = graph(), torch.ones(4, 2, 8)
    kc, vc = (tg.BlockScaled.zeros(PAGES * SIZE, 2, 8, block=BLOCK) for _ in range(2))
    for other in (kc, tg.BlockScaled(kc.codes, vc.scales, block=BLOCK),
                  tg.BlockScaled(vc.codes, kc.scales, block=BLOCK)):
        with pytest.raises(ValueError, match="share"):
            g.append(kc, x, other, x)
    g.append(kc, x, vc, x)


def test_native_entries_refuse_what_they_do_not_take():
    """Bad arguments come back as a status before anything is launched."""
    p = _native.Paged(None, 0, 0, 0x1000, 2, 1, 3, 8, 12, 1)
    p.page_table_dev = 0x1000
    ref = ctypes.byref(p)
    bytes_ = ctypes.c_size_t()
    one, eight, four = 0x1000, (ctypes.c_int64 * 8)(*[8] * 8), (ctypes.c_int64 * 4)(*[8] * 4)
    nine = (ctypes.c_int64 * 9)(*[16] * 9)

    def view(window=0, sinks=0, code=1, block=4, scales=one):
        return ctypes.byref(_native.PagedView(window, sinks, code, block, scales, scales))

    for v in (view(window=-1), view(sinks=3), view(window=2, sinks=-1), view(code=3),
              view(block=3), view(block=0)):
        with pytest.raises(RuntimeError):
            _native.call("tgx_paged_attn_view_workspace", ref, v, 2, 4, 64, 0, ctypes.byref(bytes_))
    with pytest.raises(RuntimeError):
        _native.call("tgx_paged_attn_view_workspace", ref, None, 2, 4, 64, 0, ctypes.byref(bytes_))
    _native.call("tgx_paged_attn_view_workspace", ref, view(window=3, sinks=1), 2, 4, 64, 0,
                 ctypes.byref(bytes_))
    attn = lambda v, q=one, k=one, s=nine: _native.call(
        "tgx_paged_attn_view", ref, v, q, k, one, s, 1.0, one, 2, 4, 64, 0, None, 0, None)
    for kw in (dict(q=None), dict(k=None), dict(k=one + 4), dict(s=(ctypes.c_int64 * 9)(*[4] * 9))):
        with pytest.raises(RuntimeError):
            attn(view(), **kw)
    with pytest.raises(RuntimeError, match="scales"):
        attn(view(scales=None))
    with pytest.raises(RuntimeError, match="16 bytes"):
        attn(view(code=0), k=one + 8)
    append = lambda k=one, x=one, s=eight, D=64, dtype=0, code=1, block=4: _native.call(
        "tgx_paged_append_scaled", ref, k, one, x, one, one, one, s, None, 2, D, dtype, code, block,
        None)
    for kw in (dict(k=None), dict(x=None), dict(k=one + 4), dict(x=one + 8), dict(dtype=7),
               dict(code=0), dict(block=3), dict(s=(ctypes.c_int64 * 8)(*[4] * 8))):
        with pytest.raises(RuntimeError):
            append(**kw)
    for D in (4, 12, 520):
        with pytest.raises(NotImplementedError):
            append(D=D)
    read = lambda k=one, out=one, s=four, D=64: _native.call(
        "tgx_paged_read", ref, k, one, one, one, s, out, one, 2, D, 0, 1, 4, None)
    for kw in (dict(k=None), dict(out=None), dict(out=one + 8), dict(s=(ctypes.c_int64 * 4)(*[4] * 4))):
        with pytest.raises(RuntimeError):
            read(**kw)
    with pytest.raises(NotImplementedError):
        read(D=12)


def signed(rng, code, heads=2, D=8, slots=PAGES * SIZE, block=BLOCK):
    """A cache stored elsewhere, whose scales are of either sign and no powers of two, and
    the same rows by positive scales: (cache, codes, scales)."""
    scales = rng.integers(8, 16, (slots // block, heads)) * \
        4.0 ** rng.integers(-11, 2, (slots // block, heads))
    sign = rng.choice([-1, 1], size=scales.shape)
    codes = want.rounded(rng.uniform(-want.LARGEST[code], want.LARGEST[code], (slots, heads, D)),
                         code)
    held = codes * np.repeat(sign, block, 0)[:, :, None]
    return tg.BlockScaled(torch.tensor(held, dtype=torch.float32).to(CODES[code]),
                          torch.tensor(scales * sign, dtype=torch.float32), block=block), codes, scales


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("queries", [1, 3, 11])
def test_scales_of_either_sign(code, queries):
    """A code by -s is the opposite code by s: append leaves the rows that it leaves of the
    same cache by positive scales."""
    rng = np.random.default_rng(20 + queries)
    lengths = torch.tensor([3, 15, 22, 40], dtype=torch.int32)
    g = graph(queries, lengths)
    (kc, kn, ks), (vc, vn, vs) = signed(rng, code), signed(rng, code)
    big = np.exp(rng.standard_normal((4 * queries, 2, 1)) * 3)
    k, v = (torch.tensor(rng.standard_normal((4 * queries, 2, 8)) * big).to(torch.float32)
            for _ in range(2))
    g.append(kc, k, vc, v)
    args = (TABLE.numpy(), lengths.numpy(), SIZE, PAGES, queries)
    for c, n, s, x in ((kc, kn, ks, k), (vc, vn, vs, v)):
        codes, scales = want.append(*args, n, s, f64(x), code, BLOCK)
        assert np.array_equal(np.abs(f64(c.scales)), scales)
        rows = [want.read(*args[:4], 24, want.values(a, b, BLOCK)) for a, b in (
            (f64(c.codes.float()), f64(c.scales)), (codes, scales))]
        assert np.array_equal(*rows)                     # (of all positions that are cached)


@pytest.mark.parametrize("code,scale,held", [("int8", -4.0, 100.0), ("int8", -8.0, 100.0),
                                             ("e4m3", -1.0, 416.0), ("e4m3", -8.0, 104.0)])
def test_small_tokens_behind_a_negative_scale(code, scale, held):
    g = tg.Graph.paged(torch.tensor([[0]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32),
                       page_size=4, num_pages=1)
    kc, vc = (tg.BlockScaled.zeros(4, 1, 8, block=4, dtype=CODES[code]) for _ in range(2))
    kc.scales.fill_(scale)
    kc.codes.view(torch.int8)[0] = torch.full((1, 8), held).to(CODES[code]).view(torch.int8)
    before = kc.dequantize()[0].clone()
    one = torch.ones(1, 1, 8)
    g.append(kc, one, vc, one)
    assert float(kc.scales) == scale
    assert torch.equal(kc.dequantize()[0], before)
    # What is new by that scale: to the nearest code, -1 / 4 and so on.
    assert np.array_equal(f64(kc.codes.float())[1], want.rounded(np.full((1, 8), 1 / scale), code))


@pytest.mark.parametrize("new,kept", [(1.0, True), (4096.0, False)])
def test_older_codes_that_are_nan_stay_nan(new, kept):
    """An older e4m3 NaN reads back as one where the scale stays and where it grows, and
    what stays is what was there to the bit."""
    g = tg.Graph.paged(torch.tensor([[0]], dtype=torch.int32), torch.tensor([3], dtype=torch.int32),
                       page_size=4, num_pages=1)
    kc, vc = (tg.BlockScaled.zeros(4, 1, 8, block=4) for _ in range(2))
    kc.scales.fill_(1.0)
    raw = kc.codes.view(torch.int8)
    raw[:2] = torch.tensor([0x7F, -1, 0, -128, 1, 0x38, -0x48, 0x7E], dtype=torch.int8)
    before = raw.clone()
    x = torch.full((1, 1, 8), new)
    g.append(kc, x, vc, x)
    rows = kc.dequantize()
    assert rows[:2, 0, :2].isnan().all() and not rows[:2, 0, 2:].isnan().any()
    assert (float(kc.scales) == 1.0) is kept and torch.equal(rows[2], x[0])
    if kept:
        assert torch.equal(raw[:2], before[:2])


def test_unlike_blocks_of_one_call_keep_their_codes():
    """Of two heads one's scale grows: the other's older codes are not written."""
    g = tg.Graph.paged(torch.tensor([[0]], dtype=torch.int32), torch.tensor([3], dtype=torch.int32),
                       page_size=4, num_pages=1)
    kc, vc = (tg.BlockScaled.zeros(4, 2, 8, block=4, dtype=torch.int8) for _ in range(2))
    kc.scales.fill_(0.5)
    kc.codes[:2] = torch.tensor([-128, 127, 3, -1, 0, 5, 64, -64], dtype=torch.int8)
    x = torch.tensor([1.0, 100.0])[None, :, None].expand(1, 2, 8)
    g.append(kc, x, vc, x)
    assert kc.scales.tolist() == [[0.5, 1.0]]
    assert kc.codes[0, 0].tolist() == [-128, 127, 3, -1, 0, 5, 64, -64]
    # Halves, ties to even.
    assert kc.codes[0, 1].tolist() == [-64, 64, 2, 0, 0, 2, 32, -32]


def test_a_prepared_call_differentiates_scales(monkeypatch):
    """prepare()'s bound launch has no gradients: a field that wants them, a cache's scales
    among them, takes the ordinary path.  (A stand-in for the launch, on the host.)"""
    from tiga import message_passing as mp

    rng = np.random.default_rng(8)
    (kc, _, _), (vc, _, _) = cache(rng, "int8"), cache(rng, "int8")
    g, kernel = graph(), Attention()
    src, dst = {"key": kc.grouped(), "value": vc.grouped()}, {"query": torch.randn(4, 2, 3, 8)}
    plain = lambda *_: Attention()(graph=g, src=src, dst=dst, scale=0.1)
    bound = torch.zeros(4, 2, 3, 8)

    def dispatch(self, *_):
        self._launch = mp._Launch(
            g, (("dst", "query"), ("src", "key"), ("src", "value")), plain, lambda: None,
            variant=mp.CompiledVariant(key=(), backend="hip", provider="", pattern="", lowering=""),
            bind=lambda *_: lambda: bound)
        return plain()

    monkeypatch.setattr(kernel, "_dispatch", dispatch.__get__(kernel))
    run = kernel.prepare(graph=g, src=src, dst=dst, scale=0.1)
    assert run() is bound
    kc.scales.requires_grad_(True)
    out = run()
    assert torch.equal(out, plain()) and out.requires_grad
    assert torch.autograd.grad(out.sum(), kc.scales)[0].abs().max() > 0


def test_what_the_tiles_take():
    """Widths 32, 64 and 128 of 16-bit queries, over codes that lie on 16 bytes."""
    from tiga import _paged

    def fields(D, heads=2, gap=0, first=0):
        slot = D + gap
        room = torch.zeros(32 * heads * slot + 16, dtype=torch.int8)
        first += -room.data_ptr() % 16
        codes = room[first:first + 32 * heads * slot].view(32, heads, slot)[..., :D]
        return tg.BlockScaled(codes, torch.zeros(4, heads), block=8).grouped()

    q = lambda D, dtype=torch.bfloat16: torch.zeros(1, 2, 4, D, dtype=dtype)
    good = fields(64)
    assert _paged.tiles_take(q(64), good, good) and _paged.tiles_take(
        q(64, torch.float16), good, fields(64, gap=16))
    assert not _paged.tiles_take(q(64, torch.float32), good, good)
    assert not _paged.tiles_take(q(40), fields(40), fields(40))
    for other in (fields(64, gap=8), fields(64, first=8)):
        assert not _paged.tiles_take(q(64), good, other)
        assert not _paged.tiles_take(q(64), other, good)
    cache16 = torch.zeros(32, 2, 1, 64, dtype=torch.bfloat16)
    assert _paged.tiles_take(q(64), cache16, cache16)


def test_what_a_cache_consists_of_is_fixed():
    """Launches go by the sizes that were checked once: other scales would be read past
    their end."""
    c = tg.BlockScaled.zeros(16, 2, 8, block=4)
    for name, value in (("scales", torch.zeros(1, 2)), ("codes", c.codes[:4]), ("block", 1),
                        ("tables", 2), ("spec", ()), ("other", 1)):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(c, name, value)
    with pytest.raises(AttributeError, match="fixed"):
        del c.scales
    c.scales.fill_(2.0)
    assert float(c.scales[3, 1]) == 2.0 and c.grouped().scales is c.scales


def test_older_codes_next_to_a_tie():
    """60 by 0.3 (in fp32 a little more) is 4.5 by 4 and a little more: 5."""
    g = tg.Graph.paged(torch.tensor([[0]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32),
                       page_size=4, num_pages=1)
    kc, vc = (tg.BlockScaled.zeros(4, 1, 8, block=4, dtype=torch.int8) for _ in range(2))
    kc.scales.fill_(0.3)
    kc.codes[0] = torch.tensor([60, -60, 100, -100, 20, -20, 127, 0], dtype=torch.int8)
    x = torch.full((1, 1, 8), 400.0)
    g.append(kc, x, vc, x)
    assert float(kc.scales) == 4.0 and (kc.codes[1] == 100).all()
    exact = np.array([60, -60, 100, -100, 20, -20, 127, 0]) * (float(np.float32(0.3)) / 4)
    assert kc.codes[0, 0].tolist() == np.rint(exact).tolist()
