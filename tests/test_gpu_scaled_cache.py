"""Caches in 8 bits on the HIP kernels against the formulas in float64: append and
read to the bit, attention within what rounding does; and attention over a window of
paged caches of either kind."""

import numpy as np
import pytest
import torch

import tiga as tg

import paged_reference as paged
import scaled_reference as want

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


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
dev = lambda x, dtype=torch.float32: torch.tensor(x, device=DEV).to(dtype)


def relation(rng, lengths, size, spare=2, width=None, missing=0):
    """(table, lengths, num_pages): shuffled pages, -1 where nothing is named."""
    used = [-(-max(n, 0) // size) for n in lengths]
    width = width or max(max(used), 1) + 1
    num_pages = sum(used) + spare
    order = rng.permutation(num_pages)
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    for _ in range(missing):
        b = int(rng.integers(len(lengths)))
        if used[b]:
            table[b, rng.integers(min(used[b], width))] = rng.choice([-5, num_pages, 2 ** 31 - 1])
    return table, np.asarray(lengths, dtype=np.int32), num_pages


def cache(rng, slots, heads, D, code, block, interleave=False):
    """(cache, its values): codes of all magnitudes by scales that differ by up to 8."""
    scales = 2.0 ** rng.integers(-9, -6, size=(slots // block, heads))
    codes = want.rounded(rng.standard_normal((slots, heads, D)) * 100, code)
    held = dev(codes).clamp(-want.LARGEST[code], want.LARGEST[code]).to(CODES[code])
    if interleave:      # codes of a slot behind others
        room = torch.zeros(slots, 2, heads, D, dtype=torch.int8, device=DEV)
        room[:, 1] = held.view(torch.int8)
        held = room[:, 1].view(CODES[code])
    c = tg.BlockScaled(held, dev(scales), block=block)
    return c, want.values(f64(held.float()), scales, block)


def check(lengths, size, block, heads, group, D, code, dtype, queries=1, seed=0, window=None,
          sinks=0, missing=0, width=None, interleave=False, scale=None):
    """Attention over an 8-bit cache, or one of the queries' type (`code` None), with
    NaN in every slot that no row sees and nothing named where nobody looks."""
    print(f"{code} {dtype} D={D} heads={heads} group={group} queries={queries} size={size} "
          f"block={block} window={window} sinks={sinks} lengths={lengths[:6]}", flush=True)
    rng = np.random.default_rng(seed)
    table, length, pages = relation(rng, lengths, size, width=width, missing=missing)
    slots = pages * size
    q = dev(rng.standard_normal((len(lengths) * queries, heads, group, D)), TYPES[dtype])
    seen = np.zeros(slots, dtype=bool)
    for b in range(len(lengths)):
        n = paged.length_of(length, b, table.shape[1], size)
        looked = np.zeros(n, dtype=bool)
        for t in range(queries):
            looked[want.seen(n - t, window, sinks)] = True
        at, named = paged.slots(table[b], n, size, pages)
        seen[at[named & looked]] = True
        for p in range(-(-n // size)):
            if not looked[p * size:(p + 1) * size].any():
                table[b, p] = rng.choice([-1, 2 ** 31 - 1, table[b, p]])
    hidden = torch.tensor(~seen, device=DEV)
    if code is None:
        k, v = (dev(rng.standard_normal((slots, heads, D)), TYPES[dtype]) for _ in range(2))
        kn, vn = f64(k), f64(v)
        k[hidden], v[hidden] = float("nan"), float("inf")
        fields = {"key": k[:, :, None], "value": v[:, :, None]}
    else:
        (kc, kn), (vc, vn) = (cache(rng, slots, heads, D, code, block, interleave)
                              for _ in range(2))
        blocks = hidden.view(-1, block).all(1)
        kc.scales[blocks], vc.scales[blocks] = float("nan"), float("inf")
        if code == "e4m3":
            for c in (kc, vc):
                c.codes.view(torch.int8)[hidden] = 0x7F
        fields = {"key": kc.grouped(), "value": vc.grouped()}
    scale = D ** -0.5 if scale is None else scale
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(length, device=DEV),
                       page_size=size, num_pages=pages, queries=queries, window=window,
                       sinks=sinks)
    tiles = dtype != "f32" and D in (32, 64, 128)
    # The parts of a weight: of the values' type in the tiles (bf16 for codes), else fp32;
    # fp16's may be off by 2^-39 of the largest as well, within the additions' share.
    part = 2 * HALF["bf16" if code else dtype] ** 2 if tiles else HALF["f32"]
    exp, lim = want.paged_attention(table, length, size, pages, queries, f64(q), kn, vn, scale,
                                    window, sinks, tiles, HALF[dtype], part)
    kernel = Attention()
    out = kernel(graph=g, src=fields, dst={"query": q}, scale=scale)
    assert kernel.last_variant.pattern == "paged-attention"
    assert out.shape == q.shape and out.dtype == TYPES[dtype]
    tiny = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24, "f32": 2.0 ** -149}[dtype]
    lim = lim + tiny + (2.0 ** -39 * np.abs(vn).max() * max(lengths) if dtype == "f16" else 0)
    err = np.abs(f64(out) - exp)
    assert (err <= lim).all(), f"error {np.nanmax(err):.3e}, {np.nanmax(err / lim):.2f} of the bound"
    return kernel, g, q, fields, out


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]


# ---------------------------------------------------------------------------
# append and read

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,heads,size,block", [
    (128, 3, 16, 16), (64, 2, 24, 8), (32, 1, 12, 3), (8, 2, 5, 1), (96, 2, 64, 32),
    (264, 1, 8, 8), (512, 2, 100, 50)])
@pytest.mark.parametrize("queries", [1, 4, 70])
def test_append_and_read_are_the_formula(code, dtype, D, heads, size, block, queries):
    print(f"{code} {dtype} D={D} heads={heads} size={size} block={block} queries={queries}",
          flush=True)
    rng = np.random.default_rng(D + queries)
    lengths = [0, 1, size, size + 1, 2 * size - 1, 150, 3 * size + 2]
    table, length, pages = relation(rng, lengths, size, missing=2)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(length, device=DEV),
                       page_size=size, num_pages=pages, queries=queries)
    rows = len(lengths) * queries
    new, caches, before = [], [], []
    for _ in range(2):
        c, _ = cache(rng, pages * size, heads, D, code, block)
        before.append((f64(c.codes.float()), f64(c.scales)))
        caches.append(c)
        # Keys and values of one projection, of magnitudes that move the scales.
        both = rng.standard_normal((rows, heads, 2, D)) * 4.0 ** rng.integers(-3, 4, (rows, heads, 1, 1))
        new.append(dev(both, TYPES[dtype])[:, :, 1])
    sums = torch.full((pages, heads, D), 7.0, device=DEV)
    args = (table, length, size, pages, queries)
    exp = [want.append(*args, *b, f64(x), code, block) for b, x in zip(before, new)]
    g.append(caches[0], new[0], caches[1], new[1], page_sums=sums)
    for c, (codes, scales) in zip(caches, exp):
        assert np.array_equal(f64(c.scales), scales)
        assert np.array_equal(f64(c.codes.float()), codes)
    held = [want.values(codes, scales, block) for codes, scales in exp]
    total = want.page_sums(*args, held[0], np.full((pages, heads, D), 7.0))
    # A page's sum: at most `size` values, each addition off by half a step of the sum so far.
    most = want.page_sums(*args, np.abs(held[0]), np.full((pages, heads, D), 7.0))
    assert (np.abs(f64(sums) - total) <= (size + 1) * 2.0 ** -24 * most).all()
    got = g.read(*caches, dtype=TYPES[dtype])
    for x, rows_ in zip(got, held):
        exact = torch.tensor(want.read(*args, rows_), device=DEV).float().to(TYPES[dtype])
        assert torch.equal(x, exact)
    # Without sums, and again: the same codes.
    g.append(caches[0], new[0], caches[1], new[1])
    assert np.array_equal(f64(caches[0].codes.float()), exp[0][0])


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_codes_cannot_hold_makes_the_block_nan(code, bad):
    rng = np.random.default_rng(3)
    table, lengths = dev([[0, 1]], torch.int32), dev([6], torch.int32)
    make = lambda q: tg.Graph.paged(table, lengths, page_size=8, num_pages=2, queries=q)
    kc, vc = (tg.BlockScaled.zeros(16, 2, 8, block=4, dtype=CODES[code], device=DEV)
              for _ in range(2))
    sums = torch.zeros(2, 2, 8, device=DEV)
    k = dev(rng.standard_normal((6, 2, 8)))
    k[5, 1, 3] = bad
    make(6).append(kc, k, vc, k.nan_to_num(0, 0, 0), page_sums=sums)
    rows = kc.dequantize()
    assert rows[4:6, 1].isnan().all() and not rows[:4].isnan().any()
    assert not rows[4:6, 0].isnan().any() and not vc.dequantize().isnan().any()
    assert sums[0, 1].isnan().all() and not sums[0, 0].isnan().any()
    lengths += 1
    fine = torch.ones(1, 2, 8, device=DEV)
    make(1).append(kc, fine, vc, fine)
    assert kc.dequantize()[4:7, 1].isnan().all() and not kc.dequantize()[4:7, 0].isnan().any()
    lengths.fill_(5)
    make(1).append(kc, fine, vc, fine, page_sums=sums)
    assert torch.equal(kc.dequantize()[4], fine[0]) and not sums.isnan().any()


@pytest.mark.parametrize("code", CODES)
def test_the_scale_is_the_smallest_power_of_two(code):
    top = want.LARGEST[code]
    amax = np.array([0.0, 2.0 ** -149, 2.0 ** -126, 1.0, top, np.nextafter(np.float32(top), np.float32(999)),
                     np.nextafter(np.float32(top), np.float32(0)), top * 2.0 ** -130, 2.0 ** 127,
                     np.finfo(np.float32).max], dtype=np.float32)
    n = len(amax)
    g = tg.Graph.paged(torch.arange(n, dtype=torch.int32, device=DEV)[:, None],
                       torch.ones(n, dtype=torch.int32, device=DEV), page_size=1, num_pages=n)
    c, other = (tg.BlockScaled.zeros(n, 1, 8, block=1, dtype=CODES[code], device=DEV)
                for _ in range(2))
    x = dev(amax)[:, None, None].repeat(1, 1, 8)
    x[:, :, 1:] *= -0.75
    g.append(c, x, other, x)
    codes, scales = want.append(np.arange(n)[:, None], np.ones(n), 1, n, 1, np.zeros((n, 1, 8)),
                                np.zeros((n, 1)), f64(x), code, 1)
    assert np.array_equal(f64(c.scales), scales) and np.array_equal(f64(c.codes.float()), codes)


@pytest.mark.parametrize("code", CODES)
def test_every_code_reads_back(code):
    """All 256 bytes, as the type has them, in every output type."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.int8).view(CODES[code]).to(DEV)
    c = tg.BlockScaled(codes.view(32, 1, 8), torch.full((32, 1), 0.5, device=DEV), block=1)
    g = tg.Graph.paged(torch.arange(32, dtype=torch.int32, device=DEV)[:, None],
                       torch.ones(32, dtype=torch.int32, device=DEV), page_size=1, num_pages=32)
    for dtype in TYPES.values():
        got = g.read(c, c, dtype=dtype)[0]
        exp = (codes.float() * 0.5).view(32, 1, 8).to(dtype)
        assert torch.equal(got.nan_to_num(999), exp.nan_to_num(999))
        assert torch.equal(got.isnan(), exp.isnan())


def test_scales_that_are_no_powers_of_two_stay():
    """A cache stored elsewhere: new tokens that fit go by its scale, others by a power."""
    table, lengths = dev([[0]], torch.int32), dev([2], torch.int32)
    g = tg.Graph.paged(table, lengths, page_size=8, num_pages=1)
    for x, scale in ((30.0, 0.3), (50.0, 0.5)):
        kc, vc = (tg.BlockScaled.zeros(8, 1, 8, block=8, dtype=torch.int8, device=DEV)
                  for _ in range(2))
        kc.scales.fill_(0.3)
        kc.codes[0] = 100
        new = torch.full((1, 1, 8), x, device=DEV)
        g.append(kc, new, vc, new)
        assert float(kc.scales) == np.float32(scale)
        # 30 / 0.3 and 50 / 0.5 are 100; the older token's 100 by 0.3 / 0.5 is 60.
        assert (kc.codes[1] == 100).all() and (kc.codes[0] == (100 if scale == 0.3 else 60)).all()


# ---------------------------------------------------------------------------
# attention over 8 bits

@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("queries", [1, 3])
def test_lengths_around_tiles_and_pages(code, dtype, D, queries):
    check(EDGES, 16, 8, 2, 4, D, code, dtype, queries=queries)


@pytest.mark.parametrize("D", [8, 24, 40, 96, 256, 320, 512])
@pytest.mark.parametrize("code,dtype", [("e4m3", "bf16"), ("int8", "f32")])
def test_other_widths(D, code, dtype):
    check([0, 1, 70, 333], 16, 16, 2, 2, D, code, dtype)


@pytest.mark.parametrize("size,block", [(1, 1), (3, 3), (8, 2), (24, 8), (48, 48), (100, 25),
                                        (256, 64)])
def test_page_and_block_sizes(size, block):
    check([5, 64, 131, 700], size, block, 2, 4, 64, "e4m3", "f16", queries=2, seed=size)
    check([5, 64, 131, 700], size, block, 2, 4, 128, "int8", "bf16", queries=2, seed=size)


@pytest.mark.parametrize("heads,group,queries", [
    (1, 1, 1), (3, 1, 1), (8, 4, 1), (1, 16, 1), (1, 17, 1), (2, 32, 1), (2, 5, 4), (2, 7, 5),
    (1, 3, 40), (2, 71, 1)])
def test_head_groups_and_queries(heads, group, queries):
    check([0, 1, 30, 64, 200], 16, 8, heads, group, 64, "int8", "bf16", queries=queries)
    check([0, 1, 30, 64, 200], 16, 8, heads, group, 128, "e4m3", "f16", queries=queries)
    check([0, 1, 30, 64, 200], 16, 8, heads, group, 32, "e4m3", "bf16", queries=queries)


@pytest.mark.parametrize("lengths", [[20000], [9000, 1, 0, 300, 4111], [3000] * 40])
@pytest.mark.parametrize("code,dtype", [("e4m3", "bf16"), ("int8", "f16"), ("int8", "f32")])
def test_long_lengths_in_pieces(lengths, code, dtype):
    check(lengths, 16, 16, 2, 4, 64 if len(lengths) > 9 else 128, code, dtype, queries=2)


@pytest.mark.parametrize("code", CODES)
def test_pages_that_are_not_there(code):
    check([40, 64, 300, 1000], 16, 8, 2, 3, 64, code, "bf16", queries=2, missing=12)
    check([40, 64, 300, 1000], 16, 8, 2, 3, 128, code, "f16", queries=20, missing=12)


@pytest.mark.parametrize("scale", [0.0, -0.25, 2.0])
def test_score_scales(scale):
    check([200, 65], 16, 16, 2, 2, 64, "e4m3", "bf16", scale=scale)
    check([200, 65], 16, 16, 2, 20, 64, "int8", "f16", scale=scale)


def test_codes_of_a_slot_next_to_others_and_on_eight_bytes():
    check([0, 77, 1000], 16, 16, 4, 2, 64, "e4m3", "bf16", interleave=True)
    check([0, 77, 1000], 16, 16, 4, 2, 40, "int8", "bf16", interleave=True)
    # Rows on 8 bytes only: the kernel that reads them by eights.
    rng = np.random.default_rng(1)
    table, length, pages = relation(rng, [100, 33], 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages)
    c, values = cache(rng, pages * 16, 1, 64, "int8", 16)
    room = torch.zeros(pages * 16, 1, 72, dtype=torch.int8, device=DEV)
    room[..., 8:] = c.codes
    odd = tg.BlockScaled(room[..., 8:], c.scales, block=16)
    q = dev(rng.standard_normal((2, 1, 4, 64)), torch.bfloat16)
    out = Attention()(graph=g, src={"key": odd.grouped(), "value": odd.grouped()},
                      dst={"query": q}, scale=0.125)
    exp, lim = want.paged_attention(table, length, 16, pages, 1, f64(q), values, values, 0.125,
                                    step=HALF["bf16"], part=HALF["f32"])
    assert (np.abs(f64(out) - exp) <= lim).all()
    # On no 8 bytes: refused when strict, from the values otherwise.
    room = torch.zeros(pages * 16, 1, 68, dtype=torch.int8, device=DEV)
    room[..., 4:] = c.codes
    odd = tg.BlockScaled(room[..., 4:], c.scales, block=16)
    call = lambda: Attention()(graph=g, src={"key": odd.grouped(), "value": odd.grouped()},
                               dst={"query": q}, scale=0.125)
    with pytest.raises(RuntimeError, match="strict"):
        call()
    with pytest.raises(RuntimeError, match="strict"):
        g.read(odd, odd)
    with pytest.raises(RuntimeError, match="strict"):
        g.append(odd, q[:, :, 0], odd, q[:, :, 0])
    tg.config.strict = False
    assert call().dtype == torch.bfloat16
    # fp32 sums of the same values, then the rounding: within twice the bound.
    assert (np.abs(f64(call()) - exp) <= 2 * lim + HALF["bf16"] * np.abs(exp)).all()
    assert torch.equal(g.read(odd, odd)[0], g.read(c, c)[0])


@pytest.mark.parametrize("queries,group", [(4, 3), (4, 8), (40, 4)])
def test_newer_tokens_never_reach_older_rows(queries, group):
    """NaN codes of the newest token, and the NaN scale of a block that only the newest
    tokens see, belong to the rows that see them and to no other."""
    rng = np.random.default_rng(1)
    lengths = [81, 45, 209]
    table, length, pages = relation(rng, lengths, 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages, queries=queries)
    q = dev(rng.standard_normal((3 * queries, 2, group, 64)), torch.bfloat16)
    for code in CODES:
        (kc, kn), (vc, vn) = (cache(rng, pages * 16, 2, 64, code, 1) for _ in range(2))
        exp, lim = want.paged_attention(table, length, 16, pages, queries, f64(q), kn, vn, 0.125,
                                        tiles=True, step=HALF["bf16"], part=2.0 ** -15)
        for b, n in enumerate(lengths):
            slot = int(table[b, (n - 1) // 16]) * 16 + (n - 1) % 16
            if code == "e4m3" and b % 2:
                vc.codes.view(torch.int8)[slot] = 0x7F
            else:
                vc.scales[slot] = float("nan")
            if b == 2:
                kc.scales[slot] = float("nan")
        out = Attention()(graph=g, src={"key": kc.grouped(), "value": vc.grouped()},
                          dst={"query": q}, scale=0.125)
        got, exp, lim = (x.reshape(3, queries, 2, group, 64) for x in (f64(out), exp, lim))
        assert (np.abs(got - exp)[:, :-1] <= lim[:, :-1]).all()
        assert np.isnan(got[:, -1]).all()


@pytest.mark.parametrize("code", CODES)
def test_a_table_per_head(code):
    rng = np.random.default_rng(16)
    B, T, P, size, pages, queries, heads, group, D = 3, 4, 6, 16, 30, 2, 2, 3, 64
    table = rng.integers(-1, pages, size=(B, T, P)).astype(np.int32)
    lengths = np.array([90, 1, 33], dtype=np.int32)
    g = tg.Graph.paged(dev(table, torch.int32), dev(lengths, torch.int32), page_size=size,
                       num_pages=pages, queries=queries)
    q = dev(rng.standard_normal((B * queries * T, heads, group, D)), torch.bfloat16)
    fields, values = [], []
    for _ in range(2):
        c, v = cache(rng, pages * size, T * heads, D, code, 8)
        codes = c.codes.view(pages * size * T, heads, D)
        fields.append(tg.BlockScaled(codes, c.scales.view(-1, heads), block=8, tables=T).grouped())
        values.append(v.reshape(pages * size, T, heads, D))
    out = Attention()(graph=g, src={"key": fields[0], "value": fields[1]}, dst={"query": q},
                      scale=0.125)
    exp = paged.attention(table, lengths, size, pages, queries, f64(q), *values, 0.125)
    _, lim = want.paged_attention(table.reshape(B * T, P), np.repeat(lengths, T), size, pages, 1,
                                  np.zeros((B * T, heads, group, D)), values[0][:, 0],
                                  values[1][:, 0], 0.125)
    # Half a step of the output, and two bf16 parts and fp32 sums of at most 90 keys of the
    # largest value; scores off by 74 products' roundings.
    vmax = np.abs(values[1]).max()
    s = 0.125 * np.abs(f64(q)).sum(-1).max() * np.abs(values[0]).max()
    lim = HALF["bf16"] * np.abs(exp) + (2.0 ** -15 + 2.0 ** -24 * (2 * 74 * s + 400)) * vmax
    assert (np.abs(f64(out) - exp) <= lim).all()
    # A field that counts its rows otherwise is not this relation's.
    flat = tg.BlockScaled(fields[0].codes, fields[0].scales, block=8)
    with pytest.raises(RuntimeError, match="strict"):
        Attention()(graph=g, src={"key": flat, "value": flat}, dst={"query": q}, scale=0.125)


def test_offsets_past_32_bits():
    """Slots whose codes lie beyond 4 GiB, and beyond 2 GiB of a head's."""
    slots, heads, D = 1 << 21, 17, 128
    rng = np.random.default_rng(2)
    table = np.array([[1, (1 << 21) // 64 - 1, (1 << 21) // 64 - 2]], dtype=np.int32)
    lengths = np.array([150], dtype=np.int32)
    pages = slots // 64
    caches = [tg.BlockScaled.zeros(slots, heads, D, block=64, device=DEV) for _ in range(2)]
    g = tg.Graph.paged(dev(table, torch.int32), dev(lengths, torch.int32), page_size=64,
                       num_pages=pages, queries=150)
    k, v = (dev(rng.standard_normal((150, heads, D)), torch.bfloat16) for _ in range(2))
    g.append(caches[0], k, caches[1], v)
    back = g.read(*caches, dtype=torch.float32)
    for x, b, c in zip((k, v), back, caches):
        # Codes with three bits behind the leading one: half a step is 2^-4 of a value, or
        # of the smallest normal one.
        scale = c.scales[(dev(table[0], torch.int64)).repeat_interleave(64)[:150]]
        assert ((b - x.float()).abs() <= 2.0 ** -4 * torch.maximum(
            x.float().abs(), scale[..., None] * 2.0 ** -6)).all()
    q = dev(rng.standard_normal((1, heads, 4, D)), torch.bfloat16)
    one = tg.Graph.paged(dev(table, torch.int32), dev(lengths, torch.int32), page_size=64,
                         num_pages=pages)
    out = Attention()(graph=one, src={"key": caches[0].grouped(), "value": caches[1].grouped()},
                      dst={"query": q}, scale=0.1)
    small = np.array([[0, 1, 2]], dtype=np.int32)
    kn, vn = (np.concatenate([f64(b), np.zeros((42, heads, D))]) for b in back)
    exp, lim = want.paged_attention(small, lengths, 64, 3, 1, f64(q), kn, vn, 0.1, tiles=True,
                                    step=HALF["bf16"], part=2.0 ** -15)
    assert (np.abs(f64(out) - exp) <= lim).all()


def test_gradients_of_queries_and_scales():
    rng = np.random.default_rng(7)
    table, length, pages = relation(rng, [40, 3, 0], 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages)
    (kc, kn), (vc, vn) = (cache(rng, pages * 16, 2, 64, "int8", 16) for _ in range(2))
    q = dev(rng.standard_normal((3, 2, 3, 64))).requires_grad_(True)
    kc.scales.requires_grad_(True)
    kernel = Attention()
    out = kernel(graph=g, src={"key": kc.grouped(), "value": vc.grouped()}, dst={"query": q},
                 scale=0.125)
    dq, ds = torch.autograd.grad(out.square().sum(), (q, kc.scales))
    host = lambda t: t.detach().cpu()
    tg.config.strict = False
    qh = host(q).double().requires_grad_(True)
    sh = host(kc.scales).requires_grad_(True)
    gh = tg.Graph.paged(torch.tensor(table), torch.tensor(length), page_size=16, num_pages=pages)
    oh = Attention()(graph=gh, src={
        "key": tg.BlockScaled(host(kc.codes), sh, block=16).grouped(),
        "value": tg.BlockScaled(host(vc.codes), host(vc.scales), block=16).grouped()},
        dst={"query": qh}, scale=0.125)
    eq, es = torch.autograd.grad(oh.square().sum(), (qh, sh))
    # fp32 sums of at most 64 * 40 products against 64 bits.
    assert np.abs(f64(dq) - eq.numpy()).max() <= 1e-4 * np.abs(eq.numpy()).max()
    assert np.abs(f64(ds) - es.double().numpy()).max() <= 1e-4 * es.abs().max()


# ---------------------------------------------------------------------------
# windows

WINDOWS = [(1, 0), (5, 0), (64, 1), (65, 4), (100, 70), (128, 128), (1000, 3)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("code,dtype", [(None, "bf16"), (None, "f16"), (None, "f32"),
                                        ("e4m3", "bf16"), ("int8", "f16"), ("int8", "f32")])
def test_windows(window, sinks, code, dtype):
    lengths = EDGES + [700, 2000]
    check(lengths, 16, 8, 2, 4, 64, code, dtype, window=window, sinks=sinks)
    check(lengths, 16, 8, 1, 3, 128, code, dtype, queries=3, window=window, sinks=sinks)
    check([5, 300, 131, 900], 24, 8, 1, 4, 32, code, dtype, queries=30, window=window, sinks=sinks)


@pytest.mark.parametrize("code", [None, "e4m3"])
def test_far_windows_in_pieces(code):
    check([30000, 9000, 1, 0, 300], 16, 16, 2, 4, 128, code, "bf16", window=6000, sinks=100)
    check([20000, 20000], 64, 64, 1, 4, 64, code, "f16", queries=2, window=3333, sinks=1)
    check([4000, 300], 16, 16, 1, 2, 128, code, "bf16", queries=200, window=500, sinks=65)


def test_a_window_past_everything_is_no_window():
    rng = np.random.default_rng(4)
    table, length, pages = relation(rng, [300, 5, 64], 16)
    q = dev(rng.standard_normal((3, 2, 4, 64)), torch.bfloat16)
    k, v = (dev(rng.standard_normal((pages * 16, 2, 1, 64)), torch.bfloat16) for _ in range(2))
    make = lambda **kw: tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32),
                                       page_size=16, num_pages=pages, **kw)
    call = lambda g: Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q}, scale=0.2)
    assert torch.equal(call(make()), call(make(window=2**31 - 1, sinks=2**31 - 1)))


@pytest.mark.parametrize("queries,group", [(4, 4), (20, 4)])
def test_older_tokens_never_reach_newer_rows(queries, group):
    """A NaN that has left the newest row's window but not the oldest's."""
    rng = np.random.default_rng(9)
    n, window = 200, 50
    table, length, pages = relation(rng, [n], 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages, queries=queries, window=window, sinks=2)
    q = dev(rng.standard_normal((queries, 1, group, 64)), torch.float16)
    k, v = (dev(rng.standard_normal((pages * 16, 1, 64)), torch.float16) for _ in range(2))
    exp, lim = want.paged_attention(table, length, 16, pages, queries, f64(q), f64(k), f64(v), 0.125,
                                    window, 2, True, HALF["f16"], 2.0 ** -21)
    pos = n - queries + 1 - window      # the oldest row's first, in no other row's window
    slot = int(table[0, pos // 16]) * 16 + pos % 16
    k[slot], v[slot] = float("inf"), float("nan")
    out = f64(Attention()(graph=g, src={"key": k[:, :, None], "value": v[:, :, None]},
                          dst={"query": q}, scale=0.125))
    lim = lim + 2.0 ** -24 + 2.0 ** -39 * 4 * n
    assert (np.abs(out - exp)[1:] <= lim[1:]).all() and np.isnan(out[0]).all()


# ---------------------------------------------------------------------------
# as a program uses them

@pytest.mark.parametrize("code", CODES)
def test_prompt_steps_selection_and_reading_back(code):
    """Prompts written, tokens answered one by one over a window and over chosen pages,
    some taken back; the cache read at the end.  Against a cache of plain values."""
    rng = np.random.default_rng(11)
    B, heads, group, D, size, block, width = 3, 2, 4, 64, 16, 8, 12
    pages = B * width
    table = dev(rng.permutation(pages).reshape(B, width), torch.int32)
    lengths = dev([0, 0, 0], torch.int32)
    make = lambda q, **kw: tg.Graph.paged(table, lengths, page_size=size, num_pages=pages,
                                          queries=q, **kw)
    prompt, one, near = make(100), make(1), make(1, window=40, sinks=3)
    kc, vc = (tg.BlockScaled.zeros(pages * size, heads, D, block=block, dtype=CODES[code],
                                   device=DEV) for _ in range(2))
    sums = torch.zeros(pages, heads, D, device=DEV)
    host = [np.zeros((pages * size, heads, D)), np.zeros((pages // 1 * size // block, heads))]
    kn, ks, vn, vs = host[0], host[1], host[0].copy(), host[1].copy()
    args = lambda q: (table.cpu().numpy(), lengths.cpu().numpy(), size, pages, q)
    lengths.copy_(dev([100, 37, 1], torch.int32))
    k, v = (dev(rng.standard_normal((B * 100, heads, D)), torch.bfloat16) for _ in range(2))
    prompt.append(kc, k, vc, v, page_sums=sums)
    kn, ks = want.append(*args(100), kn, ks, f64(k), code, block)
    vn, vs = want.append(*args(100), vn, vs, f64(v), code, block)
    chosen = None
    for step in range(12):
        lengths += 1 if step != 6 else -2       # two tokens are taken back
        k, v = (dev(rng.standard_normal((B, heads, D)) * (step + 1), torch.bfloat16)
                for _ in range(2))
        one.append(kc, k, vc, v, page_sums=sums)
        kn, ks = want.append(*args(1), kn, ks, f64(k), code, block)
        vn, vs = want.append(*args(1), vn, vs, f64(v), code, block)
        q = dev(rng.standard_normal((B, heads, group, D)), torch.bfloat16)
        rows = [want.values(c, s, block) for c, s in ((kn, ks), (vn, vs))]
        out = Attention()(graph=near, src={"key": kc.grouped(), "value": vc.grouped()},
                          dst={"query": q}, scale=0.125)
        exp, lim = want.paged_attention(*args(1), f64(q), *rows, 0.125, 40, 3, True, HALF["bf16"],
                                        2.0 ** -15)
        assert (np.abs(f64(out) - exp) <= lim).all()
        chosen = one.select_pages(q, sums, 3, out=chosen)
        out = Attention()(graph=chosen, src={"key": kc.per_head(), "value": vc.per_head()},
                          dst={"query": q.view(-1, group, D)}, scale=0.125)
        by = [r.reshape(-1, heads, 1, D) for r in rows]
        exp = paged.attention(chosen.page_table.cpu().numpy(), chosen.lengths.cpu().numpy(), size,
                              pages, 1, f64(q).reshape(-1, 1, group, D), *by, 0.125)
        vmax = np.abs(rows[1]).max()
        s = 0.125 * np.abs(f64(q)).sum(-1).max() * np.abs(rows[0]).max()
        lim = HALF["bf16"] * np.abs(exp) + (2.0 ** -15 + 2.0 ** -24 * (150 * s + 400)) * vmax
        assert (np.abs(f64(out).reshape(exp.shape) - exp) <= lim).all()
    whole = make(width * size)
    got = whole.read(kc, vc, dtype=torch.float32)
    for x, r in zip(got, rows):
        assert np.array_equal(f64(x), want.read(*args(width * size), r))


@pytest.mark.parametrize("window", [None, 30])
def test_captured_steps_follow_the_live_tables(window):
    """append, attention and read in one captured graph, replayed as the lengths grow."""
    rng = np.random.default_rng(12)
    table = dev(rng.permutation(24).reshape(2, 12), torch.int32)
    lengths = dev([50, 3], torch.int32)
    g = tg.Graph.paged(table, lengths, page_size=16, num_pages=24, window=window,
                       sinks=0 if window is None else 2)
    kc, vc = (cache(rng, 24 * 16, 2, 64, "e4m3", 16)[0] for _ in range(2))
    k, v = (dev(rng.standard_normal((2, 2, 64)), torch.bfloat16) for _ in range(2))
    q = dev(rng.standard_normal((2, 2, 4, 64)), torch.bfloat16)
    sums = torch.zeros(24, 2, 64, device=DEV)
    attend = Attention().prepare(graph=g, src={"key": kc.grouped(), "value": vc.grouped()},
                                 dst={"query": q}, scale=0.125)

    def step():
        g.append(kc, k, vc, v, page_sums=sums)
        return (attend(), *g.read(kc, vc))

    state = (kc.codes.view(torch.int8), kc.scales, vc.codes.view(torch.int8), vc.scales, lengths,
             sums)
    kept = [t.clone() for t in state]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        outs = step()

    def restore():
        for t, b in zip(state, kept):
            t.copy_(b)

    def run(play):
        restore()
        got = []
        gen = torch.Generator(device=DEV).manual_seed(5)
        for i in range(5):
            lengths.add_(7)
            k.copy_(torch.randn(k.shape, device=DEV, generator=gen))
            v.copy_(torch.randn(v.shape, device=DEV, generator=gen))
            res = play()
            torch.cuda.synchronize()
            got.append([t.clone() for t in res] + [sums.clone()])
        return got

    eager = run(step)

    def replay():
        captured.replay()
        return outs

    for a, b in zip(eager, run(replay)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_another_stream():
    rng = np.random.default_rng(13)
    table, length, pages = relation(rng, [900, 50], 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages, window=100, sinks=4)
    (kc, _), (vc, _) = (cache(rng, pages * 16, 2, 128, "int8", 16) for _ in range(2))
    q = dev(rng.standard_normal((2, 2, 4, 128)), torch.bfloat16)
    call = lambda: Attention()(graph=g, src={"key": kc.grouped(), "value": vc.grouped()},
                               dst={"query": q}, scale=0.1)
    a = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        b, (rk, rv) = call(), g.read(kc, vc)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(a, b) and torch.equal(rk, g.read(kc, vc)[0])


def test_codes_of_one_layout_at_other_addresses():
    """A kept call takes codes that do not start on 8 bytes, too."""
    rng = np.random.default_rng(5)
    table, length, pages = relation(rng, [100, 33], 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages)
    c, _ = cache(rng, pages * 16, 2, 64, "int8", 16)
    n = c.codes.numel()
    room = torch.zeros(n + 8, dtype=torch.int8, device=DEV)
    q = dev(rng.standard_normal((2, 2, 64)), torch.bfloat16)
    kernel, got = Attention(), []
    for at in (0, 8, 4, 3, 0):
        codes = room[at:at + n].view(c.codes.shape)
        codes.copy_(c.codes)
        held = tg.BlockScaled(codes, c.scales, block=16)
        got.append(kernel(graph=g, src={"key": held, "value": held}, dst={"query": q}, scale=0.125))
    # (By eights or sixteens: each within half a step of the same value, and sums of
    # values below 4 in two parts of a weight and another order within 4 2^-15.)
    assert all(torch.allclose(x.float(), got[0].float(), rtol=2 * HALF["bf16"], atol=2.0 ** -13)
               for x in got)


def test_empty_calls():
    table = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    lengths = torch.zeros(0, dtype=torch.int32, device=DEV)
    g = tg.Graph.paged(table, lengths, page_size=16, num_pages=4, window=5)
    c = tg.BlockScaled.zeros(64, 2, 64, block=16, device=DEV)
    x = torch.zeros(0, 2, 64, device=DEV, dtype=torch.bfloat16)
    g.append(c, x, c, x)
    assert g.read(c, c)[0].shape == (0, 2, 64)
    out = Attention()(graph=g, src={"key": c.grouped(), "value": c.grouped()},
                      dst={"query": x[:, :, None].expand(0, 2, 3, 64)}, scale=1.0)
    assert out.shape == (0, 2, 3, 64)
    # A cache of no pages, and tables that name none.
    none = tg.Graph.paged(dev([[0, 1]], torch.int32), dev([20], torch.int32), page_size=16,
                          num_pages=0)
    c = tg.BlockScaled.zeros(0, 2, 64, block=16, device=DEV)
    x = torch.ones(1, 2, 64, device=DEV, dtype=torch.bfloat16)
    none.append(c, x, c, x)
    assert not none.read(c, c)[0].any()
    out = Attention()(graph=none, src={"key": c.grouped(), "value": c.grouped()},
                      dst={"query": x[:, :, None]}, scale=1.0)
    assert not out.any()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("queries", [1, 5, 40])
@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_either_sign(code, queries, dtype):
    """Caches stored elsewhere, with negative scales that are no powers of two: a code by -s
    is the opposite code by s, so what append leaves follows from positive scales."""
    print(f"{code} {dtype} queries={queries}", flush=True)
    rng = np.random.default_rng(40 + queries)
    size, block, heads, D = 16, 8, 3, 64
    table, length, pages = relation(rng, [3, 15, 22, 60], size)
    g = tg.Graph.paged(torch.tensor(table, device=DEV), torch.tensor(length, device=DEV),
                       page_size=size, num_pages=pages, queries=queries)
    args = (table, length, size, pages)
    caches, new, exp = [], [], []
    for _ in range(2):
        # (Of few bits, as the new values: a code times a scale is exact in 32 bits, and a
        # quotient lies on a tie or away from it by far more than its rounding.)
        scales = rng.integers(8, 16, (pages * size // block, heads)) * \
            4.0 ** rng.integers(-8, 2, (pages * size // block, heads))
        sign = rng.choice([-1, 1], size=scales.shape)
        codes = want.rounded(rng.uniform(-want.LARGEST[code], want.LARGEST[code],
                                         (pages * size, heads, D)), code)
        held = dev(codes * np.repeat(sign, block, 0)[:, :, None]).to(CODES[code])
        caches.append(tg.BlockScaled(held, dev(scales * sign), block=block))
        big = 4.0 ** rng.integers(-3, 6, (len(length) * queries, heads, 1))
        new.append(dev(rng.standard_normal((len(length) * queries, heads, D)) * big,
                       torch.bfloat16).to(TYPES[dtype]))
        exp.append(want.append(*args, queries, codes, scales, f64(new[-1]), code, block))
    sums = torch.zeros(pages, heads, D, device=DEV)
    g.append(caches[0], new[0], caches[1], new[1], page_sums=sums)
    every = table.shape[1] * size
    for c, (codes, scales) in zip(caches, exp):
        assert np.array_equal(np.abs(f64(c.scales)), scales)
        got = want.values(f64(c.codes.float()), f64(c.scales), block)
        assert np.array_equal(want.read(*args, every, got),
                              want.read(*args, every, want.values(codes, scales, block)))
    total, most = (want.page_sums(*args, queries, x, np.zeros((pages, heads, D)))
                   for x in (want.values(*exp[0], block), np.abs(want.values(*exp[0], block))))
    # A page's sum: at most 16 values, each addition off by half a step of the sum so far.
    assert (np.abs(f64(sums) - total) <= (size + 1) * 2.0 ** -24 * most).all()


@pytest.mark.parametrize("new", [1.0, 4096.0])
def test_older_codes_that_are_nan_stay_nan(new):
    """As on host tensors: an older e4m3 NaN reads back as one, whether the scale stays or
    grows, and the other codes are those of the host's append."""
    make = lambda where: tg.Graph.paged(
        torch.tensor([[0]], dtype=torch.int32, device=where),
        torch.tensor([3], dtype=torch.int32, device=where), page_size=4, num_pages=1)
    raw = torch.zeros(4, 1, 8, dtype=torch.int8)
    raw[:2] = torch.tensor([0x7F, -1, 0, -128, 1, 0x38, -0x48, 0x7E], dtype=torch.int8)
    got = []
    for where in ("cpu", DEV):
        kc, vc = (tg.BlockScaled(raw.to(where, copy=True).view(CODES["e4m3"]),
                                 torch.ones(1, 1, device=where), block=4) for _ in range(2))
        x = torch.full((1, 1, 8), new, device=where)
        make(where).append(kc, x, vc, x)
        got.append((kc.dequantize().cpu(), kc.scales.cpu(), vc.dequantize().cpu()))
    assert got[1][0][:2, 0, :2].isnan().all() and not got[1][0][:2, 0, 2:].isnan().any()
    for a, b in zip(*got):
        assert torch.equal(a.nan_to_num(9999), b.nan_to_num(9999))


def test_a_prepared_call_differentiates_scales():
    rng = np.random.default_rng(9)
    table, length, pages = relation(rng, [40, 3], 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages)
    (kc, _), (vc, _) = (cache(rng, pages * 16, 2, 64, "int8", 16) for _ in range(2))
    q = dev(rng.standard_normal((2, 2, 3, 64)))
    call = dict(graph=g, src={"key": kc.grouped(), "value": vc.grouped()}, dst={"query": q},
                scale=0.125)
    before = Attention().prepare(**call)
    fast = before()
    assert not fast.requires_grad
    vc.scales.requires_grad_(True)
    exp = torch.autograd.grad(Attention()(**call).square().sum(), vc.scales)[0]
    for run in (before, Attention().prepare(**call)):
        out = run()
        # fp32 sums of at most 40 products, by two kernels.
        assert torch.allclose(out, fast, rtol=1e-5, atol=1e-5 * float(fast.abs().max()))
        assert torch.equal(torch.autograd.grad(out.square().sum(), vc.scales)[0], exp)
    with torch.no_grad():
        assert not before().requires_grad


def test_a_variant_tells_how_rows_are_read():
    rng = np.random.default_rng(1)
    table, length, pages = relation(rng, [100], 16)
    g = tg.Graph.paged(dev(table, torch.int32), dev(length, torch.int32), page_size=16,
                       num_pages=pages)
    c, _ = cache(rng, pages * 16, 1, 64, "int8", 16)
    room = torch.zeros(pages * 16, 1, 72, dtype=torch.int8, device=DEV)
    room[..., 8:] = c.codes
    odd = tg.BlockScaled(room[..., 8:], c.scales, block=16)
    q = dev(rng.standard_normal((1, 1, 4, 64)), torch.bfloat16)
    for held, text in ((c, "once for 128 queries"), (odd, "once for each query")):
        kernel = Attention()
        kernel(graph=g, src={"key": held.grouped(), "value": held.grouped()}, dst={"query": q},
               scale=0.125)
        assert text in kernel.last_variant.lowering
