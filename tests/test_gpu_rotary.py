"""tg.nn.norm_rotary on the HIP kernels, forward and backward, against the
formula in float64: types, widths, partial and several-axis rotation, strides,
far positions, captured passes."""

import numpy as np
import pytest
import torch

import tiga as tg

import paged_reference as want

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F32 = 2.0 ** -24


@pytest.fixture(autouse=True)
def _strict():
    tg.config.strict = True
    yield
    tg.config.strict = False


f64 = lambda t: t.detach().double().cpu().numpy()


def make(n, hq, hk, D, sections, dtype, seed=0, far=5000, wdtype=None, bits=64):
    rng = np.random.default_rng(seed)
    half = sum(sections)
    freqs = torch.tensor(10000.0 ** (-np.arange(half) / max(half, 1)), device=DEV).float()
    pos = torch.tensor(rng.integers(-far, far, size=(n, len(sections))), device=DEV,
                       dtype=torch.int64 if bits == 64 else torch.int32)
    qkv = torch.tensor(rng.standard_normal((n, hq + 2 * hk, D)), device=DEV).to(dtype)
    q, k = (t.detach().requires_grad_(True) for t in (qkv[:, :hq], qkv[:, hq:hq + hk]))
    w = [torch.tensor(1 + 0.2 * rng.standard_normal(D), device=DEV).to(wdtype or dtype)
         .requires_grad_(True) for _ in range(2)]
    dy = [torch.tensor(rng.standard_normal((n, h, D)), device=DEV).to(dtype) for h in (hq, hk)]
    return q, k, w, pos, freqs, dy


def check(n, hq, hk, D, sections, dtype, interleaved=False, norm=True, eps=1e-6, **kw):
    print(f"rotary {dtype} n={n} heads={hq},{hk} D={D} {sections} inter={interleaved} "
          f"norm={norm}", flush=True)
    q, k, w, pos, freqs, dy = make(n, hq, hk, D, sections, dtype, **kw)
    weights = dict(query_weight=w[0], key_weight=w[1]) if norm else {}
    outs = tg.nn.norm_rotary(q, k, pos, freqs, norm=norm, eps=eps, sections=sections,
                             interleaved=interleaved, **weights)
    with torch.no_grad():
        again = tg.nn.norm_rotary(q, k, pos, freqs, norm=norm, eps=eps, sections=sections,
                                  interleaved=interleaved, **weights)
    assert all(torch.equal(a, b) for a, b in zip(outs, again))
    leaves = (q, k, *w) if norm else (q, k)
    grads = torch.autograd.grad(outs, leaves, dy)
    angle = want.angles(pos.cpu().numpy(), freqs.cpu().numpy(), sections)
    half = torch.finfo(dtype).eps / 2
    # Angles in 64 bits: one rounding of 2^-53 of the angle in the oracle's product,
    # three in the kernel's (the product, 1 / 2 pi and the product with it).
    turn = 4 * 2.0 ** -53 * (np.abs(angle).max() if angle.size else 0.0)
    for i, (x, h) in enumerate(((q, hq), (k, hk))):
        assert outs[i].dtype == dtype and grads[i].dtype == dtype
        xw, xx, xd = f64(w[i]) if norm else None, f64(x), f64(dy[i])
        exp = want.norm_rotary(xx, xw, angle, eps, norm, interleaved)
        dx, dw = want.norm_rotary_grad(xx, xw, angle, eps, norm, interleaved, xd)
        if exp.size == 0:
            continue
        # Half a step of the result, and of the some 16 fp32 operations on the way
        # (products, a sine to 4 half steps, the mean of D squares in D / 16 + 4
        # additions a lane) that each move a value of the row's largest size.
        ops = 24 + D / 16
        assert (np.abs(f64(outs[i]) - exp) <= half * np.abs(exp) + (ops * F32 + turn) *
                np.abs(exp).max(-1, keepdims=True) * 2).all()
        big = np.abs(dx).max(-1, keepdims=True)
        r = 1 / np.sqrt((xx ** 2).mean(-1, keepdims=True) + eps) if norm else 1.0
        # dx = r (h - n mean(h n)): both terms may be larger than their difference.
        hn = np.abs(xd).max(-1, keepdims=True) * 2 * (np.abs(xw).max() if norm else 1) * r * \
            (1 + (np.abs(xx) * r).max(-1, keepdims=True) ** 2 if norm else 1)
        assert (np.abs(f64(grads[i]) - dx) <= half * np.abs(dx) + (ops * F32 + turn) *
                (big + hn)).all()
        if norm:
            # n * heads terms, added in fp32 by lanes, waves and workgroups; the
            # sum of the terms' sizes bounds what the roundings of all levels move.
            g = want.rotate(xd, angle, interleaved, -1.0)
            size = (np.abs(g) * np.abs(xx * r)).sum((0, 1))
            depth = min(n * h, 4096) / 4 + n * h / 4096 + 64
            got, whalf = f64(grads[2 + i]), torch.finfo(w[i].dtype).eps / 2
            assert (np.abs(got - dw) <= whalf * np.abs(dw) + ((ops + depth) * F32 + turn) *
                    2 * size).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,sections", [
    (32, (16,)), (64, (32,)), (64, (16,)), (80, (40,)), (96, (16, 16, 16)), (128, (64,)),
    (128, (16, 24, 24)), (192, (96,)), (256, (128,)), (256, (24, 40)), (128, (0,)),
    (4, (2,)), (20, (4, 2)), (100, (50,)), (64, (10,)), (132, (20, 2, 10, 4))])
def test_forward_and_gradients(dtype, interleaved, D, sections):
    check(37, 5, 2, D, sections, TYPES[dtype], interleaved=interleaved)


@pytest.mark.parametrize("n", [0, 1, 2, 3, 63, 4095, 4097])
def test_token_counts(n):
    check(n, 6, 2, 64, (32,), torch.bfloat16)
    check(n, 3, 1, 20, (10,), torch.float32)


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 0), (32, 8), (7, 13)])
def test_head_counts(hq, hk):
    check(65, hq, hk, 128, (64,), torch.bfloat16)
    check(65, hq, hk, 128, (64,), torch.float16, norm=False, interleaved=True)


def test_other_forms():
    check(33, 3, 2, 64, (32,), torch.bfloat16, wdtype=torch.float32)
    check(33, 3, 2, 64, (32,), torch.float32, wdtype=torch.bfloat16)
    check(33, 3, 2, 64, (32,), torch.float16, bits=32)
    check(33, 3, 2, 64, (8, 8, 8, 8), torch.float32, far=2 ** 40, eps=0.0)


def test_rows_on_odd_addresses_and_query_alone():
    q, k, w, pos, freqs, dy = make(9, 4, 2, 64, (32,), torch.bfloat16)
    outs = tg.nn.norm_rotary(q, k, pos, freqs, query_weight=w[0], key_weight=w[1])
    for shift in (1, 2):
        odd = torch.zeros(9 * 4 * 80 + shift, device=DEV, dtype=torch.bfloat16)
        view = torch.as_strided(odd, (9, 4, 64), (4 * 80, 80, 1), shift).copy_(q.detach())
        got = tg.nn.norm_rotary(view, k, pos, freqs, query_weight=w[0], key_weight=w[1])
        assert (got[0] - outs[0]).abs().max() <= outs[0].abs().max() * 2.0 ** -8
    across = q.detach().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(tg.nn.norm_rotary(across, None, pos[:, 0], freqs, query_weight=w[0]),
                       outs[0])
    wide = q.detach().transpose(1, 2).contiguous().transpose(1, 2)   # width not dense
    assert torch.equal(tg.nn.norm_rotary(wide, None, pos, freqs, query_weight=w[0]), outs[0])
    # Gradients where only some are wanted, or the output's is missing or expanded.
    part = tg.nn.norm_rotary(q, k.detach(), pos, freqs, query_weight=w[0].detach(),
                             key_weight=w[1])
    full = tg.nn.norm_rotary(q, k, pos, freqs, query_weight=w[0], key_weight=w[1])
    one = torch.ones((), device=DEV, dtype=torch.bfloat16).expand_as(part[0])
    a = torch.autograd.grad(part[0], (q, w[1]), one, allow_unused=True)
    b = torch.autograd.grad(full, (q, w[1]), (one.contiguous(), torch.zeros_like(part[1])))
    assert torch.equal(a[0], b[0]) and (a[1] is None or not a[1].any())


@pytest.mark.parametrize("dtype", TYPES)
def test_one_layout_on_even_and_odd_addresses(dtype):
    """Rows of one shape and strides, forward and back, wherever they start."""
    dtype = TYPES[dtype]
    q, k, w, pos, freqs, dy = make(9, 4, 2, 64, (32,), dtype)
    results = []
    for shift in (0, 1, 0, 3):
        leaves = []
        for x in (q, k):
            room = torch.zeros(x.numel() + shift, device=DEV, dtype=dtype)[shift:]
            leaves.append(room.view(x.shape).copy_(x.detach()).requires_grad_(True))
        outs = tg.nn.norm_rotary(*leaves, pos, freqs, query_weight=w[0], key_weight=w[1])
        results.append((*outs, *torch.autograd.grad(outs, (*leaves, *w), dy)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_calls_of_one_shape_keep_their_own_forms():
    q, k, w, pos, freqs, dy = make(7, 2, 2, 32, (16,), torch.float32)
    for forms in (dict(eps=1e-6), dict(eps=0.5), dict(interleaved=True), dict(norm=False),
                  dict(sections=(16,)), dict(eps=1e-6)):
        weights = dict(query_weight=w[0], key_weight=w[1]) if forms.get("norm", True) else {}
        got = tg.nn.norm_rotary(q, k, pos, freqs, **forms, **weights)
        same = tg.nn.norm_rotary(q.cpu(), k.cpu(), pos.cpu(), freqs.cpu(), **forms,
                                 **{name: x.cpu() for name, x in weights.items()})
        for a, b in zip(got, same):
            assert (a.cpu() - b).abs().max() <= 64 * F32 * b.abs().max()


def test_what_no_kernel_covers():
    q = torch.randn(3, 2, 6, device=DEV)
    pos, freqs = torch.arange(3, device=DEV), torch.ones(3, device=DEV)
    with pytest.raises(RuntimeError, match="no HIP kernel"):
        tg.nn.norm_rotary(q, None, pos, freqs)
    tg.config.strict = False
    got = tg.nn.norm_rotary(q, None, pos, freqs)
    exp = tg.nn.norm_rotary(q.cpu(), None, pos.cpu(), freqs.cpu())
    assert (got.cpu() - exp).abs().max() <= 16 * F32 * exp.abs().max()


def test_captured_forward_and_backward_replay_on_new_values():
    q, k, w, pos, freqs, dy = make(50, 4, 2, 128, (64,), torch.bfloat16)
    call = lambda: tg.nn.norm_rotary(q, k, pos, freqs, query_weight=w[0], key_weight=w[1])

    def both():
        outs = call()
        return (*outs, *torch.autograd.grad(outs, (q, k, *w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = both()
    for step in range(4):
        with torch.no_grad():
            for t in (q, k, *dy):
                t.mul_(-1.25)
            pos.add_(3)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, both()):
            assert torch.equal(a, b)


def test_training_attention_on_normed_and_rotated_fields():
    """norm_rotary into varlen attention and back: the gradients of its inputs
    from the attention's own, by the formula."""
    class Attention(tg.MessagePassing):
        reducer = tg.online_softmax()

        def edge(self, src, dst, edge, scale):
            return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)

    lengths, H, D = [40, 1, 90], 2, 64
    n = sum(lengths)
    q, k, w, _, freqs, dy = make(n, H, H, D, (32,), torch.float16)
    pos = torch.cat([torch.arange(l, device=DEV) for l in lengths])
    v = torch.randn(n, H, D, device=DEV).half()
    graph = tg.Graph.cat([tg.Graph.triangular(l, device=DEV) for l in lengths])
    qr, kr = tg.nn.norm_rotary(q, k, pos, freqs, query_weight=w[0], key_weight=w[1])
    kernel = Attention()
    out = kernel(graph=graph, src={"key": kr, "value": v}, dst={"query": qr}, scale=D ** -0.5)
    assert kernel.last_variant.pattern == "block-attention"
    mid = torch.autograd.grad(out, (qr, kr), dy[0], retain_graph=True)
    got = torch.autograd.grad(out, (q, k, *w), dy[0])
    angle = want.angles(pos.cpu().numpy()[:, None], freqs.cpu().numpy(), (32,))
    for i, x in enumerate((q, k)):
        dx, dw = want.norm_rotary_grad(f64(x), f64(w[i]), angle, 1e-6, True, False, f64(mid[i]))
        # (As in `check`, relative to the largest value.)
        assert np.abs(f64(got[i]) - dx).max() <= (2.0 ** -11 + 200 * F32) * np.abs(dx).max()
        assert np.abs(f64(got[2 + i]) - dw).max() <= (2.0 ** -11 + 200 * F32) * np.abs(dw).max()


def same_kind(got, exp):
    """NaN, Inf and -Inf in the same places."""
    return all(np.array_equal(kind(got), kind(exp))
               for kind in (np.isnan, np.isposinf, np.isneginf))


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,half,dtype", [
    (8, 2, "f32"), (64, 16, "bf16"), (64, 10, "f16"), (128, 32, "f32"), (20, 6, "bf16"),
    (64, 0, "bf16"), (64, 2, "f32"), (256, 64, "f16")])
def test_infinite_values_in_columns_that_are_not_rotated(D, half, dtype, interleaved, norm):
    """They come out as the formula has them, and reach no other column but
    through the norm; the same of output gradients on the way back."""
    n, h = 2 * (D - 2 * half) + 1, 3
    q, _, w, pos, freqs, dy = make(n, h, 0, D, (half,), TYPES[dtype])
    weights = dict(query_weight=w[0]) if norm else {}
    call = lambda x: tg.nn.norm_rotary(x, None, pos, freqs, norm=norm, interleaved=interleaved,
                                       **weights)

    def spoiled(x):
        """Token 2 i has an Inf, 2 i + 1 a -Inf in column 2 half + i of its first
        head, and every third token a NaN there in its second."""
        x = x.detach().clone()
        for t in range(n - 1):
            x[t, 0, 2 * half + t // 2] = float("-inf") if t % 2 else float("inf")
            if t % 3 == 0:
                x[t, 1, 2 * half + t // 2] = float("nan")
        return x

    angle = want.angles(pos.cpu().numpy(), freqs.cpu().numpy(), (half,))
    xw, step = f64(w[0]) if norm else None, torch.finfo(TYPES[dtype]).eps / 2
    # (As in `check`; a row's finite values are those of a clean row, or zero.)
    ops, turn = 24 + D / 16, 4 * 2.0 ** -53 * np.abs(angle).max(initial=0.0)
    with np.errstate(invalid="ignore"):
        x = spoiled(q)
        exp = want.norm_rotary(f64(x), xw, angle, 1e-6, norm, interleaved)
        got = f64(call(x))
        assert same_kind(got, exp)
        fin = np.isfinite(exp)
        top = np.where(fin, np.abs(exp), 0.0)
        lim = step * top + (ops * F32 + turn) * 2 * top.max(-1, keepdims=True)
        assert (np.abs(got - exp)[fin] <= lim[fin]).all()

        d = spoiled(dy[0])
        leaves = (q, w[0]) if norm else (q,)
        grads = torch.autograd.grad(call(q), leaves, d)
        dx, dw = want.norm_rotary_grad(f64(q), xw, angle, 1e-6, norm, interleaved, f64(d))
        assert same_kind(f64(grads[0]), dx)
        if norm:
            assert same_kind(f64(grads[1]), dw)
        else:
            fin = np.isfinite(dx)
            top = np.where(fin, np.abs(dx), 0.0)
            lim = step * top + (ops * F32 + turn) * 2 * top.max(-1, keepdims=True)
            assert (np.abs(f64(grads[0]) - dx)[fin] <= lim[fin]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 20])
@pytest.mark.parametrize("exponent", [-60, -63, -64, -66, -68])
def test_rows_whose_mean_square_is_below_the_normal_numbers(exponent, D, dtype):
    """eps = 0 and values whose squares are subnormal: the root is finite, and
    the row's norm is that of the same row at an ordinary size."""
    rng = np.random.default_rng(20)
    # Multiples of 2^exponent up to 15: their squares, multiples of 2^-136 at
    # least, and the sum of 64 of them are exact in 32 bits.
    whole = rng.integers(1, 16, size=(5, 3, D)) * rng.choice([-1, 1], size=(5, 3, D))
    q = torch.tensor(whole * 2.0 ** exponent, device=DEV).to(TYPES[dtype]).requires_grad_(True)
    assert np.array_equal(f64(q), whole * 2.0 ** exponent)
    pos = torch.arange(5, device=DEV)
    freqs = torch.tensor(100.0 ** (-np.arange(D // 2) / (D // 2)), device=DEV).float()
    w = torch.tensor(1 + 0.2 * rng.standard_normal(D), device=DEV).to(TYPES[dtype])
    out = tg.nn.norm_rotary(q, None, pos, freqs, query_weight=w, eps=0.0)
    angle = want.angles(pos.cpu().numpy()[:, None], freqs.cpu().numpy(), (D // 2,))
    exp = want.norm_rotary(whole.astype(np.float64), f64(w), angle, 0.0, True, False)
    step = torch.finfo(TYPES[dtype]).eps / 2
    # The mean's product with 1 / D rounds in units of 2^-149; half of one against
    # a mean of 2^-136 or more.  The rest as in `check`.
    mean = (whole.astype(np.float64) ** 2).mean() * 4.0 ** exponent
    mean_off = 2.0 ** -150 / min(mean, 4.0 ** exponent)
    off = (24 + D / 16) * F32 + mean_off
    assert (np.abs(f64(out) - exp) <= step * np.abs(exp) +
            2 * off * np.abs(exp).max(-1, keepdims=True)).all()
    # dx = r (h - n mean(h n)), with r = 2^-exponent times the ordinary row's.
    d = torch.tensor(rng.standard_normal((5, 3, D)), device=DEV).to(TYPES[dtype])
    (dx,) = torch.autograd.grad(out, (q,), d)
    edx, _ = want.norm_rotary_grad(whole.astype(np.float64), f64(w), angle, 0.0, True, False,
                                   f64(d))
    got = f64(dx) * 2.0 ** exponent
    size = np.abs(f64(d)).max() * 2 * np.abs(f64(w)).max() * \
        (1 + 15.0 ** 2) / np.sqrt((whole.astype(np.float64) ** 2).mean(-1)).min()
    assert (np.abs(got - edx) <= step * np.abs(edx) + 2 * off * size).all()


def test_forward_mode_is_refused_on_the_kernels():
    """A launch would drop the tangent without a word."""
    q, k, w, pos, freqs, _ = make(3, 2, 2, 32, (16,), torch.float32)
    args = [t.detach() for t in (q, k, *w, freqs)]
    call = lambda q, k, wq, wk, f: tg.nn.norm_rotary(q, k, pos, f, query_weight=wq, key_weight=wk)
    for i in range(5):
        with torch.autograd.forward_ad.dual_level():
            dual = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t
                    for j, t in enumerate(args)]
            with pytest.raises(NotImplementedError, match="forward"):
                call(*dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
                call(*dual)
            call(*args)     # (a level alone changes nothing)
    call(*args)


def test_one_token_whose_strides_are_odd():
    """The stride of a dimension of one element moves nothing."""
    q, k, w, pos, freqs, _ = make(1, 2, 2, 64, (32,), torch.bfloat16)
    call = lambda q, k: tg.nn.norm_rotary(q, k, pos, freqs, query_weight=w[0], key_weight=w[1])
    exp = call(q, k)
    odd = lambda t: torch.zeros(3, 129, device=DEV, dtype=t.dtype)[:, :128].view(3, 2, 64)[:1] \
        .copy_(t.detach())
    assert odd(q).stride() == (129, 64, 1)
    for a, b in zip(call(odd(q), odd(k)), exp):
        assert torch.equal(a, b)
    one = torch.zeros(1, 2, 65, device=DEV, dtype=q.dtype)[:, :1, :64].copy_(q.detach()[:, :1])
    assert torch.equal(call(one, k)[0], exp[0][:, :1])
