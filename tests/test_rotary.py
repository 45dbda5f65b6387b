"""tg.nn.norm_rotary on host tensors against its formula in float64, its
gradients against the formula's and against differences, and its refusals."""

import numpy as np
import pytest
import torch

import tiga as tg

import paged_reference as want


def inputs(n, hq, hk, D, sections, seed=0, far=1000):
    rng = np.random.default_rng(seed)
    half = sum(sections)
    freqs = (10000.0 ** (-np.arange(half) / max(half, 1))).astype(np.float32)
    positions = rng.integers(-far, far, size=(n, len(sections)))
    mk = lambda *s: rng.standard_normal(s)
    return mk(n, hq, D), mk(n, hk, D), 1 + 0.2 * mk(D), 1 + 0.2 * mk(D), positions, freqs


FORMS = [(8, (4,), False), (8, (4,), True), (12, (2, 1), False), (12, (2, 1, 1), True),
         (6, (0,), False), (10, (1, 0, 3), True)]


@pytest.mark.parametrize("D,sections,interleaved", FORMS)
@pytest.mark.parametrize("norm", [True, False])
def test_forward_and_gradients_match_the_formula(D, sections, interleaved, norm):
    q, k, wq, wk, positions, freqs = inputs(5, 3, 2, D, sections)
    t = lambda x: torch.tensor(x).requires_grad_(True)
    tq, tk, twq, twk = t(q), t(k), t(wq), t(wk)
    weights = dict(query_weight=twq, key_weight=twk) if norm else {}
    outs = tg.nn.norm_rotary(tq, tk, torch.tensor(positions), torch.tensor(freqs), eps=1e-3,
                             norm=norm, sections=sections, interleaved=interleaved, **weights)
    rng = np.random.default_rng(9)
    dy = [rng.standard_normal(o.shape) for o in outs]
    angle = want.angles(positions, freqs, sections)
    grads = torch.autograd.grad(outs, (tq, tk, twq, twk), [torch.tensor(d) for d in dy],
                                allow_unused=True)
    for x, w, out, d, dx, dw in zip((q, k), (wq, wk), outs, dy, grads, grads[2:]):
        exp = want.norm_rotary(x, w, angle, 1e-3, norm, interleaved)
        edx, edw = want.norm_rotary_grad(x, w, angle, 1e-3, norm, interleaved, d)
        # 64-bit arithmetic throughout.
        assert np.abs(out.detach().numpy() - exp).max() <= 1e-12
        assert np.abs(dx.numpy() - edx).max() <= 1e-12
        assert (dw is None) == (not norm)
        if norm:
            assert np.abs(dw.numpy() - edw).max() <= 1e-11


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_gradient_formula_agrees_with_differences(interleaved):
    q, _, w, _, positions, freqs = inputs(2, 2, 1, 8, (2, 1))
    angle = want.angles(positions, freqs, (2, 1))
    d = np.random.default_rng(1).standard_normal(q.shape)
    f = lambda x, w: (want.norm_rotary(x, w, angle, 1e-3, True, interleaved) * d).sum()
    dx, dw = want.norm_rotary_grad(q, w, angle, 1e-3, True, interleaved, d)
    h = 1e-5   # central differences: h^2 times third derivatives of order 10
    for i in np.ndindex(q.shape):
        e = np.zeros_like(q)
        e[i] = h
        assert abs((f(q + e, w) - f(q - e, w)) / (2 * h) - dx[i]) <= 1e-7
    for i in range(8):
        e = np.zeros_like(w)
        e[i] = h
        assert abs((f(q, w + e) - f(q, w - e)) / (2 * h) - dw[i]) <= 1e-7


def test_far_positions_keep_their_angles():
    q, _, _, _, _, freqs = inputs(3, 2, 1, 8, (4,))
    positions = np.array([10 ** 6 + 1, 2 ** 31 - 5, -(10 ** 9)])
    out = tg.nn.norm_rotary(torch.tensor(q).float(), None, torch.tensor(positions),
                            torch.tensor(freqs), norm=False)
    exp = want.norm_rotary(q.astype(np.float32).astype(np.float64), None,
                           want.angles(positions[:, None], freqs, (4,)), 0, False, False)
    # Angles to 1e-6 in 64 bits (2^-53 of 2e9), sines and products in 32.
    assert np.abs(out.numpy() - exp).max() <= (1e-6 + 4 * 2 ** -24) * 2 * np.abs(q).max()


def test_query_alone_and_one_dimensional_positions():
    q, k, wq, wk, positions, freqs = inputs(4, 2, 2, 8, (4,))
    args = torch.tensor(positions[:, 0]), torch.tensor(freqs)
    both = tg.nn.norm_rotary(torch.tensor(q), torch.tensor(k), *args,
                             query_weight=torch.tensor(wq))
    alone = tg.nn.norm_rotary(torch.tensor(q), None, *args, query_weight=torch.tensor(wq))
    assert torch.equal(alone, both[0])
    assert tg.nn.norm_rotary(torch.tensor(q[:0]), None, args[0][:0], args[1]).shape == (0, 2, 8)


def test_refusals():
    q, k = torch.zeros(4, 2, 8), torch.zeros(4, 1, 8)
    pos, freqs, w = torch.arange(4), torch.ones(4), torch.ones(8)
    f = tg.nn.norm_rotary
    with pytest.raises(TypeError, match="query must be"):
        f(None, k, pos, freqs)
    with pytest.raises(ValueError, match="floating-point"):
        f(q[0], k, pos, freqs)
    with pytest.raises(ValueError, match="key"):
        f(q, k.half(), pos, freqs)
    with pytest.raises(ValueError, match="key"):
        f(q, k[:3], pos, freqs)
    with pytest.raises(TypeError, match="positions"):
        f(q, k, pos.float(), freqs)
    with pytest.raises(TypeError, match="frequencies"):
        f(q, k, pos, freqs.double())
    with pytest.raises(ValueError, match="frequencies must be"):
        f(q, k, pos, torch.ones(5))
    with pytest.raises(ValueError, match="positions must be"):
        f(q, k, pos[:3], freqs)
    with pytest.raises(ValueError, match="positions must be"):
        f(q, k, pos[:, None].expand(4, 2), freqs)
    for bad in ((3,), (5, -1), (2, 3)):
        with pytest.raises(ValueError, match="sections"):
            f(q, k, pos[:, None].expand(4, len(bad)), freqs, sections=bad)
    with pytest.raises(ValueError, match="norm=True"):
        f(q, k, pos, freqs, query_weight=w, norm=False)
    with pytest.raises(ValueError, match="query_weight"):
        f(q, k, pos, freqs, query_weight=w[:4])
    with pytest.raises(ValueError, match="needs a key"):
        f(q, None, pos, freqs, key_weight=w)
    with pytest.raises(ValueError, match="eps"):
        f(q, k, pos, freqs, eps=-1.0)
    with pytest.raises(NotImplementedError, match="gradient"):
        f(q, k, pos, freqs.clone().requires_grad_())


def test_forms_go_by_value():
    """A number that a program keeps in a tensor and changes is read at each call."""
    q, _, _, _, positions, freqs = inputs(3, 2, 1, 8, (4,))
    eps, norm = torch.tensor(1e-3), torch.tensor(True)
    call = lambda eps, norm: tg.nn.norm_rotary(torch.tensor(q), None, torch.tensor(positions),
                                               torch.tensor(freqs), eps=eps, norm=norm)
    call(eps, norm)
    eps.fill_(0.5)
    assert torch.equal(call(eps, norm), call(0.5, True))
    norm.fill_(False)
    assert torch.equal(call(eps, norm), call(0.5, False))
