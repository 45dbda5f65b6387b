"""``tg.nn.norm_rotary`` on csrc/tgx_rotary.hip, and on Torch operations for
host tensors and the shapes the kernels do not take."""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _native

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


@dataclass(frozen=True)
class Form:
    """What a call fixes beside its tensors."""

    eps: float
    norm: bool
    sections: tuple[int, ...]
    interleaved: bool


def covered(form: Form, query, key, weights) -> bool:
    """Whether the kernels take these tensors."""
    D, dtype = query.shape[-1], query.dtype
    given = {w.dtype for w in weights if w is not None}
    return (query.is_cuda and dtype in _DTYPES and D % 4 == 0 and 4 <= D <= 256 and
            sum(form.sections) % 2 == 0 and len(form.sections) <= 4 and
            (key is None or key.dtype == dtype) and given <= set(_DTYPES) and len(given) <= 1)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with dense rows that start on two values."""
    pair = 2 * t.element_size()
    if t.numel() and (t.stride(-1) != 1 or t.stride(0) % 2 or t.stride(1) % 2):
        t = t.contiguous()
    return t if t.data_ptr() % pair == 0 else t.clone(memory_format=torch.contiguous_format)


def _operands(form: Form, query, key, query_weight, key_weight, positions, frequencies):
    """The native operands, and the tensors they point into."""
    sides = [None if t is None else _rows(t) for t in (query, key)]
    weights = [None if w is None else w.contiguous() for w in (query_weight, key_weight)]
    p = _native.NormRotary()
    for i, (x, w) in enumerate(zip(sides, weights)):
        if x is not None:
            p.x_dev[i] = x.data_ptr()
            p.token_stride[i], p.head_stride[i] = x.stride(0), x.stride(1)
            p.heads[i] = x.shape[1]
        p.w_dev[i] = _native.ptr(w)
    p.w_dtype = next((_DTYPES[w.dtype] for w in weights if w is not None), 2)
    p.positions_dev, p.freqs_dev = positions.data_ptr(), frequencies.data_ptr()
    p.positions_bits = _native.idx_bits(positions)
    p.axes = len(form.sections)
    for i, n in enumerate(form.sections):
        p.sections[i] = n
    p.n_freqs = frequencies.numel()
    p.norm, p.interleaved, p.eps = int(form.norm), int(form.interleaved), form.eps
    p.n_tokens, p.D = query.shape[0], query.shape[-1]
    p.dtype = _DTYPES[query.dtype]
    return p, (*sides, *weights, positions, frequencies)


def forward(form: Form, query, key, query_weight, key_weight, positions, frequencies):
    p, keep = _operands(form, query, key, query_weight, key_weight, positions, frequencies)
    outs = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
            for t in (query, key)]
    with _native.on_device(query):
        _native.call("tgx_norm_rotary_fwd", ctypes.byref(p), _native.ptr(outs[0]),
                     _native.ptr(outs[1]), _native.stream_of(query))
    return outs


class NormRotaryFunction(torch.autograd.Function):
    """(query, key) normed and rotated; gradients of query, key and weights."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, frequencies, form):
        ctx.form = form
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, frequencies)
        ctx.set_materialize_grads(True)
        outs = forward(form, query, key, query_weight, key_weight, positions, frequencies)
        return outs[0] if key is None else tuple(outs)

    @staticmethod
    @once_differentiable
    def backward(ctx, *douts):
        query, key, query_weight, key_weight, positions, frequencies = ctx.saved_tensors
        p, keep = _operands(ctx.form, query, key, query_weight, key_weight, positions,
                            frequencies)
        pair = 2 * query.element_size()
        dense = []
        for t, d in zip((query, key), douts):
            d = d.to(t.dtype).contiguous()
            dense.append(d if d.data_ptr() % pair == 0 else d.clone())
        grads = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
                 for t in (query, key)]
        dw = [torch.empty_like(w, memory_format=torch.contiguous_format)
              if w is not None and need else None
              for w, need in zip((query_weight, key_weight), ctx.needs_input_grad[2:4])]
        work, size = None, ctypes.c_size_t(0)
        if any(w is not None for w in dw):
            _native.call("tgx_norm_rotary_bwd_workspace", ctypes.byref(p), ctypes.byref(size))
            work = torch.empty(size.value, dtype=torch.uint8, device=query.device)
        dense += [None] * (2 - len(dense))
        with _native.on_device(query):
            _native.call("tgx_norm_rotary_bwd", ctypes.byref(p),
                         *(_native.ptr(t) for t in (*dense, *grads, *dw, work)), size.value,
                         _native.stream_of(query))
        return (*grads, *dw, None, None, None)


def apply(form: Form, query, key, query_weight, key_weight, positions, frequencies):
    tensors = [t for t in (query, key, query_weight, key_weight) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return NormRotaryFunction.apply(query, key, query_weight, key_weight, positions,
                                        frequencies, form)
    outs = forward(form, query, key, query_weight, key_weight, positions, frequencies)
    return outs[0] if key is None else tuple(outs)


def reference(form: Form, query, key, query_weight, key_weight, positions, frequencies):
    """The same on Torch operations: 32 bits (64 for 64-bit tensors), angles
    in 64."""
    half = frequencies.numel()
    axis = torch.repeat_interleave(
        torch.arange(len(form.sections), device=query.device),
        torch.tensor(form.sections, device=query.device), output_size=half)
    angle = (positions.double()[:, axis] * frequencies.double())[:, None]

    def one(x, weight):
        wide = torch.promote_types(x.dtype, torch.float32)
        y = x.to(wide)
        if form.norm:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + form.eps)
            if weight is not None:
                y = y * weight.to(wide)
        c, s = torch.cos(angle).to(wide), torch.sin(angle).to(wide)
        turned, rest = y[..., :2 * half], y[..., 2 * half:]
        if form.interleaved:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        else:
            a, b = turned[..., :half], turned[..., half:]
            turned = torch.cat([a * c - b * s, b * c + a * s], -1)
        return torch.cat([turned, rest], -1).to(x.dtype)

    out = one(query, query_weight)
    return out if key is None else (out, one(key, key_weight))
