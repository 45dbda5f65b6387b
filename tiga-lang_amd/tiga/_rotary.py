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
    s = t.stride()
    if (s[2] != 1 or s[0] % 2 or s[1] % 2) and t.numel():
        t = t.contiguous()
    return t if t.data_ptr() % (2 * t.element_size()) == 0 else t.clone(memory_format=torch.contiguous_format)


_TEMPLATES: dict[tuple, _native.NormRotary] = {}


def _operands(form: Form, query, key, query_weight, key_weight, positions, frequencies):
    """The native operands, and the tensors they point into."""
    query, key = _rows(query), None if key is None else _rows(key)
    spec = (form, query.dtype, query.shape, query.stride(),
            None if key is None else (key.shape, key.stride()),
            None if query_weight is None else query_weight.dtype,
            None if key_weight is None else key_weight.dtype, positions.dtype)
    template = _TEMPLATES.get(spec)
    if template is None:
        template = _native.NormRotary()
        for i, x in enumerate((query, key)):
            if x is not None:
                template.token_stride[i], template.head_stride[i] = x.stride()[:2]
                template.heads[i] = x.shape[1]
        template.w_dtype = next((_DTYPES[w.dtype] for w in (query_weight, key_weight)
                                 if w is not None), 2)
        template.positions_bits = _native.idx_bits(positions)
        template.axes = len(form.sections)
        for i, n in enumerate(form.sections):
            template.sections[i] = n
        template.n_freqs = frequencies.numel()
        template.norm, template.interleaved = int(form.norm), int(form.interleaved)
        template.eps = form.eps
        template.n_tokens, template.D = query.shape[0], query.shape[-1]
        template.dtype = _DTYPES[query.dtype]
        if len(_TEMPLATES) >= 1024:
            _TEMPLATES.clear()
        _TEMPLATES[spec] = template
    p = _native.NormRotary.from_buffer_copy(template)
    p.x_dev[0] = query.data_ptr()
    if key is not None:
        p.x_dev[1] = key.data_ptr()
    weights = [query_weight, key_weight]
    for i in (0, 1):
        if weights[i] is not None:
            weights[i] = weights[i].contiguous()
            p.w_dev[i] = weights[i].data_ptr()
    p.positions_dev, p.freqs_dev = positions.data_ptr(), frequencies.data_ptr()
    return p, (query, key, *weights, positions, frequencies)


def forward(form: Form, query, key, query_weight, key_weight, positions, frequencies):
    p, keep = _operands(form, query, key, query_weight, key_weight, positions, frequencies)
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    key_out = None if key is None else torch.empty(key.shape, dtype=key.dtype, device=key.device)
    with _native.on_device(query):
        _native.call("tgx_norm_rotary_fwd", ctypes.byref(p), out.data_ptr(),
                     None if key is None else key_out.data_ptr(), _native.stream_of(query))
    return out, key_out


class NormRotaryFunction(torch.autograd.Function):
    """(query, key) normed and rotated; gradients of query, key and weights."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, frequencies, form):
        ctx.form = form
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, frequencies)
        ctx.set_materialize_grads(True)
        outs = forward(form, query, key, query_weight, key_weight, positions, frequencies)
        return outs[0] if key is None else outs

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
    if torch.is_grad_enabled() and any(
            [t is not None and t.requires_grad for t in (query, key, query_weight, key_weight)]):
        return NormRotaryFunction.apply(query, key, query_weight, key_weight, positions,
                                        frequencies, form)
    outs = forward(form, query, key, query_weight, key_weight, positions, frequencies)
    return outs[0] if key is None else outs


def reference(form: Form, query, key, query_weight, key_weight, positions, frequencies):
    """The same on Torch operations: 32 bits (64 for 64-bit tensors), angles
    in 64."""
    half = frequencies.numel()
    axis = torch.repeat_interleave(
        torch.arange(len(form.sections), device=query.device),
        torch.tensor(form.sections, device=query.device), output_size=half)
    positions = positions[:, None] if positions.ndim == 1 else positions
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
