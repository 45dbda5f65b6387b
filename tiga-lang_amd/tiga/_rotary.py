"""``tg.nn.norm_rotary`` on csrc/tgx_rotary.hip, and on Torch operations for
host tensors and the shapes the kernels do not take."""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _native
from ._dual import carries_tangent

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


def _steps(t: torch.Tensor) -> tuple[int, int]:
    """Strides of tokens and heads; 0 where there is one, whose stride may be any."""
    (n, heads, _), s = t.shape, t.stride()
    return s[0] if n > 1 else 0, s[1] if heads > 1 else 0


def _rows_ok(t: torch.Tensor) -> bool:
    """Rows are dense and start on two values, counted from the tensor's start."""
    if t.numel() == 0:
        return True
    token, head = _steps(t)
    return t.stride(2) == 1 and token % 2 == 0 and head % 2 == 0


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` with dense rows that start on two values."""
    if not _rows_ok(t):
        t = t.contiguous()
    return t if t.data_ptr() % (2 * t.element_size()) == 0 else \
        t.clone(memory_format=torch.contiguous_format)


def _struct(form: Form, query, key, query_weight, key_weight, positions,
            frequencies) -> _native.NormRotary:
    """The native operands but for their pointers."""
    p = _native.NormRotary()
    for i, x in enumerate((query, key)):
        if x is not None:
            p.token_stride[i], p.head_stride[i] = _steps(x)
            p.heads[i] = x.shape[1]
    p.w_dtype = next((_DTYPES[w.dtype] for w in (query_weight, key_weight) if w is not None), 2)
    p.positions_bits = _native.idx_bits(positions)
    p.axes = len(form.sections)
    for i, n in enumerate(form.sections):
        p.sections[i] = n
    p.n_freqs = frequencies.numel()
    p.norm, p.interleaved, p.eps = int(form.norm), int(form.interleaved), form.eps
    p.n_tokens, p.D = query.shape[0], query.shape[-1]
    p.dtype = _DTYPES[query.dtype]
    return p


class Plan:
    """What norm_rotary found for operands of some types, shapes and strides:
    the form, whether the kernels take them, and the native operands of
    rows that need no copy."""

    def __init__(self, form: Form, query, key, query_weight, key_weight, positions, frequencies):
        self.form = form
        self.covered = covered(form, query, key, (query_weight, key_weight))
        self.template, self.mask = None, 0
        self.work_bytes = None      # of the backward pass, asked at its first use
        if self.covered and _rows_ok(query) and (key is None or _rows_ok(key)):
            self.template = _struct(form, query, key, query_weight, key_weight, positions,
                                    frequencies)
            self.mask = 2 * query.element_size() - 1


def _operands(plan: Plan, query, key, query_weight, key_weight, positions, frequencies):
    """The native operands, and the tensors they point into."""
    q_at, k_at = query.data_ptr(), 0 if key is None else key.data_ptr()
    if plan.template is None or (q_at | k_at) & plan.mask:
        query, key = _rows(query), None if key is None else _rows(key)
        q_at, k_at = query.data_ptr(), 0 if key is None else key.data_ptr()
        p = _struct(plan.form, query, key, query_weight, key_weight, positions, frequencies)
    else:
        p = _native.NormRotary.from_buffer_copy(plan.template)
    p.x_dev[0], p.x_dev[1] = q_at, k_at or None
    if query_weight is not None:
        query_weight = query_weight.contiguous()
        p.w_dev[0] = query_weight.data_ptr()
    if key_weight is not None:
        key_weight = key_weight.contiguous()
        p.w_dev[1] = key_weight.data_ptr()
    p.positions_dev, p.freqs_dev = positions.data_ptr(), frequencies.data_ptr()
    return p, (query, key, query_weight, key_weight, positions, frequencies)


def forward(plan: Plan, query, key, query_weight, key_weight, positions, frequencies):
    p, keep = _operands(plan, query, key, query_weight, key_weight, positions, frequencies)
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    key_out = None if key is None else torch.empty(key.shape, dtype=key.dtype, device=key.device)
    _native.launch(query, "tgx_norm_rotary_fwd", ctypes.byref(p), out.data_ptr(),
                   None if key is None else key_out.data_ptr())
    return out, key_out


class NormRotaryFunction(torch.autograd.Function):
    """(query, key) normed and rotated; gradients of query, key and weights."""

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, positions, frequencies, plan):
        ctx.plan = plan
        ctx.save_for_backward(query, key, query_weight, key_weight, positions, frequencies)
        ctx.set_materialize_grads(True)
        outs = forward(plan, query, key, query_weight, key_weight, positions, frequencies)
        return outs[0] if key is None else outs

    @staticmethod
    @once_differentiable
    def backward(ctx, *douts):
        query, key, query_weight, key_weight, positions, frequencies = ctx.saved_tensors
        p, keep = _operands(ctx.plan, query, key, query_weight, key_weight, positions,
                            frequencies)
        pair = 2 * query.element_size()
        given, grads = [None, None], [None, None]   # of the outputs; of query and key
        for i, (t, d) in enumerate(zip((query, key), douts)):
            d = (d if d.dtype == t.dtype else d.to(t.dtype)).contiguous()
            given[i] = d if d.data_ptr() % pair == 0 else d.clone()
            grads[i] = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        dw = [torch.empty(w.shape, dtype=w.dtype, device=w.device)
              if w is not None and need else None
              for w, need in zip((query_weight, key_weight), ctx.needs_input_grad[2:4])]
        work, size = None, 0
        if dw[0] is not None or dw[1] is not None:
            size = ctx.plan.work_bytes
            if size is None:
                asked = ctypes.c_size_t()
                _native.call("tgx_norm_rotary_bwd_workspace", ctypes.byref(p),
                             ctypes.byref(asked))
                size = ctx.plan.work_bytes = asked.value
            work = torch.empty(size, dtype=torch.uint8, device=query.device)
        _native.launch(query, "tgx_norm_rotary_bwd", ctypes.byref(p),
                       *[None if t is None else t.data_ptr() for t in (*given, *grads, *dw, work)],
                       size)
        return (*grads, *dw, None, None, None)


def apply(plan: Plan, query, key, query_weight, key_weight, positions, frequencies):
    if not plan.covered:
        return reference(plan.form, query, key, query_weight, key_weight, positions, frequencies)
    if carries_tangent(query, key, query_weight, key_weight, frequencies):
        raise NotImplementedError("norm_rotary has no forward-mode derivative on the HIP kernels")
    if torch.is_grad_enabled() and (
            query.requires_grad or (key is not None and key.requires_grad) or
            (query_weight is not None and query_weight.requires_grad) or
            (key_weight is not None and key_weight.requires_grad)):
        return NormRotaryFunction.apply(query, key, query_weight, key_weight, positions,
                                        frequencies, plan)
    outs = forward(plan, query, key, query_weight, key_weight, positions, frequencies)
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
