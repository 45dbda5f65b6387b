"""Forward-mode differentiation and launches that know nothing of it."""

from __future__ import annotations

from torch.autograd import forward_ad


def carries_tangent(*tensors) -> bool:
    """Whether one of these tensors (None among them) carries a tangent, which
    a launch on its data pointer would drop without a word."""
    # (No level is open in an ordinary call, which pays for a comparison.)
    if forward_ad._current_level < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
