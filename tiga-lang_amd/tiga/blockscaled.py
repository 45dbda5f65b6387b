"""``tiga.BlockScaled``: a cache's rows as 8-bit codes, with one scale for
each block of slots and head."""

from __future__ import annotations

import torch

# Code types and TGX_CODE_* of the kernels.
CODES = {torch.float8_e4m3fn: 1, torch.int8: 2}
# The largest code M, and the power of two above it.
LARGEST = {torch.float8_e4m3fn: (448.0, 9), torch.int8: (127.0, 7)}


class BlockScaled:
    """Rows of a cache held in 8 bits: row (slot, h) is

        codes[slot, h, :] * scales[slot // block, h].

    codes [slots, heads, D] (or [slots, heads, 1, D]: `grouped`) of type
    torch.float8_e4m3fn or torch.int8, strided as they come but for their dense
    last dimension; scales [slots / block, heads] fp32, contiguous.  With
    ``tables=T`` the rows are ``slot * T + t`` and the scales
    [slots / block * T, heads], as a paged relation with a table per head counts
    its sources (`per_head`).

    ``Graph.append`` writes such caches, ``Graph.read`` reads them back, and
    attention over ``Graph.paged`` takes them as its key and value fields; every
    other edge function over a paged relation sees them as `dequantize` gives
    them.  The tensors are the caller's: their contents are read as they stand,
    which tensors they are is fixed.

    A scale may be any finite number; `append` stores by powers of two, and a
    block that holds a NaN or an infinity by the scale NaN, with which all of
    its rows read back as NaN."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, *, block: int, tables: int = 1):
        for name, t in (("codes", codes), ("scales", scales)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
        if codes.dtype not in CODES:
            raise TypeError(f"codes must be float8_e4m3fn or int8, got {codes.dtype}")
        if scales.dtype != torch.float32:
            raise TypeError(f"scales must be float32, got {scales.dtype}")
        for name, n in (("block", block), ("tables", tables)):
            if not isinstance(n, int) or isinstance(n, bool) or n < 1:
                raise ValueError(f"{name} must be a positive integer")
        if codes.ndim not in (3, 4) or (codes.ndim == 4 and codes.shape[2] != 1):
            raise ValueError("codes must be [slots, heads, D] or [slots, heads, 1, D], got "
                             f"{tuple(codes.shape)}")
        if codes.shape[0] % (block * tables):
            raise ValueError(f"codes of {codes.shape[0]} rows are no whole blocks of {block} slots")
        want = (codes.shape[0] // block, codes.shape[1])
        if tuple(scales.shape) != want or not scales.is_contiguous():
            raise ValueError(f"scales must be contiguous {list(want)}, got {tuple(scales.shape)}")
        if scales.device != codes.device:
            raise ValueError(f"scales are on {scales.device}, codes on {codes.device}")
        if codes.shape[-1] > 1 and codes.stride(-1) != 1:
            raise ValueError("the rows of codes must be dense")
        vars(self).update(
            codes=codes, scales=scales, block=block, tables=tables,
            # Whether rows start a multiple of 8 bytes from the first.
            eights=all(n <= 1 or s % 8 == 0 for n, s in zip(codes.shape[:-1], codes.stride())),
            # What a launch depends on beside the contents and addresses.
            spec=(codes.dtype, codes.shape, codes.stride(), codes.device, scales.shape, block,
                  tables))

    def __setattr__(self, name, value):
        # (Launches go by what was checked here.)
        raise AttributeError(f"a BlockScaled's {name} is fixed: write into its tensors, or make "
                             "another of others")

    def __delattr__(self, name):
        self.__setattr__(name, None)

    @classmethod
    def zeros(cls, slots: int, heads: int, width: int, *, block: int,
              dtype: torch.dtype = torch.float8_e4m3fn, device=None) -> "BlockScaled":
        """An empty cache of `slots` rows of `heads` * `width` values."""
        if dtype not in CODES:
            raise TypeError(f"dtype must be float8_e4m3fn or int8, got {dtype}")
        if not isinstance(block, int) or block < 1 or slots % block:
            raise ValueError(f"{slots} slots are no whole blocks of {block}")
        codes = torch.zeros(slots, heads, width, dtype=torch.int8, device=device).view(dtype)
        return cls(codes, torch.zeros(slots // block, heads, device=device), block=block)

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def ndim(self) -> int:
        return self.codes.ndim

    @property
    def dtype(self) -> torch.dtype:
        """The codes' type."""
        return self.codes.dtype

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def requires_grad(self) -> bool:
        return self.scales.requires_grad

    def grouped(self) -> "BlockScaled":
        """The rows as [slots, heads, 1, D], for query heads grouped on key heads."""
        if self.ndim == 4:
            return self
        return BlockScaled(self.codes[:, :, None], self.scales, block=self.block,
                           tables=self.tables)

    def per_head(self) -> "BlockScaled":
        """The same memory as rows of (slot, head), [slots * heads, 1, D]: the
        sources of a relation that `Graph.select_pages` returns."""
        if self.tables != 1:
            raise ValueError("the rows are counted by head already")
        slots, heads, D = self.shape[0], self.shape[1], self.shape[-1]
        try:
            codes = self.codes.view(slots * heads, 1, D)
        except RuntimeError:
            raise ValueError("codes whose heads do not follow each other cannot be counted by "
                             "head") from None
        return BlockScaled(codes, self.scales.view(-1, 1), block=self.block, tables=heads)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The rows' values, formed in fp32 (fp64 for float64) and rounded once."""
        wide = torch.promote_types(dtype, torch.float32)
        blocks = self.scales.view(-1, self.tables, self.shape[1])
        scales = blocks.repeat_interleave(self.block, 0).view(*self.shape[:2],
                                                              *(1,) * (self.ndim - 2))
        return (self.codes.to(wide) * scales).to(dtype)

    def __repr__(self) -> str:
        return (f"BlockScaled({str(self.dtype).split('.')[-1]} {list(self.shape)}, "
                f"block={self.block}, device={self.device})")


def power_of_two(exponent: torch.Tensor) -> torch.Tensor:
    """2^exponent in fp32 for whole numbers in [-126, 127], by its bits."""
    return ((exponent.to(torch.int32) + 127) << 23).view(torch.float32)


def scale_of(amax: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The scale of a block of largest magnitude `amax` (fp32): the smallest
    power of two s >= 2^-126 with amax <= M s, NaN for a NaN or an infinity."""
    largest, shift = LARGEST[dtype]
    finite = torch.isfinite(amax)
    part, exponent = torch.frexp(torch.where(finite, amax, 1.0))
    exponent = torch.where(amax == 0, -126, exponent - shift + (part > largest / 2 ** shift))
    return torch.where(finite, power_of_two(exponent.clamp(min=-126)), torch.nan)


def encode(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """fp32 values of at most M as codes, to the nearest, ties to even; a NaN as 0."""
    x = torch.where(torch.isnan(x), 0.0, x)
    return (torch.round(x) if dtype == torch.int8 else x).to(dtype)


__all__ = ["BlockScaled"]
