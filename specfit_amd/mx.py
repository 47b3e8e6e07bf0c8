"""Tensors in microscaled 8 and 4 bits, as ``ops.mx_quantize`` and
``ops.mx_quantize_weight`` make them and ``ops.mx_linear`` multiplies them.

32 neighbours of a row share the scale 2^e, held as the byte e + 127, with e
the least integer from -127 up at which no value rounds past the type's
largest; values are rounded to nearest, ties to even.  A block that held an
infinity or a NaN has the byte 255 and reads as NaN.  ``MXRows`` keeps the
codes row by row, ``MXWeight`` in the order in which the matrix instructions
read them (csrc/mx.h); ``blocks`` and ``from_blocks`` translate to and from the
plain order in which checkpoints hold microscaled weights.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

BLOCK = 32
TILE = 128


def _up(n: int, to: int) -> int:
    return -(-n // to)


def _rows(shape: tuple) -> int:
    n = 1
    for s in shape[:-1]:
        n *= s
    return n


@functools.lru_cache(maxsize=256)
def row_bytes(dim: int) -> tuple[int, int]:
    """Bytes of codes and of scales that one of MXRows' rows takes."""
    return _up(dim, TILE) * TILE, _up(dim, 4 * TILE) * 16


def weight_bytes(rows: int, dim: int) -> tuple[int, int]:
    """Bytes of codes and of scales of an MXWeight."""
    tiles = _up(rows, 32) * 2
    return tiles * _up(dim, TILE) * 1024, tiles * _up(dim, 4 * TILE) * 256


def _check(name: str, t: torch.Tensor, nbytes: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or not t.is_contiguous() \
            or t.numel() != nbytes:
        raise ValueError(f"{name} must be {nbytes} contiguous uint8")


class MXRows:
    """Activations in e4m3: ``shape`` [..., dim], ``dtype`` the type they came
    in, which a product with them gives too (of fp32 the caller names one).
    Whoever makes ``codes`` and ``scales`` leaves zeros behind a row's end in its
    last tile of 128: a product reads them."""

    __slots__ = ("shape", "dtype", "rows", "dim", "_codes", "_scales", "_both")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple,
                 dtype: torch.dtype) -> None:
        shape = tuple(shape)
        if len(shape) < 1 or shape[-1] < 1:
            raise ValueError("rows must have at least one column")
        self.shape, self.dtype, self.dim = shape, dtype, shape[-1]
        self.rows = _rows(shape)
        code, scale = row_bytes(self.dim)
        _check("codes", codes, self.rows * code)
        _check("scales", scales, self.rows * scale)
        if codes.device != scales.device:
            raise ValueError("codes and scales must share a device")
        self._codes, self._scales, self._both = codes, scales, None

    @classmethod
    def _of(cls, both: torch.Tensor, shape: tuple, rows: int, dtype: torch.dtype) -> "MXRows":
        """Over one buffer, the codes in front (what the operators make: a
        call that only passes them on makes no views)."""
        new = cls.__new__(cls)
        new.shape, new.dtype, new.rows, new.dim = shape, dtype, rows, shape[-1]
        new._codes = new._scales = None
        new._both = both
        return new

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._both[:self.rows * row_bytes(self.dim)[0]]
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._both[self.rows * row_bytes(self.dim)[0]:]
        return self._scales

    @property
    def device(self) -> torch.device:
        return (self._codes if self._both is None else self._both).device

    def _pointers(self) -> tuple[int, int]:
        """Addresses of the codes and of the scales."""
        if self._both is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        at = self._both.data_ptr()
        return at, at + self.rows * row_bytes(self.dim)[0]

    def values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values held, [..., dim] (exact in any of the three types but for
        the ends of fp16's range)."""
        from . import ops

        return ops.mx_values(self, dtype)

    def blocks(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes uint8 [rows, dim], scale bytes [rows, ceil(dim / 32)])."""
        code, scale = row_bytes(self.dim)
        codes = self.codes.view(self.rows, code)[:, :self.dim]
        scales = self.scales.view(self.rows, scale // 16, 4, 4).transpose(2, 3)
        return (codes.contiguous(),
                scales.reshape(self.rows, scale)[:, :_up(self.dim, BLOCK)].contiguous())


@dataclass(frozen=True, eq=False)
class MXWeight:
    """A weight [rows, dim] in e2m1.  Whoever makes ``codes`` and ``scales``
    (rather than ``from_blocks``) leaves zeros behind a row's end in its last tile."""

    codes: torch.Tensor
    scales: torch.Tensor
    rows: int
    dim: int

    def __post_init__(self) -> None:
        if self.rows < 1 or self.dim < 1:
            raise ValueError("a weight must have rows and columns")
        code, scale = weight_bytes(self.rows, self.dim)
        _check("codes", self.codes, code)
        _check("scales", self.scales, scale)
        if self.codes.device != self.scales.device:
            raise ValueError("codes and scales must share a device")

    @property
    def shape(self) -> tuple:
        return (self.rows, self.dim)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def _pointers(self) -> tuple[int, int]:
        return self.codes.data_ptr(), self.scales.data_ptr()

    def values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values held, [rows, dim]."""
        from . import ops

        return ops.mx_values(self, dtype)

    def to(self, device: torch.device | str) -> "MXWeight":
        return MXWeight(self.codes.to(device), self.scales.to(device), self.rows, self.dim)

    @classmethod
    def from_blocks(cls, codes: torch.Tensor, scales: torch.Tensor, dim: int) -> "MXWeight":
        """From the plain order: codes uint8 [rows, ceil(dim / 32) * 16], the
        first of two values in a byte's low half, and scale bytes [rows,
        ceil(dim / 32)].  Codes behind a row's end are taken as zeros."""
        n = _up(dim, BLOCK)
        if dim < 1 or codes.dim() != 2 or codes.dtype != torch.uint8 or codes.shape[1] != 16 * n:
            raise ValueError("codes must be uint8 [rows, ceil(dim / 32) * 16]")
        rows = codes.shape[0]
        if rows < 1 or scales.dtype != torch.uint8 or scales.shape != (rows, n) \
                or scales.device != codes.device:
            raise ValueError("scales must be uint8 [rows, ceil(dim / 32)] beside the codes")
        if dim % BLOCK:
            codes = codes.clone()
            codes[:, (dim + 1) // 2:] = 0
            if dim % 2:
                codes[:, dim // 2] &= 15
        tiles, quads, row_tiles = _up(dim, TILE), _up(dim, 4 * TILE), _up(rows, 32) * 2
        c = codes.new_zeros((row_tiles * 16, tiles * 64))
        c[:rows, :16 * n] = codes
        c = c.view(row_tiles, 16, tiles, 4, 16).permute(0, 2, 3, 1, 4)
        s = scales.new_zeros((row_tiles * 16, quads * 16))
        s[:rows, :n] = scales
        s = s.view(row_tiles, 16, quads, 4, 4).permute(0, 2, 4, 1, 3)
        return cls(c.reshape(-1), s.reshape(-1), rows, dim)

    def blocks(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes, scale bytes) in ``from_blocks``' order."""
        n = _up(self.dim, BLOCK)
        tiles, quads, row_tiles = _up(self.dim, TILE), _up(self.dim, 4 * TILE), _up(self.rows, 32) * 2
        c = self.codes.view(row_tiles, tiles, 4, 16, 16).permute(0, 3, 1, 2, 4)
        s = self.scales.view(row_tiles, quads, 4, 16, 4).permute(0, 3, 1, 4, 2)
        return (c.reshape(row_tiles * 16, tiles * 64)[:self.rows, :16 * n].contiguous(),
                s.reshape(row_tiles * 16, quads * 16)[:self.rows, :n].contiguous())
