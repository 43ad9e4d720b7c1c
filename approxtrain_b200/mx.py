"""Matrices and products in 4-bit floats with a scale per 32 elements (the OCP microscaling format MXFP4: E2M1 elements, E8M0
scales), beside the products through a multiplier's table.

=====================  ==================================================================
``mx_quantize``        a matrix, along its last or its first axis
``mx_quantize_both``   along both with one read (a training step contracts either)
``mx_matmul``          product of two quantised matrices over their quantised axes
=====================  ==================================================================

Exported by :mod:`approxtrain_b200.ops`; ``layers.mxdense`` is the dense layer with gradients.
"""
from __future__ import annotations

import torch

from ._lib import ACT_NONE, ACT_RELU, lib
from .train_ops import _TYPES, _call, _tensor


_TILE = 17408   # bytes of a tile: 128 rows x 256 elements


def _bytes(rows: int, k: int) -> int:
    """``amsim_mx_bytes``."""
    return -(-rows // 128) * (-(-k // 256) or 1) * _TILE


def _tiles(data: torch.Tensor, shape, axis: int) -> "MXTensor":
    """An MXTensor of tiles that the library has written."""
    t = object.__new__(MXTensor)
    t.data, t.shape, t.axis = data, tuple(shape), axis
    return t


class MXTensor:
    """A matrix in 4-bit floats.  ``shape``: of the matrix as it was; ``axis``: the quantised one (1: blocks of 32 along the
    rows' elements, 0: along the columns').  ``data``: the library's tiles (uint8)."""

    def __init__(self, data: torch.Tensor, shape, axis: int):
        self.data, self.shape, self.axis = data, tuple(shape), axis
        if len(self.shape) != 2 or axis not in (0, 1):
            raise ValueError(f"a matrix and one of its axes (0, 1) expected, got {self.shape}, {axis}")
        if not data.is_cuda or data.dtype != torch.uint8 or not data.is_contiguous() or data.numel() != _bytes(self.rows, self.k):
            raise ValueError(f"data must be {_bytes(self.rows, self.k)} contiguous bytes on a CUDA device")

    @property
    def rows(self) -> int:
        """Rows of the stored matrix: the length of the axis that is not quantised."""
        return self.shape[1 - self.axis]

    @property
    def k(self) -> int:
        """Length of the quantised axis, which a product contracts."""
        return self.shape[self.axis]

    @property
    def device(self) -> torch.device:
        return self.data.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, in the matrix's shape."""
        if dtype not in _TYPES:
            raise TypeError(f"float32, bfloat16 or float16, got {dtype}")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        if out.numel():
            _call(self.device, lib.amsim_mx_dequantize, self.data.data_ptr(), self.rows, self.k, 1 - self.axis, out.data_ptr(), _TYPES[dtype])
        return out


def _matrix(x):
    x = _tensor(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be a matrix, got {list(x.shape)}")
    return x.contiguous()


def _quantize(x, along: bool, across: bool, sums=None):
    rows, cols = x.shape
    one = torch.empty(_bytes(rows, cols), dtype=torch.uint8, device=x.device) if along else None
    two = torch.empty(_bytes(cols, rows), dtype=torch.uint8, device=x.device) if across else None
    size = -(-rows // 128) * cols * 4 if sums is not None else 0   # (amsim_mx_quantize_workspace)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    if (along and rows) or (across and cols):
        _call(x.device, lib.amsim_mx_quantize, x.data_ptr(), rows, cols, _TYPES[x.dtype], one.data_ptr() if along else None,
              two.data_ptr() if across else None, sums.data_ptr() if sums is not None else None, ws.data_ptr() if size else None, size)
    return (_tiles(one, (rows, cols), 1) if along else None), (_tiles(two, (rows, cols), 0) if across else None)


def mx_quantize(x: torch.Tensor, axis: int = -1) -> MXTensor:
    """x (a matrix; float32, bfloat16 or float16) with blocks of 32 along `axis`.  A block's scale is the power of two that puts
    its largest element in [4, 8); elements are rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times it, ties to the even
    code, beyond 6 to 6.  An infinity or NaN makes its block NaN."""
    x = _matrix(x)
    if axis not in (-2, -1, 0, 1):
        raise ValueError(f"axis must be one of a matrix's two, got {axis}")
    along = axis in (-1, 1)
    return _quantize(x, along, not along)[0 if along else 1]


def mx_quantize_both(x: torch.Tensor, sums: torch.Tensor = None):
    """``(mx_quantize(x, 1), mx_quantize(x, 0))`` with one read of x.  ``sums`` (float32 [columns], optional): receives the sums of
    x's columns from the same read, FP32 in a fixed order (the bias gradient, where x is an output's gradient)."""
    x = _matrix(x)
    if sums is not None and (not isinstance(sums, torch.Tensor) or sums.dtype != torch.float32 or tuple(sums.shape) != (x.shape[1],) or sums.device != x.device
                             or not sums.is_contiguous()):
        raise ValueError(f"sums must be contiguous float32 of shape [{x.shape[1]}] on {x.device}")
    return _quantize(x, True, True, sums)


def mx_matmul(a: MXTensor, b: MXTensor, bias=None, activation=None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``act(a . b + bias)``, contracting the quantised axes: with a [m, k] (axis 1) or [k, m] (axis 0), b [k, n] (axis 0) or
    [n, k] (axis 1), the result is [m, n].  Products are exact, sums FP32, rounded once to `out_dtype` (float32, bfloat16 or
    float16).  ``bias``: float32 [n]; ``activation``: None or "relu"."""
    if not isinstance(a, MXTensor) or not isinstance(b, MXTensor):
        raise TypeError("a and b must be MXTensors (mx_quantize)")
    if a.device != b.device:
        raise ValueError(f"a is on {a.device}, b on {b.device}")
    if a.k != b.k:
        raise ValueError(f"quantised axes of lengths {a.k} and {b.k} cannot be contracted")
    if out_dtype not in _TYPES:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    if activation not in (None, "linear", "relu"):
        raise ValueError(f"only None / 'relu' can be fused into the product, got {activation!r}")
    m, n = a.rows, b.rows
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.dtype != torch.float32 or tuple(bias.shape) != (n,) or bias.device != a.device:
            raise ValueError(f"bias must be float32 of shape [{n}] on {a.device}")
        bias = bias.contiguous()
    out = torch.empty((m, n), dtype=out_dtype, device=a.device)
    if m and n:
        _call(a.device, lib.amsim_mx_matmul, a.data.data_ptr(), b.data.data_ptr(), m, n, a.k, bias.data_ptr() if bias is not None else None,
              ACT_RELU if activation == "relu" else ACT_NONE, out.data_ptr(), _TYPES[out_dtype])
    return out
