"""Weights in 8-bit integers with a scale for every output channel."""

from __future__ import annotations

import torch

STAGE = 128        # columns that the kernels take at a time: rows are held in whole stages
MOST_WIDTH = 1 << 17  # whole sums stay below 2^31


class Int8Weight:
    """A matrix ``[n, k]`` = ``values * scale[:, None]``: int8 rows, each padded with zeros to ``width`` columns (``k`` up to a
    multiple of 128), and float32 scales. ``HipOps.linear``, ``gated_linear`` and ``linear_for_residual`` take one
    in place of a weight of floats, and quantise the activations token by token (csrc/int8.h has the formulas)."""

    __slots__ = ("values", "scale", "shape", "width")

    def __init__(self, values: torch.Tensor, scale: torch.Tensor):
        if values.dim() != 2 or values.dtype != torch.int8 or not values.numel():
            raise ValueError(f"an 8-bit weight is a matrix of int8, not {tuple(values.shape)} of {values.dtype}")
        n, k = values.shape
        if scale.dtype != torch.float32 or tuple(scale.shape) != (n,) or scale.device != values.device:
            raise ValueError(f"an 8-bit weight of {n} rows has {n} float32 scales beside it, not {tuple(scale.shape)} of {scale.dtype} on {scale.device}")
        self.width = -(-k // STAGE) * STAGE
        if self.width > MOST_WIDTH:
            raise ValueError(f"rows of {k} in 8 bits: whole sums need {MOST_WIDTH} columns or fewer")
        self.shape = torch.Size((n, k))
        if self.width == k and values.is_contiguous() and values.data_ptr() % 16 == 0:
            self.values = values
        else:
            self.values = values.new_zeros((n, self.width))
            self.values[:, :k] = values
        self.scale = scale.contiguous()

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Int8Weight":
        """Every row by its largest magnitude over 127, rounded to the nearest integer. Rows must be finite."""
        if w.dim() != 2 or not w.is_floating_point():
            raise ValueError(f"a matrix of floats is quantised, not {tuple(w.shape)} of {w.dtype}")
        values = torch.empty(w.shape, dtype=torch.int8, device=w.device)
        scale = torch.empty(w.shape[0], dtype=torch.float32, device=w.device)
        for first in range(0, w.shape[0], 8192):  # a piece at a time: the float32 copy of a large matrix is four times its codes
            rows = w[first: first + 8192].float()
            most = rows.abs().amax(-1)
            if not bool(torch.isfinite(most).all()):
                raise ValueError("a weight that holds an infinity or a NaN has no 8-bit form")
            top = torch.full_like(most, 127)  # a tensor: a quotient with a number is a product with its reciprocal
            scale[first: first + 8192] = most / top
            by = torch.where(most < 2.0 ** -100, 0.0, top / most)
            values[first: first + 8192] = (rows * by[:, None]).round().to(torch.int8)
        return cls(values, scale)

    @property
    def dtype(self) -> torch.dtype:
        return torch.int8

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def num_bytes(self) -> int:
        return self.values.numel() + 4 * self.scale.numel()
