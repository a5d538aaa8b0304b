"""Layers that read the features of a grid or an embedding: the dense layer with
bias, activation and residual in one kernel, and the root-mean-square norm with
the residual's addition, both with gradients of first and second order (an
eikonal loss differentiates a decoder twice), and 8-bit rows for serving.

The reference leaves these to torch (ash/mlp.py:43-285 and the networks of its
tests, unittests/test_sparsedense_grid.py:218-220).
"""
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import core
from .common import stands_alone

ACTIVATIONS = ("none", "relu", "silu", "gelu", "softplus", "sine")


class QuantizedRows(NamedTuple):
    """Rows in 8 bits: row i stands for `data[i] * scales[i]`.

    data    float8_e4m3fn (..., width)
    scales  float32 (...)
    """

    data: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def of(cls, rows: torch.Tensor) -> "QuantizedRows":
        """Rows of 1 to 16384 values rounded to 8 bits, each by its largest
        magnitude (which becomes 448, the type's largest number).  A row of zeros
        has the scale 1; one that holds an infinity or NaN has the scale NaN and
        is NaN as a whole.  No gradients: a layer's weights are laid out so once,
        for serving."""
        _must_stand_alone("QuantizedRows", rows)
        return cls(*core.backend.host.quantize_rows(rows.detach()))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values that the rows stand for, as a tensor of `dtype`."""
        return (self.data.float() * self.scales.unsqueeze(-1)).to(dtype)


def _must_stand_alone(what: str, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and not stands_alone(t):
            raise RuntimeError(
                f"{what} takes plain tensors (no subclasses, function transforms, forward-mode "
                "tangents or traces)")


def linear(
    input: Union[torch.Tensor, QuantizedRows],
    weight: Union[torch.Tensor, QuantizedRows],
    bias: Optional[torch.Tensor] = None,
    activation: str = "none",
    scale: float = 1.0,
    residual: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """activation(input @ weight.T + bias) + residual, in one kernel.

    input     (..., in), float32, bfloat16 or float16
    weight    (out, in), bias (out,), residual of a shape that broadcasts to the
              output's; all of the input's type
    activation  "none", "relu", "silu", "gelu" (by the error function),
              "softplus" (log(1 + exp(scale z)) / scale) or "sine" (sin(scale z));
              `scale` is read by the last two only, and positive

    Sums are float32 throughout; results are rounded once.  float32 operands are
    multiplied as the sum of three bfloat16 numbers each, which keeps their 24
    bits; one of infinite (or, above 3.38e38, nearly infinite) magnitude gives
    NaN, where a product in float32 might be infinite.

    Gradients of first and second order exist for every operand (of the gradient
    of a weight too, not of third order).  For them the forward keeps the slope of
    the activation at every output, in float32 (float16 for bfloat16 operands), or,
    for float32 relu and softplus without a residual, the output itself, which must
    not be changed in place before the backward pass then.  They are the same
    numbers on every run.  While a graph is captured, a broadcast residual that
    needs a gradient is refused, and so are leaves that an eager graph still holds.

    With 8-bit rows (`QuantizedRows`, both or neither) every sum of products is
    multiplied by the scales of its two rows; bias and residual have the type of
    the output, which is `out_dtype`, the type of the bias or that of the
    residual, whichever is given first, or bfloat16.  No gradients."""
    if isinstance(input, QuantizedRows) or isinstance(weight, QuantizedRows):
        if not (isinstance(input, QuantizedRows) and isinstance(weight, QuantizedRows)):
            raise RuntimeError("linear: 8-bit rows need an 8-bit weight, and it them")
        _must_stand_alone("linear", *input, *weight, bias, residual)
        return core.backend.host.linear_quantized(*input, *weight, bias, activation, scale, residual, out_dtype)
    if out_dtype is not None and out_dtype != input.dtype:
        raise RuntimeError(f"linear: the output has the type of the input, {input.dtype}")
    _must_stand_alone("linear", input, weight, bias, residual)
    return core.backend.host.linear(input, weight, bias, activation, scale, residual)


def rms_norm(
    input: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    quantize: bool = False,
) -> Union[torch.Tensor, QuantizedRows, Tuple[Union[torch.Tensor, QuantizedRows], torch.Tensor]]:
    """s / sqrt(mean(s * s) + eps) * weight over the last axis, of s = input +
    residual, in one pass over the rows.

    input     (..., width), float32, bfloat16 or float16, width up to 16384
    weight    (width,) or None: ones
    residual  of a shape that broadcasts to the input's, or None

    Returns the normed rows, or with a residual (normed rows, s).  With `quantize`
    the normed rows are `QuantizedRows`, rounded to 8 bits from float32 by the
    same kernel (no gradients then).  Gradients of first and second order exist
    for every operand.  Squares are float32: a row of values beyond 1e19 gives
    zeros."""
    _must_stand_alone("rms_norm", input, weight, residual)
    normed, total, scales = core.backend.host.rms_norm(input, weight, residual, eps, quantize)
    if quantize:
        normed = QuantizedRows(normed, scales)
    return normed if residual is None else (normed, total)
