"""FeatureDecoder: the network behind a grid's features.

Stands for the multi-layer perceptrons that the reference's users put there
(ash/mlp.py:43-285: SirenNet and a softplus network for signed distances).
"""
import math
from typing import Optional

import torch
import torch.nn as nn

from .layers import ACTIVATIONS, QuantizedRows, linear, rms_norm


class FeatureDecoder(nn.Module):
    """features (N, in_dim) -> values (N, out_dim).

    A first layer widens the features to `width`; each of `blocks` residual blocks
    adds linear(activation(linear(rms_norm(h)))) to h, the addition being part of
    the next norm; a last norm and layer give the values.  Every step is one of
    the package's kernels, with gradients of first and second order, so that the
    values may be differentiated by the positions under a loss (`SparseDenseGrid`'s
    features carry such gradients).

    `quantize_()` lays the blocks' weights out in 8 bits for serving: norms then
    round their rows to 8 bits, and the products of the blocks are made of 8-bit
    rows.  The first and the last layer keep their type.
    """

    def __init__(
        self,
        in_dim: int,
        out_dim: int,
        width: int = 64,
        blocks: int = 2,
        activation: str = "softplus",
        scale: float = 1.0,
        device: Optional[torch.device] = None,
        dtype: torch.dtype = torch.float32,
    ):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
        self.in_dim, self.out_dim, self.width = int(in_dim), int(out_dim), int(width)
        self.activation, self.scale = activation, float(scale)
        like = {"device": device, "dtype": dtype}

        def layer(n_in, n_out):
            return nn.ParameterDict({
                "weight": nn.Parameter(torch.empty(n_out, n_in, **like)),
                "bias": nn.Parameter(torch.empty(n_out, **like)),
            })

        self.first = layer(self.in_dim, self.width)
        self.up = nn.ModuleList(layer(self.width, self.width) for _ in range(blocks))
        self.down = nn.ModuleList(layer(self.width, self.width) for _ in range(blocks))
        self.last = layer(self.width, self.out_dim)
        self.norms = nn.ParameterList(torch.empty(self.width, **like) for _ in range(blocks + 1))
        self._served = None
        self.reset_parameters()

    def reset_parameters(self) -> None:
        """Uniform weights at the scale that keeps features of unit size so, or
        the argument of a sine; unit norms."""
        with torch.no_grad():
            for one in (self.first, *self.up, *self.down, self.last):
                bound = math.sqrt(3.0 / one["weight"].shape[1])
                if self.activation == "sine":
                    bound *= math.sqrt(2.0) / self.scale
                one["weight"].uniform_(-bound, bound)
                one["bias"].uniform_(-bound, bound).mul_(0.1)
            for norm in self.norms:
                norm.fill_(1.0)

    def extra_repr(self) -> str:
        return (f"in_dim={self.in_dim}, out_dim={self.out_dim}, width={self.width}, "
                f"blocks={len(self.up)}, activation={self.activation}")

    def quantize_(self) -> "FeatureDecoder":
        """From now on the blocks' products are of 8-bit rows, with the weights as
        they are at this moment; `dequantize_` takes it back.  Call forward under
        torch.no_grad() then."""
        self._served = [tuple(QuantizedRows.of(one["weight"]) for one in pair)
                        for pair in zip(self.up, self.down)]
        return self

    def dequantize_(self) -> "FeatureDecoder":
        self._served = None
        return self

    def _apply(self, fn, recurse=True):
        self._served = None   # of other weights, or elsewhere
        return super()._apply(fn, recurse)

    def _layer(self, one, rows, activation="none", residual=None):
        return linear(rows, one["weight"], one["bias"], activation, self.scale, residual)

    def forward(self, features: torch.Tensor) -> torch.Tensor:
        h = self._layer(self.first, features, self.activation)
        added = None
        quantize = self._served is not None
        for i, (up, down) in enumerate(zip(self.up, self.down)):
            normed = rms_norm(h, self.norms[i], residual=added, quantize=quantize)
            if added is not None:
                normed, h = normed
            if quantize:
                weight, back = self._served[i]
                inner = linear(normed, weight, up["bias"], self.activation, self.scale)
                added = linear(QuantizedRows.of(inner), back, down["bias"], "none", self.scale)
            else:
                inner = self._layer(up, normed, self.activation)
                added = self._layer(down, inner)
        normed = rms_norm(h, self.norms[-1], residual=added)
        return self._layer(self.last, normed if added is None else normed[0])
