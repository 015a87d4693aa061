"""4-bit weights in the OCP microscaling format MXFP4: E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 with a sign) and one
power-of-two scale (E8M0) per 32 columns, 4.25 bits a value.

``mx4_quantize`` / ``mx4_dequantize`` make and read an ``Mx4``; ``mx4_linear`` multiplies by a frozen ``Mx4`` weight,
quantising its activation in the call; ``mx4_lora_linear`` adds the LoRA side path in the same product. The backward
passes are straight-through: dX = dY W with the quantised weight and an unquantised dY; gradients cannot be differentiated
again (an error says so). CUDA tensors only."""

from __future__ import annotations

from typing import NamedTuple

import torch


class Mx4(NamedTuple):
    """A quantised matrix [rows, cols]. codes uint8 [rows, ceil(cols/32)*16], two codes a byte, the even column in the
    low nibble; scales uint8 [ceil(rows/128), ceil(cols/128), 32, 4, 4], the scale 2^(code - 127) of row r and block
    j = col // 32 at [r // 128, j // 4, r % 32, r % 128 // 32, j % 4] (the tensor core's order). A block that held an
    infinity or a NaN has the scale 255 and reads back as NaN."""

    codes: torch.Tensor
    scales: torch.Tensor
    cols: int

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.cols))

    def to(self, device):
        return Mx4(self.codes.to(device), self.scales.to(device), self.cols)


def mx4_quantize(x: torch.Tensor) -> Mx4:
    """Quantise a matrix (fp32, bf16 or f16; rows may be strided). The scale of a block is
    2^(floor(log2(largest magnitude)) - 2); elements round to the nearest code, ties to the even one, and magnitudes
    above 6 scales become 6."""
    codes, scales = torch.ops.b2.mx4_quantize(x.detach() if x.requires_grad else x)
    return Mx4(codes, scales, x.shape[1])


def mx4_dequantize(w: Mx4, dtype=torch.bfloat16) -> torch.Tensor:
    """The values an Mx4 stands for (exact in bf16 and fp32), [rows, cols]."""
    return torch.ops.b2.mx4_dequantize(w.codes, w.scales, w.cols, dtype)


def mx4_linear(x: torch.Tensor, w: Mx4, bias: torch.Tensor | None = None) -> torch.Tensor:
    """y = Q(x) W^T + bias: x bf16 [..., K] is quantised to MXFP4 in the call, the element products are exact and
    summed in fp32. Differentiable in x (straight-through: dx = dy W) and bias; W is frozen."""
    return torch.ops.b2.mx4_linear(x, w.codes, w.scales, bias)


def mx4_lora_linear(x, w: Mx4, bias, a, b) -> torch.Tensor:
    """y = Q(x) W^T + bias + (x a^T) b^T: a frozen 4-bit linear with its LoRA side path, a [r, K] the down-projection
    and b [N, r] the up-projection already multiplied by alpha / r (r a multiple of 8, at most 64). The side path reads
    the unquantised x and is added inside the product; in the backward dX = dY W + (dY b) a is one product too.
    Differentiable in x, a, b (and bias). bf16."""
    return torch.ops.b2.mx4_lora_linear(x, w.codes, w.scales, bias, a, b)
