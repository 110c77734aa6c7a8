"""Products of microscaled 4-bit operands (csrc/mx4_gemm.cu), and a frozen
projection that is one: the base of a QLoRA layer whose weight and input both
enter the tensor cores in 4 bits, at four times the rate of 16-bit operands.
"""
from typing import Optional

import torch
import torch.nn as nn

from rocm_qlora import _native as nat
from rocm_qlora.mx4.packed import PackedMx4, pack_mx4, unpack_mx4


def mx4_matmul(a: PackedMx4, b: PackedMx4, bias: Optional[torch.Tensor] = None,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a . b^T (+ bias)`` of packed a [..., K] and b [N, K]: [..., N] in
    ``dtype`` (bfloat16 or float16; the bias too), summed in 32 bits and
    rounded once.  No gradients."""
    if len(b.shape) != 2 or not a.shape or a.shape[-1] != b.shape[-1]:
        raise ValueError(f"a {a.shape} and b {b.shape} do not fit")
    try:
        y = nat.loaded_ops().mx4_matmul(a.codes, a.scales, b.codes, b.scales, b.shape[-1], bias, dtype)
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None
    return y if len(a.shape) == 2 else y.view(*a.shape[:-1], b.shape[0])


def mx4_linear(x: torch.Tensor, weight: PackedMx4, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``pack_mx4(x) . weight^T (+ bias)`` for x [..., K] (bfloat16 or float16)
    and a packed frozen weight [N, K].  Differentiable in x, whose rounding is
    passed through: dx = dy . weight, with dy in 16 bits (in float16 weights
    below 2^-24 of the largest scale count as 0).  Nothing of x is kept."""
    if len(weight.shape) != 2:
        raise ValueError(f"the weight must be [N, K], got {weight.shape}")
    try:
        return nat.loaded_ops().mx4_linear(x, weight.codes, weight.scales, weight.shape[-1], bias)
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None


class Mx4Linear(nn.Module):
    """A frozen ``nn.Linear`` in microscaled 4 bits."""

    def __init__(self, in_features: int, out_features: int, bias: bool = False,
                 dtype: torch.dtype = torch.bfloat16, device: Optional[torch.device] = None):
        super().__init__()
        self.in_features, self.out_features, self.dtype = in_features, out_features, dtype
        pitch, tiles = -(-in_features // 128) * 128, -(-out_features // 128)
        byte = dict(dtype=torch.uint8, device=device)
        self.register_buffer("codes", torch.zeros(out_features, pitch // 2, **byte))
        self.register_buffer("scales", torch.zeros(tiles, pitch // 128, 512, **byte))
        self.register_buffer("bias", torch.zeros(out_features, dtype=dtype, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "Mx4Linear":
        """Pack an ``nn.Linear``; its weight is not kept."""
        w = linear.weight.detach()
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, w.dtype, "meta")
        packed = pack_mx4(nat.to_cuda(w))
        m.codes, m.scales = packed.codes, packed.scales
        if linear.bias is not None:
            m.bias = linear.bias.detach().to(packed.codes.device)
        return m

    @property
    def weight(self) -> PackedMx4:
        return PackedMx4(self.codes, self.scales, (self.out_features, self.in_features), self.dtype)

    def dequantized(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        return unpack_mx4(self.weight, dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        return mx4_linear(x, self.weight, bias)

    def extra_repr(self) -> str:
        return f"in={self.in_features}, out={self.out_features}, bias={self.bias is not None}"
