"""The 8-bit packed form of an activation (csrc/act8.cu).

Training a LoRA layer keeps the layer's input for the gradient of ``lora_A``.
Packed, it takes 1.03 bytes a value instead of 2: int8 codes with one fp32
scale per 128 values of a row,

    scale = max|x| / 127,   code = round(x * (127 / max|x|)).

One packed input serves every projection that reads it (q, k and v; gate and
up): ``packed_x=`` of ``LoRALinear``, ``MultiLoRALinear`` and
``adapters_add``, whose backward multiplies the codes themselves.
"""
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from rocm_qlora import _native as nat

#: values of a row that share one scale
BLOCK = 128


@dataclass
class PackedActivation:
    """``codes`` int8 [rows, ceil(K / 128) * 128] and ``scales`` fp32
    [rows, ceil(K / 128)] of an activation of ``shape`` [..., K]."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, columns] with contiguous columns, its rows apart or one row
    for all (stride 0): a view where its strides allow."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    columns = t.shape[1] <= 1 or t.stride(1) == 1
    rows = t.shape[0] <= 1 or t.stride(0) == 0 or t.stride(0) >= t.shape[1]
    return t if columns and rows else t.contiguous()


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """Pack x [..., K] (float32, bfloat16 or float16).  A block whose largest
    magnitude is below 2^-100 is stored as zeros; one that holds an infinity
    or NaN unpacks to NaN."""
    try:
        codes, scales = nat.loaded_ops().pack_activation(x)
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None
    return PackedActivation(codes, scales, tuple(x.shape), x.dtype)


def unpack_activation(packed: PackedActivation, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """code * scale, rounded to ``dtype`` (default: the dtype that was packed)."""
    try:
        return nat.loaded_ops().unpack_activation(packed.codes, packed.scales, packed.shape,
                                                  packed.dtype if dtype is None else dtype)
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None
