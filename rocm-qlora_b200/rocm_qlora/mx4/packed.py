"""The microscaled 4-bit form of rows (csrc/mx4.cu).

32 values of a row share the scale 2^e, one byte, and take 4 bits each:

    e = max(floor(log2 max|x|) - 2, -127),
    code = the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} to x / 2^e, ties to
           the even code, 6 beyond it.

That is 0.53 bytes a value.  The scales lie in the order that the tensor
cores read them, so a packed tensor is an operand as it is.
"""
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from rocm_qlora import _native as nat

#: values of a row that share one scale
BLOCK = 32


@dataclass
class PackedMx4:
    """``codes`` uint8 [rows, Kp / 2] (two a byte, the even column low) and
    ``scales`` uint8 [ceil(rows / 128), Kp / 128, 512] of a tensor of
    ``shape`` [..., K], with Kp = K rounded up to 128."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def scale_rows(self) -> torch.Tensor:
        """The scale bytes (e + 127) as [rows, Kp / 32], in the columns' order."""
        tiles, pieces = self.scales.shape[:2]
        s = self.scales.view(tiles, pieces, 32, 4, 4).permute(0, 3, 2, 1, 4)
        return s.reshape(tiles * 128, pieces * 4)[:self.codes.shape[0]]


def pack_mx4(x: torch.Tensor) -> PackedMx4:
    """Pack x [..., K] (float32, bfloat16 or float16).  A block that holds an
    infinity or NaN unpacks to NaN."""
    try:
        codes, scales = nat.loaded_ops().pack_mx4(x)
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None
    return PackedMx4(codes, scales, tuple(x.shape), x.dtype)


def unpack_mx4(packed: PackedMx4, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """code * 2^e, rounded to ``dtype`` (default: the dtype that was packed)."""
    try:
        return nat.loaded_ops().unpack_mx4(packed.codes, packed.scales, packed.shape,
                                           packed.dtype if dtype is None else dtype)
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None
