"""silu(gate) * up that keeps gate and up in 8 bits for its backward."""
from typing import Tuple, Union

import torch

from rocm_qlora import _native as nat
from rocm_qlora.activation8.packed import PackedActivation


def swiglu8(gate: torch.Tensor, up: torch.Tensor,
            pack_output: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, PackedActivation]]:
    """``silu(gate) * up`` for gate and up [..., K] of one dtype (float32,
    bfloat16 or float16; row strides allowed, such as the two halves of one
    projection's output).

    The product is of the values as given; for the backward only their packed
    forms are kept (2.06 bytes a column instead of 4).  ``pack_output=True``
    also returns the packed form of the product, written in the same pass,
    for the projection that reads it (``packed_x=``)."""
    try:
        h, codes, scales = nat.loaded_ops().swiglu8(gate, up, 3 if pack_output else 2)
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None
    return (h, PackedActivation(codes, scales, tuple(h.shape), h.dtype)) if pack_output else h
