"""Activations kept in 8 bits between forward and backward."""
from rocm_qlora.activation8.packed import BLOCK, PackedActivation, pack_activation, unpack_activation
from rocm_qlora.activation8.swiglu import swiglu8

__all__ = ["BLOCK", "PackedActivation", "pack_activation", "unpack_activation", "swiglu8"]
