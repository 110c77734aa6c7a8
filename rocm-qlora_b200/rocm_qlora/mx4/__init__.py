"""Microscaled 4-bit values, and products on the block-scaled tensor cores."""
from rocm_qlora.mx4.linear import Mx4Linear, mx4_linear, mx4_matmul
from rocm_qlora.mx4.packed import BLOCK, PackedMx4, pack_mx4, unpack_mx4

__all__ = ["BLOCK", "PackedMx4", "pack_mx4", "unpack_mx4", "mx4_matmul", "mx4_linear", "Mx4Linear"]
