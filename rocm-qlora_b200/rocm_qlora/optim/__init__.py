"""The optimizer of adapters: AdamW over many tensors at once."""
from rocm_qlora.optim.adamw import AdamW, grad_norm

__all__ = ["AdamW", "grad_norm"]
