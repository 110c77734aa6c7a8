"""LoRA adapter layer for rocm-qlora."""
from rocm_qlora.lora.lora_layer import LoRALinear
from rocm_qlora.lora.adapter_bank import AdapterBank, AdapterPlan, MultiLoRALinear, adapters_add

__all__ = ["LoRALinear", "AdapterBank", "AdapterPlan", "MultiLoRALinear", "adapters_add"]
