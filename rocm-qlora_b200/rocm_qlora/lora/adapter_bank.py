"""Adapters of many requests beside one shared projection.

An ``AdapterBank`` holds the LoRA adapters of one projection, an
``AdapterPlan`` says which adapter each row of a batch uses (made once a
batch, shared by all layers), and ``adapters_add`` computes

    y[m] = base[m] + scaling[a] * (x[m] @ A[a]) @ B[a].T,    a = ids[m]

for all rows at once, in one launch, with its gradients (csrc/adapters.cu).
``MultiLoRALinear`` is the layer: a QuantLinear and its bank.
"""
from typing import Optional, Sequence

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from rocm_qlora import _native as nat
from rocm_qlora.activation8.packed import BLOCK, PackedActivation, rows_of
from rocm_qlora.quantization import layer_ops

MAX_RANK = 128
MAX_ADAPTERS = 4096


class AdapterPlan:
    """Which adapter each row uses.  ``ids`` [rows] (int64 or int32): 0 to
    ``count - 1``, or -1 for none.  Ids on the CPU are checked; ids on the GPU
    are not read back, and a row whose id names no adapter gets NaN outputs.

    The plan lives on the GPU (``device``: for ids on the CPU) and belongs to
    the stream it was made on, like any tensor."""

    def __init__(self, ids: torch.Tensor, count: int, device: Optional[torch.device] = None):
        if ids.dim() != 1 or ids.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"ids must be a 1-D int64 or int32 tensor, got {tuple(ids.shape)} {ids.dtype}")
        if not 1 <= count <= MAX_ADAPTERS:
            raise ValueError(f"count must be between 1 and {MAX_ADAPTERS}, got {count}")
        if not ids.is_cuda:
            if ids.numel() and (int(ids.min()) < -1 or int(ids.max()) >= count):
                raise ValueError(f"ids must lie between -1 and {count - 1}")
            ids = nat.to_cuda(ids) if device is None else ids.to(device)
        self.rows, self.count = ids.shape[0], count
        self.tile = tile_rows(self.rows, count)
        self.data = nat.require_ops(ids).adapter_plan(ids.contiguous(), count, self.tile)


def tile_rows(rows: int, count: int) -> int:
    """Rows computed together: about as many as an adapter has, and 128 only
    where there are enough of them to fill the GPU."""
    for tile in (16, 32, 64):
        if rows <= tile * count:
            return tile
    return 128 if rows > 4096 else 64


def _plan_args(plan: Optional[AdapterPlan], rows: int, count: int):
    if plan is None:
        if count != 1:
            raise ValueError("a bank of several adapters needs a plan")
        return None, 0
    if plan.rows != rows or plan.count != count:
        raise ValueError(f"the plan is for {plan.rows} rows and {plan.count} adapters, not {rows} and {count}")
    return plan.data, plan.tile


def _packed_args(packed_x: Optional[PackedActivation], x: torch.Tensor):
    if packed_x is None:
        return None, None
    codes, scales = packed_x.codes, packed_x.scales
    if packed_x.shape[-1] != x.shape[-1] or codes.shape[0] != x.numel() // max(1, x.shape[-1]):
        raise ValueError(f"packed_x is of {packed_x.shape}, x of {tuple(x.shape)}")
    if codes.dtype != torch.int8 or scales.dtype != torch.float32 or codes.numel() != scales.numel() * BLOCK:
        raise ValueError(f"packed_x holds int8 codes and a float32 scale for each {BLOCK} of them, got {codes.dtype} "
                         f"{tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}")
    return codes, scales


def _check_bank(x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, scaling: torch.Tensor) -> None:
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"adapters take bfloat16 or float16 activations, got {x.dtype}")
    if A.dim() != 3 or B.dim() != 3 or A.shape[0] != B.shape[0] or A.shape[2] != B.shape[2]:
        raise ValueError(f"A must be [count, in, rank] and B [count, out, rank]; got {tuple(A.shape)}, {tuple(B.shape)}")
    if A.dtype != x.dtype or B.dtype != x.dtype:
        raise TypeError(f"adapters are {A.dtype} and {B.dtype}, activations {x.dtype}")
    if A.shape[2] % 8 or not 8 <= A.shape[2] <= MAX_RANK:
        raise ValueError(f"rank must be a multiple of 8 up to {MAX_RANK}, got {A.shape[2]} (AdapterBank pads)")
    if not 1 <= A.shape[0] <= MAX_ADAPTERS:
        raise ValueError(f"a bank holds 1 to {MAX_ADAPTERS} adapters, got {A.shape[0]}")
    if scaling.shape != (A.shape[0],) or scaling.dtype != torch.float32:
        raise ValueError(f"scaling must be float32 [{A.shape[0]}], got {scaling.dtype} {tuple(scaling.shape)}")


def adapters_add(base: torch.Tensor, x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, scaling: torch.Tensor,
                 plan: Optional[AdapterPlan] = None, packed_x: Optional[PackedActivation] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``base + scaling * (x @ A) @ B.T`` per row with the row's own adapter.

    base [..., N] and x [..., K] (bfloat16 or float16, rows may be strided or
    expanded), A [count, K, rank], B [count, N, rank] (contiguous), scaling
    [count] float32; ``plan`` may be None for a bank of one.  All on one
    device.  Products are accumulated in 32 bits and the sum is rounded once.
    With ``packed_x`` (the packed form of x) the backward of A reads it and x
    is not kept.  Differentiable once, in reverse mode.  ``out`` (no gradients
    then) takes the result and may be ``base`` itself."""
    args = (plan.data, plan.rows, plan.count, plan.tile) if plan is not None else (None, 0, 0, 0)
    if packed_x is not None:
        _packed_args(packed_x, x)
    if out is not None:
        return _add_out(base, x, A, B, scaling, plan, out)
    try:
        return nat.loaded_ops().adapters_add(base, x, A, B, scaling, *args,
                                             *((None, None) if packed_x is None else (packed_x.codes, packed_x.scales)))
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None


def _add_out(base, x, A, B, scaling, plan, out) -> torch.Tensor:
    _check_bank(x, A, B, scaling)
    if (torch.is_grad_enabled() and any(t.requires_grad for t in (base, x, A, B, out))
            or any(unpack_dual(t).tangent is not None for t in (base, x, A, B, scaling, out))):
        raise RuntimeError("adapters_add(out=...) does not support automatic differentiation")
    if out.shape != base.shape or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("out must be contiguous, of base's shape and dtype")
    if x.shape[:-1] != base.shape[:-1] or x.shape[-1] != A.shape[1] or base.shape[-1] != B.shape[1]:
        raise ValueError(f"base {tuple(base.shape)} and x {tuple(x.shape)} do not fit A {tuple(A.shape)} and "
                         f"B {tuple(B.shape)}")
    x2, base2 = rows_of(x), rows_of(base)
    data, tile = _plan_args(plan, x2.shape[0], A.shape[0])
    nat.require_ops(base, x, A, B, scaling, out, data).adapters_apply_(
        out.view(base2.shape), x2, A.contiguous(), B.contiguous(), scaling.contiguous(), base2, data, tile)
    return out


class _BankLinear(torch.autograd.Function):
    """QuantLinear and its bank: the adapters' sum goes in place into the
    shared projection's output, and in the backward into its input gradient."""

    @staticmethod
    def forward(ctx, x, A, B, w, bias, scaling, plan, codes, scales):
        data, tile = plan
        ops = nat.require_ops(x, A, B, scaling, data, codes, scales)
        rows = x.reshape(-1, w.K).contiguous()
        y = layer_ops.forward(w, rows, bias.to(x.dtype).contiguous() if bias is not None else None, None, None, 1.0)
        mid = ops.adapters_apply_(y, rows, A, B, scaling, y, data, tile)
        z = (None, None) if not ctx.needs_input_grad[1] else (rows, None) if codes is None else (codes, scales)
        ctx.save_for_backward(*z, A, B, scaling, mid, data)
        ctx.w, ctx.tile, ctx.shape = w, tile, x.shape
        return y.view(*x.shape[:-1], w.N)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        z, scales, A, B, scaling, mid, data = ctx.saved_tensors
        w, tile = ctx.w, ctx.tile
        need_x, need_A, need_B = ctx.needs_input_grad[:3]
        rows = dy.reshape(-1, w.N).contiguous()
        ops = nat.require_ops(rows, A)
        dx = dA = dB = None
        if need_x:
            dx = layer_ops.dx(w, rows, None, None, 1.0)
            gmid = ops.adapters_apply_(dx, rows, B, A, scaling, dx, data, tile)
            dx = dx.view(ctx.shape)
        elif need_A:
            gmid = ops.adapters_mid(rows, B, A, scaling, data, tile)
        if need_A:
            dA = ops.adapters_grad(z, scales, gmid, A.shape[1], A.shape[0], A.dtype, data, tile)
        if need_B:
            dB = ops.adapters_grad(rows, None, mid, B.shape[1], B.shape[0], B.dtype, data, tile)
        return dx, dA, dB, None, None, None, None, None, None


def bank_linear(x: torch.Tensor, w: layer_ops.WeightView, bias: Optional[torch.Tensor], A: torch.Tensor,
                B: torch.Tensor, scaling: torch.Tensor, plan: Optional[AdapterPlan] = None,
                packed_x: Optional[PackedActivation] = None) -> torch.Tensor:
    """``adapters_add`` onto ``x @ deq(w).T + bias``, which is rounded to x's dtype first."""
    _check_bank(x, A, B, scaling)
    if x.shape[-1] != w.K or A.shape[1] != w.K or B.shape[1] != w.N:
        raise ValueError(f"x {tuple(x.shape)}, A {tuple(A.shape)} and B {tuple(B.shape)} do not fit a "
                         f"{w.N} x {w.K} weight")
    args = _plan_args(plan, x.numel() // w.K, A.shape[0])
    return _BankLinear.apply(x, A.contiguous(), B.contiguous(), w, bias, scaling.contiguous(), args,
                             *_packed_args(packed_x, x))


class AdapterBank(nn.Module):
    """``count`` adapters over a projection of ``in_features`` to
    ``out_features``: parameters ``lora_A`` [count, in, rank] and ``lora_B``
    [count, out, rank], the rank padded with zeros to a multiple of 8 (the
    padding gets no gradient and stays zero).  A new bank adds nothing."""

    def __init__(self, in_features: int, out_features: int, count: int, rank: int,
                 dtype: torch.dtype = torch.bfloat16, device: Optional[torch.device] = None):
        super().__init__()
        if not 1 <= rank <= MAX_RANK:
            raise ValueError(f"rank must be between 1 and {MAX_RANK}, got {rank}")
        if not 1 <= count <= MAX_ADAPTERS:
            raise ValueError(f"count must be between 1 and {MAX_ADAPTERS}, got {count}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"adapters are bfloat16 or float16, got {dtype}")
        self.in_features, self.out_features, self.count, self.rank = in_features, out_features, count, rank
        stored = -(-rank // 8) * 8
        self.lora_A = nn.Parameter(torch.zeros(count, in_features, stored, dtype=dtype, device=device))
        self.lora_B = nn.Parameter(torch.zeros(count, out_features, stored, dtype=dtype, device=device))
        self.register_buffer("scaling", torch.ones(count, dtype=torch.float32, device=device))

    @torch.no_grad()
    def set_adapter(self, index: int, lora_A: torch.Tensor, lora_B: torch.Tensor, scaling: float) -> None:
        """Store an adapter as LoRALinear keeps it: lora_A [r, in], lora_B [out, r], r up to the bank's rank."""
        r = lora_A.shape[0]
        if not 0 <= index < self.count:
            raise IndexError(f"the bank holds {self.count} adapters, not number {index}")
        if (lora_A.dim() != 2 or lora_B.dim() != 2 or not 1 <= r <= self.rank or lora_A.shape[1] != self.in_features
                or tuple(lora_B.shape) != (self.out_features, r)):
            raise ValueError(f"lora_A {tuple(lora_A.shape)} and lora_B {tuple(lora_B.shape)} do not fit a bank of "
                             f"{self.in_features} to {self.out_features}, rank {self.rank}")
        self.lora_A[index].zero_()
        self.lora_B[index].zero_()
        self.lora_A[index, :, :r] = lora_A.t().to(self.lora_A)
        self.lora_B[index, :, :r] = lora_B.to(self.lora_B)
        self.scaling[index] = float(scaling)

    @classmethod
    def from_lora_layers(cls, layers: Sequence[nn.Module], dtype: torch.dtype = torch.bfloat16) -> "AdapterBank":
        """The adapters of several LoRALinear layers over the same projection."""
        if not layers:
            raise ValueError("no layers")
        base = layers[0].base_layer
        bank = cls(base.in_features, base.out_features, len(layers), max(m.r for m in layers), dtype,
                   layers[0].lora_A.device)
        for i, m in enumerate(layers):
            bank.set_adapter(i, m.lora_A, m.lora_B, m.scaling)
        return bank

    def forward(self, base: torch.Tensor, x: torch.Tensor, plan: Optional[AdapterPlan] = None,
                packed_x: Optional[PackedActivation] = None) -> torch.Tensor:
        return adapters_add(base, x, self.lora_A, self.lora_B, self.scaling, plan, packed_x)

    def extra_repr(self) -> str:
        return f"in={self.in_features}, out={self.out_features}, count={self.count}, rank={self.rank}"


class MultiLoRALinear(nn.Module):
    """A frozen QuantLinear shared by the rows of all requests, and its bank."""

    def __init__(self, quant_linear: nn.Module, bank: AdapterBank):
        super().__init__()
        if (quant_linear.in_features, quant_linear.out_features) != (bank.in_features, bank.out_features):
            raise ValueError(f"the layer is {quant_linear.in_features} to {quant_linear.out_features}, the bank "
                             f"{bank.in_features} to {bank.out_features}")
        self.base_layer, self.bank = quant_linear, bank
        for p in quant_linear.parameters():
            p.requires_grad_(False)

    def forward(self, x: torch.Tensor, plan: Optional[AdapterPlan] = None,
                packed_x: Optional[PackedActivation] = None) -> torch.Tensor:
        b = self.base_layer
        if b.merged_mode and b.merged_fp16_weight is not None:
            return self.bank(b(x), x, plan, packed_x)
        return bank_linear(x, b.weight_view(), b.bias, self.bank.lora_A, self.bank.lora_B, self.bank.scaling, plan,
                           packed_x)


def one_adapter(lora_A: torch.Tensor, lora_B: torch.Tensor, dtype: torch.dtype):
    """A LoRALinear's parameters [r, in] and [out, r] as a bank of one in
    ``dtype`` (differentiable; the rank padded to a multiple of 8)."""
    A, B = lora_A.to(dtype).t(), lora_B.to(dtype)
    pad = -A.shape[1] % 8
    if pad:
        A, B = F.pad(A, (0, pad)), F.pad(B, (0, pad))
    return A.unsqueeze(0).contiguous(), B.unsqueeze(0).contiguous()
