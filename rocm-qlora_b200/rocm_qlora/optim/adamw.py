"""AdamW over many tensors in one launch, its moments in 32 or in 8 bits
(csrc/adamw.cu), and the norm of many gradients.
"""
import copy
from typing import Any, Dict, Iterable, List, Optional, Tuple, Union

import torch

from torch.optim.optimizer import _global_optimizer_post_hooks, _global_optimizer_pre_hooks

from rocm_qlora import _native as nat

#: values of a tensor that share the scales of its 8-bit moments
BLOCK = 256


def grad_norm(tensors: Iterable[torch.Tensor]) -> torch.Tensor:
    """sqrt(sum of all squares) of the tensors' values (float32, bfloat16 or
    float16, on one device), summed in 64 bits: one float32 on the device."""
    try:
        return nat.loaded_ops().grad_norm([t.detach() for t in tensors])
    except NotImplementedError as e:
        raise nat.NativeUnavailable(str(e)) from None


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay, as ``torch.optim.AdamW`` computes it:

        m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
        p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    in 32 bits (root and quotient by the approximate instructions: a step is off
    by at most 14 x 2^-24 of what it adds up) and rounded once to the type.

    Parameters are contiguous float32, bfloat16 or float16 tensors on one
    CUDA device; a step is one launch, or two with clipping, for up to 1024 of a
    dtype, without host synchronisation, and can be captured into a CUDA graph (steps
    are counted on the device; make ``lr`` a float32 tensor there to change it
    between replays).

    ``state_bits=8`` keeps the moments in blocks of 256 values: m as e4m3
    codes, sqrt(v) as floats of 4 exponent and 4 mantissa bits, each times a
    float32 scale of the block; 2.03 bytes a value instead of 8.
    ``remainder=True`` (bfloat16 parameters) keeps the lower half of a 32-bit
    value beside each parameter, so that small updates are not rounded away.
    ``max_grad_norm`` scales all gradients (the ``.grad`` stay as they are) by
    min(1, max_grad_norm / (norm + 1e-6)); ``grad_norm`` is the last step's
    norm, on the device."""

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32, remainder: bool = False,
                 max_grad_norm: Optional[float] = None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError(f"max_grad_norm must be positive, got {max_grad_norm}")
        self.state_bits, self.remainder, self.max_grad_norm = state_bits, bool(remainder), max_grad_norm
        self.grad_norm: Optional[torch.Tensor] = None
        self._arenas, self._native = [], None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    # ------------------------------------------------------------- groups

    @staticmethod
    def _check_numbers(group: Dict[str, Any]) -> None:
        lr, (b1, b2) = group["lr"], group["betas"]
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be at least 0 and below 1, got {group['betas']}")
        if not group["eps"] >= 0.0 or not group["weight_decay"] >= 0.0:
            raise ValueError(f"eps and weight_decay must not be negative, got {group['eps']}, {group['weight_decay']}")

    def add_param_group(self, param_group: Dict[str, Any]) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_numbers(group)
            self._check_params(group["params"])
            self._arenas.append(self._make_state(group["params"]))
        except Exception:
            self.param_groups.pop()
            raise
        self._native = None

    @property
    def _device(self) -> torch.device:
        """The first parameter's; a group may have none."""
        return next((p.device for g in self.param_groups for p in g["params"]), torch.device("cpu"))

    def _check_params(self, params) -> None:
        device = self._device
        if len(params) > 65536:
            raise ValueError(f"a parameter group holds at most 65536 tensors, got {len(params)}")
        # one launch updates them side by side
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size())
                       for p in params if p.numel() and p.is_contiguous() and not p.is_meta)
        if any(end > start for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("a parameter group holds a parameter twice, or two that share memory")
        for p in params:
            if not p.is_cuda:
                raise nat.NativeUnavailable(
                    "rocm_qlora (B200 build) computes on the GPU only: move the parameters to a CUDA device")
            if p.device != device:
                raise ValueError(f"parameters are on different devices: {device} and {p.device}")
            nat.dtype_code(p.dtype)
            if not p.is_contiguous():
                raise ValueError(f"parameters must be contiguous, got one of strides {p.stride()}")
            if self.remainder and p.dtype != torch.bfloat16:
                raise TypeError(f"remainder keeps what bfloat16 parameters leave, got a parameter of {p.dtype}")

    def _make_state(self, params) -> Dict[str, Any]:
        device = self._device
        blocks = [-(-p.numel() // BLOCK) for p in params]
        total = sum(blocks)
        of = torch.uint8 if self.state_bits == 8 else torch.float32
        a = dict(m=torch.zeros(total * BLOCK, dtype=of, device=device),
                 v=torch.zeros(total * BLOCK, dtype=of, device=device),
                 scales=torch.zeros(total, 2, device=device) if self.state_bits == 8 else None,
                 low=torch.zeros(total * BLOCK, dtype=torch.int16, device=device) if self.remainder else None,
                 steps=torch.zeros(len(params), dtype=torch.int32, device=device),
                 ticket=torch.zeros(1, dtype=torch.int32, device=device))
        at = 0
        for i, (p, n) in enumerate(zip(params, blocks)):
            part = slice(at * BLOCK, at * BLOCK + p.numel())
            s = self.state[p]
            s["step"] = a["steps"][i]
            s["exp_avg"], s["exp_avg_sq"] = a["m"][part].view(p.shape), a["v"][part].view(p.shape)
            if a["scales"] is not None:
                s["scales"] = a["scales"][at:at + n]
            if a["low"] is not None:
                s["remainder"] = a["low"][part].view(p.shape)
            at += n
        return a

    def _held(self):
        nat.loaded_ops()
        held = torch.classes.rocm_qlora.AdamW(self.state_bits)
        for group, a in zip(self.param_groups, self._arenas):
            if group["params"]:
                held.add_group(group["params"], a["m"], a["v"], a["scales"], a["low"], a["steps"], a["ticket"])
        if self.grad_norm is not None and self.grad_norm.device != self._device:
            self.grad_norm = None  # made before the first parameter came
        self._native = held
        return held

    # --------------------------------------------------------------- step

    def step(self, closure=None):
        """One step of every parameter that has a gradient."""
        if self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_optimizer_pre_hooks \
                or _global_optimizer_post_hooks or torch.autograd._profiler_enabled():
            return _step_with_hooks(self, closure)
        return self._step(closure)

    # the base class wraps step() in hooks and a profiler's range, at twice a
    # small step's cost: they run where there are any
    step.hooked = True

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        held = self._held() if self._native is None else self._native
        hyper, lrs = [], []
        for group in self.param_groups:
            self._check_numbers(group)
            if not group["params"]:
                continue
            lr, (b1, b2) = group["lr"], group["betas"]
            on_device = isinstance(lr, torch.Tensor)
            hyper += (0.0 if on_device else lr, b1, b2, group["eps"], group["weight_decay"])
            lrs.append(lr if on_device else None)
        clip = self.max_grad_norm is not None
        if clip:
            if not self.max_grad_norm > 0.0:
                raise ValueError(f"max_grad_norm must be positive, got {self.max_grad_norm}")
            if self.grad_norm is None:
                self.grad_norm = torch.zeros((), device=self._device)
        held.step(hyper, lrs, self.max_grad_norm if clip else -1.0,
                  self.grad_norm if clip else self._arenas[0]["ticket"])
        return loss

    # ------------------------------------------------------------- states

    def moments(self, group: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """m and v of a parameter group as float32, each tensor's values at the
        start of whole blocks of 256, in the parameters' order.  With 32-bit
        states these are the states themselves."""
        a = self._arenas[group]
        if self.state_bits == 32:
            return a["m"], a["v"]
        if not a["m"].numel():  # a group without parameters
            return a["m"].float(), a["v"].float()
        return nat.loaded_ops().adam_unpack(a["m"], a["v"], a["scales"])

    @torch.no_grad()
    def set_moments(self, m: torch.Tensor, v: torch.Tensor, step: int, group: int = 0) -> None:
        """Take over moments in the layout of ``moments()``, after ``step``
        steps; rounded to codes where states have 8 bits."""
        a = self._arenas[group]
        for t in (m, v):
            if t.shape != a["m"].shape or t.dtype != torch.float32 or t.device != a["m"].device:
                raise ValueError(f"moments must be float32 {tuple(a['m'].shape)} on {a['m'].device}, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
        if self.state_bits == 32:
            a["m"].copy_(m)
            a["v"].copy_(v)
        elif m.numel():
            nat.loaded_ops().adam_pack_(m.contiguous(), v.contiguous(), a["m"], a["v"], a["scales"])
        a["steps"].fill_(int(step))

    @torch.no_grad()
    def load_state_dict(self, state_dict: Dict[str, Any]) -> None:
        """Copies the saved values into the states, and saved learning rates into
        the tensors that hold them here: both stay where they are, so that
        captured graphs see the loaded values, and nothing is shared with
        ``state_dict``.  Hooks that are registered for loading run."""
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        groups, saved = self.param_groups, state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in saved]:
            raise ValueError("the saved state is of other parameter groups")
        pairs = []
        for g, s in zip(groups, saved):
            for p, index in zip(g["params"], s["params"]):
                own, new = self.state[p], state_dict["state"].get(index, {})
                if set(own) != set(new) or any(own[k].shape != new[k].shape or own[k].dtype != new[k].dtype for k in own):
                    raise ValueError("the saved state is of other parameters, or of other state_bits or remainder")
                pairs += [(own[k], new[k]) for k in own]
        for own, new in pairs:
            own.copy_(new)
        taken: List[torch.Tensor] = []
        for g, s in zip(groups, saved):
            for k, value in s.items():
                if k == "lr":
                    self._load_rate(g, value, taken)
                elif k != "params":
                    g[k] = tuple(value) if k == "betas" else copy.deepcopy(value)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    def _load_rate(self, group: Dict[str, Any], value: Union[float, torch.Tensor], taken: List[torch.Tensor]) -> None:
        """taken: the tensors that have taken a group's rate so far."""
        own = group["lr"]
        if not isinstance(own, torch.Tensor):
            if isinstance(value, torch.Tensor):
                value = value.detach().to(self._device, torch.float32, copy=True)
            group["lr"] = value
            return
        if any(own is t for t in taken) and float(own) != float(value):
            own = group["lr"] = own.clone()  # groups that had one rate and now have two
        own.copy_(value.reshape(own.shape) if isinstance(value, torch.Tensor) else torch.full_like(own, value))
        taken.append(own)

    def __getstate__(self):
        raise TypeError("an AdamW is not copied or pickled: save its state_dict()")


_step_with_hooks = torch.optim.Optimizer.profile_hook_step(AdamW._step)
