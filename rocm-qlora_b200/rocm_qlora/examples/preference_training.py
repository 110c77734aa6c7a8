"""Preference training of adapters over one quantized base, and their serving.

    python -m rocm_qlora.examples.preference_training --steps 20
    python -m rocm_qlora.examples.preference_training --base mx4 --state-bits 8

A small decoder with a vocabulary of its own (random weights, synthetic
prompts) is quantized to NF4, or to microscaled 4 bits.  Its projections carry a bank of two adapters,
both trained in the same batch: each pair of answers belongs to one of them.
The reference model is the same decoder with no adapter on any row.

* ``AdapterPlan`` / ``MultiLoRALinear``: every token uses its pair's adapter;
* ``pack_activation`` / ``swiglu8``: q, k and v share one packed input, gate
  and up another, the down projection takes the one swiglu8 wrote, and the
  backward reads those instead of 16-bit activations;
* ``token_logprobs`` / ``preference_loss``: the reference's log-probabilities
  and the loss, straight from bf16 logits;
* ``Mx4Linear``: the base's weights and inputs in 4 bits (``--base mx4``);
* ``optim.AdamW``: the step of all adapters in two launches, clipped, moments
  in 8 or 32 bits, what bf16 parameters round away kept (``--state-bits``);
* serving: one decode step for rows of both adapters and of none.
"""
import argparse
from typing import List, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from rocm_qlora.activation8 import pack_activation, swiglu8
from rocm_qlora.lora import AdapterBank, AdapterPlan, MultiLoRALinear
from rocm_qlora.mx4 import Mx4Linear
from rocm_qlora.optim import AdamW
from rocm_qlora.preference import preference_loss, token_logprobs
from rocm_qlora.quantization import QuantLinear


class Projection(MultiLoRALinear):
    """An NF4 or MX4 projection with its bank of adapters (A random, B zero: no effect yet)."""

    def __init__(self, k: int, n: int, adapters: int, rank: int, base: str = "nf4"):
        linear = nn.Linear(k, n, bias=False, device="cuda", dtype=torch.bfloat16)
        bank = AdapterBank(k, n, adapters, rank, torch.bfloat16, linear.weight.device)
        nn.init.normal_(bank.lora_A, std=k ** -0.5)
        bank.scaling.fill_(2.0)
        super().__init__(Mx4Linear.from_linear(linear) if base == "mx4" else QuantLinear.from_linear(linear, bits=4), bank)


class Block(nn.Module):
    def __init__(self, d: int, f: int, heads: int, adapters: int, rank: int, base: str = "nf4"):
        super().__init__()
        self.heads = heads
        self.norm1 = nn.RMSNorm(d, device="cuda", dtype=torch.bfloat16)
        self.norm2 = nn.RMSNorm(d, device="cuda", dtype=torch.bfloat16)
        self.q, self.k, self.v, self.o = (Projection(d, d, adapters, rank, base) for _ in range(4))
        self.gate, self.up = Projection(d, f, adapters, rank, base), Projection(d, f, adapters, rank, base)
        self.down = Projection(f, d, adapters, rank, base)

    def forward(self, x: torch.Tensor, plan: AdapterPlan) -> torch.Tensor:
        keep = torch.is_grad_enabled()
        h = self.norm1(x)
        packed = pack_activation(h) if keep else None
        b, length, d = x.shape
        q, k, v = (p(h, plan, packed).view(b, length, self.heads, -1).transpose(1, 2)
                   for p in (self.q, self.k, self.v))
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).reshape(b, length, d)
        x = x + self.o(a, plan, pack_activation(a) if keep else None)
        h = self.norm2(x)
        packed = pack_activation(h) if keep else None
        gate, up = self.gate(h, plan, packed), self.up(h, plan, packed)
        if keep:
            y, packed = swiglu8(gate, up, pack_output=True)
            return x + self.down(y, plan, packed)
        return x + self.down(F.silu(gate) * up, plan)


class Decoder(nn.Module):
    def __init__(self, vocab: int, d: int, f: int, heads: int, layers: int, adapters: int, rank: int,
                 base: str = "nf4"):
        super().__init__()
        self.embed = nn.Embedding(vocab, d, device="cuda", dtype=torch.bfloat16)
        self.blocks = nn.ModuleList(Block(d, f, heads, adapters, rank, base) for _ in range(layers))
        self.norm = nn.RMSNorm(d, device="cuda", dtype=torch.bfloat16)
        self.head = nn.Linear(d, vocab, bias=False, device="cuda", dtype=torch.bfloat16)
        self.requires_grad_(False)
        for m in self.modules():
            if isinstance(m, AdapterBank):
                m.requires_grad_(True)

    def forward(self, ids: torch.Tensor, plan: AdapterPlan) -> torch.Tensor:
        x = self.embed(ids)
        for block in self.blocks:
            x = block(x, plan)
        return self.head(self.norm(x))


def batch_of(pairs: int, length: int, prompt: int, vocab: int, device) -> torch.Tensor:
    """Token ids [2 * pairs, length], chosen answers first: a pair shares its
    prompt; the answer its adapter is to prefer counts up, the other is noise."""
    ids = torch.randint(0, vocab, (2 * pairs, length), device=device)
    ids[pairs:, :prompt] = ids[:pairs, :prompt]
    steps = torch.arange(1, length - prompt + 1, device=device)
    ids[:pairs, prompt:] = (ids[:pairs, prompt - 1:prompt] + steps) % vocab
    return ids


def train(steps: int = 20, pairs: int = 4, length: int = 48, prompt: int = 8, vocab: int = 1000, d: int = 256,
          f: int = 512, heads: int = 4, layers: int = 2, rank: int = 16, lr: float = 2e-3, seed: int = 0,
          report: Optional[int] = None, base: str = "nf4", state_bits: Optional[int] = None) -> List[float]:
    """Train and return the loss of each step; ends with a decode step served
    for both adapters and for none.  ``state_bits`` 8 or 32: the optimizer of
    this package, None: torch's."""
    torch.manual_seed(seed)
    adapters = 2
    model = Decoder(vocab, d, f, heads, layers, adapters, rank, base)
    trained = [p for p in model.parameters() if p.requires_grad]
    if state_bits is None:
        optimizer = torch.optim.AdamW(trained, lr=lr)
    else:
        optimizer = AdamW(trained, lr=lr, state_bits=state_bits, remainder=True, max_grad_norm=1.0)
    device = model.head.weight.device
    owner = torch.arange(pairs, device=device) % adapters        # the adapter that a pair trains
    per_row = owner.repeat(2).repeat_interleave(length)
    plan = AdapterPlan(per_row, adapters)
    no_adapter = AdapterPlan(torch.full_like(per_row, -1), adapters)
    losses = []
    for step in range(steps):
        ids = batch_of(pairs, length, prompt, vocab, device)
        labels = ids.clone()
        labels[:, :prompt] = -100
        with torch.no_grad():
            ref = token_logprobs(model(ids, no_adapter), labels)
        out = preference_loss(model(ids, plan), labels, ref, beta=0.1)
        optimizer.zero_grad(set_to_none=True)
        out.loss.backward()
        optimizer.step()
        losses.append(out.loss.detach())
        if report and step % report == 0:
            margin = (out.chosen_rewards - out.rejected_rewards).mean()
            print(f"step {step}: loss {float(losses[-1]):.4f}, reward margin {float(margin):.4f}")
    with torch.no_grad():  # one token for a request of each adapter and one of none
        rows = AdapterPlan(torch.tensor([0, 1, -1]), adapters)
        logits = model(torch.zeros(3, 1, dtype=torch.long, device=device), rows)
    if report:
        print(f"served: next tokens {logits[:, -1].argmax(-1).tolist()} of adapter 0, adapter 1 and the base")
    return [float(v) for v in losses]


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--pairs", type=int, default=4)
    p.add_argument("--length", type=int, default=48)
    p.add_argument("--base", choices=("nf4", "mx4"), default="nf4")
    p.add_argument("--state-bits", type=int, choices=(8, 32), default=None)
    a = p.parse_args()
    train(steps=a.steps, pairs=a.pairs, length=a.length, report=max(1, a.steps // 10), base=a.base,
          state_bits=a.state_bits)


if __name__ == "__main__":
    main()
