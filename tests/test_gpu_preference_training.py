"""The example that runs adapters, 8-bit activations and the preference loss
together: it starts at log 2 (no adapter has an effect yet) and the loss falls."""
import math

import pytest
import torch


@pytest.mark.gpu
def test_preference_training_example():
    from rocm_qlora.examples.preference_training import train
    losses = train(steps=25)
    assert all(math.isfinite(v) for v in losses)
    # B = 0: policy and reference differ only through the base's two calls on equal rows
    assert abs(losses[0] - math.log(2.0)) < 0.05
    assert sum(losses[-5:]) / 5 < 0.8 * losses[0]


@pytest.mark.gpu
def test_packed_inputs_change_the_gradients_little():
    """One block with packed inputs against the same block without: gradients of
    lora_A differ by the packing alone.  A block's largest value is up to 8
    times its rms (a product of two normal values), so rounding to 1/127 of it
    errs by 8 / 127 / sqrt(12) = 1.8 % of the rms; two packed factors in a
    gradient: 2.6 % of its norm, 3 % with the 16-bit roundings."""
    from rocm_qlora.examples.preference_training import Block
    from rocm_qlora.lora import AdapterPlan
    torch.manual_seed(1)
    block = Block(256, 512, 4, 2, 16)
    for p in block.parameters():
        p.requires_grad_(False)
    banks = [m.bank for m in (block.q, block.gate, block.down)]
    for bank in banks:
        bank.requires_grad_(True)
        with torch.no_grad():
            bank.lora_B.normal_(0.0, 0.02)
    plan = AdapterPlan(torch.arange(96) % 2, 2)
    x = torch.randn(2, 48, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn_like(x)
    import rocm_qlora.examples.preference_training as ex
    pack, swiglu = ex.pack_activation, ex.swiglu8
    leaves = [b.lora_A for b in banks] + [b.lora_B for b in banks]
    packed = torch.autograd.grad(block(x, plan), leaves, dy)
    try:
        ex.pack_activation = lambda t: None
        ex.swiglu8 = lambda g, u, pack_output: (torch.nn.functional.silu(g.float()).mul(u.float()).to(g.dtype), None)
        plain = torch.autograd.grad(block(x, plan), leaves, dy)
    finally:
        ex.pack_activation, ex.swiglu8 = pack, swiglu
    for a, b in zip(packed, plain):
        assert float((a.float() - b.float()).norm()) <= 0.03 * float(b.float().norm())
