"""The operators of a training step together: a base in microscaled 4 bits, its
adapters, packed activations, clipping and AdamW, against the same step in 64
bits; and the example that runs them."""
import math

import pytest
import torch

from tests.test_mx4 import kept

F8, BF = torch.float64, torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(48, 256, 192), (300, 200, 136)])
def test_layer_over_a_4_bit_base(rows, k, n):
    """Output and gradients of MultiLoRALinear over Mx4Linear.  The base's output
    is rounded to bf16 before the adapters' sum is added and rounded again; a
    product's terms are summed in 32 bits (2^-23 a term of their magnitudes)."""
    from rocm_qlora.lora import AdapterBank, AdapterPlan, MultiLoRALinear
    from rocm_qlora.mx4 import Mx4Linear
    torch.manual_seed(rows)
    linear = torch.nn.Linear(k, n, dtype=BF, device="cuda")
    bank = AdapterBank(k, n, 2, 8, BF, linear.weight.device)
    with torch.no_grad():
        bank.lora_A.normal_(0, k ** -0.5)
        bank.lora_B.normal_(0, 0.3)
        bank.scaling.copy_(torch.tensor([0.5, 1.5]))
    layer = MultiLoRALinear(Mx4Linear.from_linear(linear), bank)
    bank.requires_grad_(True)
    ids = torch.arange(rows, device="cuda") % 3 - 1
    x = torch.randn(rows, k, device="cuda", dtype=BF, requires_grad=True)
    dy = torch.randn(rows, n, device="cuda", dtype=BF) * 0.1
    y = layer(x, AdapterPlan(ids, 2))
    dx, dA, dB = torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), dy)
    w, xk = kept(linear.weight), kept(x)
    x8, d8 = x.detach().to(F8), dy.to(F8)
    base = xk @ w.t() + linear.bias.to(F8)
    want, wx = base.clone(), d8 @ w
    a_part = torch.zeros_like(x8)
    for a in range(2):
        at = ids == a
        A, B, s = bank.lora_A[a].to(F8), bank.lora_B[a].to(F8), float(bank.scaling[a])
        t, g = s * (x8[at] @ A), s * (d8[at] @ B)
        want[at] += t @ B.t()
        a_part[at] = g @ A.t()
        for got, ref, terms in ((dA[a], x8[at].t() @ g, x8[at].abs().t() @ g.abs()),
                                (dB[a], d8[at].t() @ t, d8[at].abs().t() @ t.abs())):
            bound = 2.0 ** -8 * ref.abs() + (rows + k) * 2.0 ** -22 * terms + 2.0 ** -100
            assert bool(((got.to(F8) - ref).abs() <= bound).all())
    slack = (k + 64) * 2.0 ** -22 * (xk.abs() @ w.abs().t() + want.abs() + 1)
    assert bool(((y.to(F8) - want).abs() <= 2.0 ** -8 * (base.abs() + want.abs()) * 1.01 + slack).all())
    # two bf16 gradients of x, each rounded, and their sum
    slack = (n + 64) * 2.0 ** -22 * (d8.abs() @ w.abs() + a_part.abs() + 1)
    bound = 2.0 ** -8 * (wx.abs() + a_part.abs() + (wx + a_part).abs()) * 1.01 + slack
    assert bool(((dx.to(F8) - wx - a_part).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_captured_training_step(bits):
    """Forward, backward and the clipped step captured as one graph: its replays
    are the eager steps."""
    from rocm_qlora.lora import AdapterBank, MultiLoRALinear
    from rocm_qlora.mx4 import Mx4Linear
    from rocm_qlora.optim import AdamW

    def made():
        torch.manual_seed(1)
        linear = torch.nn.Linear(160, 96, bias=False, dtype=BF, device="cuda")
        bank = AdapterBank(160, 96, 1, 8, BF, linear.weight.device)
        torch.nn.init.normal_(bank.lora_A, std=160 ** -0.5)
        bank.scaling.fill_(2.0)
        bank.requires_grad_(True)
        return MultiLoRALinear(Mx4Linear.from_linear(linear), bank), AdamW(
            bank.parameters(), lr=1e-2, state_bits=bits, remainder=True, max_grad_norm=0.5)

    x = torch.randn(40, 160, device="cuda", dtype=BF)
    target = torch.randn(40, 96, device="cuda", dtype=BF)

    def step(layer, opt):
        loss = (layer(x) - target).float().square().mean()
        grads = torch.autograd.grad(loss, list(layer.bank.parameters()))
        for p, g in zip(layer.bank.parameters(), grads):
            p.grad = g
        opt.step()
        return loss

    eager, eager_opt = made()
    for _ in range(5):
        step(eager, eager_opt)
    layer, opt = made()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(layer, opt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(layer, opt)
    for _ in range(4):
        graph.replay()
    for p, q in zip(layer.bank.parameters(), eager.bank.parameters()):
        assert int(opt.state[p]["step"]) == 5 and torch.equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("base,bits", [("mx4", 8), ("mx4", 32), ("nf4", 8)])
def test_example_with_a_4_bit_base_and_its_own_optimizer(base, bits):
    from rocm_qlora.examples.preference_training import train
    losses = train(steps=3, base=base, state_bits=bits)
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses)
