"""swiglu8 where the sigmoid is below the smallest normal fp32 number: a bf16
product there can still be a normal number, and its gradients too.

Bounds: one rounding to bf16; before it the exponential's argument, up to 140
in magnitude, is rounded (2^-24 of it) and the sigmoid itself may be a
denormal number, whose spacing is 2^-149.
"""
import pytest
import torch

F8 = torch.float64


@pytest.mark.gpu
@pytest.mark.parametrize("k", [128, 131])
def test_products_and_gradients(k):
    from rocm_qlora.activation8 import swiglu8
    gates = torch.arange(-96.0, -79.5, 0.5, device="cuda")
    gate = gates[:, None].expand(-1, k).to(torch.bfloat16).contiguous().requires_grad_()
    up = torch.full_like(gate, 1.5).requires_grad_()
    h = swiglu8(gate, up)
    dgate, dup = torch.autograd.grad(h, (gate, up), torch.full_like(h, 2.0))
    g = gate.detach().to(F8)
    p = torch.sigmoid(g)
    # the packed gate is 127 * (|g| / 127), up to 2^-23 of it off; p by |g| times that
    e = p * (g.abs() * 2.0 ** -22 + 2.0 ** -20) + 2.0 ** -149
    scale = 2.0 ** -8
    for got, want, err in ((h, g * p * 1.5, 1.5 * g.abs() * e), (dup, 2 * g * p, 2 * g.abs() * e),
                           (dgate, 3 * p * (1 + g * (1 - p)), 3 * (1 + g.abs()) * e)):
        off = (got.to(F8) - want).abs()
        bound = scale * (want.abs() + err) + err + 2.0 ** -134  # half of bf16's smallest step
        assert bool((off <= bound).all()), float((off / want.abs()).max())
