"""Banks and packed codes that are views into a larger buffer at an address
that is no multiple of 16 bytes: the results are those of aligned copies."""
import pytest
import torch


def off(t):
    """t's values in a view one element further than a fresh allocation starts."""
    buffer = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    view = buffer[1:].view(t.shape)
    view.copy_(t)
    assert view.is_contiguous() and view.data_ptr() % 16
    return view


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [3, 200])
def test_adapters(rows, dtype):
    from rocm_qlora.activation8 import PackedActivation, pack_activation, unpack_activation
    from rocm_qlora.lora import AdapterPlan, adapters_add
    g = torch.Generator(device="cuda").manual_seed(rows)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, base, dy, A, B = draw(rows, 264), draw(rows, 136), draw(rows, 136), draw(2, 264, 16), draw(2, 136, 16)
    s, plan, p = torch.ones(2, device="cuda"), AdapterPlan(torch.arange(rows) % 2, 2), pack_activation(x)
    moved = PackedActivation(off(p.codes), off(p.scales), p.shape, p.dtype)
    assert torch.equal(unpack_activation(moved), unpack_activation(p))
    results = []
    for a, b, q in ((A, B, p), (off(A), off(B), moved)):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        y = adapters_add(base, x, a, b, s, plan, packed_x=q)
        with torch.no_grad():
            assert torch.equal(adapters_add(base, x, a, b, s, plan), y)
            assert torch.equal(adapters_add(base, x, a, b, s, plan, out=base.clone()), y)
        results.append((y, *torch.autograd.grad(y, (a, b), dy)))
    assert all(torch.equal(u, v) for u, v in zip(*results))
