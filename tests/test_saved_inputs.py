"""What a node does not need for its backward it does not keep: neither the
memory nor the right to change the tensor afterwards."""
import pytest
import torch


def operands():
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    return [e(4, 32), e(4, 16), e(1, 16, 8), e(1, 32, 8), e(1, dtype=torch.float32)]


@pytest.mark.parametrize("needs", [(0,), (1,), (3,), (0, 1, 3)])
def test_x_without_a_gradient_of_a(needs):
    from rocm_qlora.lora import adapters_add
    t = operands()
    for i in needs:
        t[i].requires_grad_()
    x = t[1] * 1  # not a leaf, so that it may be written where it needs a gradient
    y = adapters_add(t[0], x, *t[2:])
    with torch.no_grad():
        x.zero_()
    grads = torch.autograd.grad(y, [t[i] for i in needs], torch.empty_like(y))
    assert [g.shape for g in grads] == [t[i].shape for i in needs]


def test_x_with_a_gradient_of_a():
    from rocm_qlora.lora import adapters_add
    t = operands()
    t[2].requires_grad_()
    y = adapters_add(*t)
    t[1].zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, t[2], torch.empty_like(y))


@pytest.mark.gpu
def test_layer_with_frozen_a():
    from rocm_qlora.lora import AdapterBank, MultiLoRALinear
    from rocm_qlora.quantization import QuantLinear
    torch.manual_seed(0)
    linear = torch.nn.Linear(256, 320, bias=False, device="cuda", dtype=torch.bfloat16)
    layer = MultiLoRALinear(QuantLinear.from_linear(linear, bits=4), AdapterBank(256, 320, 1, 16, device="cuda"))
    torch.nn.init.normal_(layer.bank.lora_A), torch.nn.init.normal_(layer.bank.lora_B)
    x = torch.randn(5, 256, device="cuda").bfloat16()
    up = torch.randn(5, 320, device="cuda").bfloat16()
    want, = torch.autograd.grad(layer(x), layer.bank.lora_B, up)
    layer.bank.lora_A.requires_grad_(False)
    y = layer(x)
    x.zero_()
    got, = torch.autograd.grad(y, layer.bank.lora_B, up)
    assert torch.equal(got, want)
