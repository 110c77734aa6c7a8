"""Tracing: on FakeTensors and under make_fx the public operators give shapes,
types and a graph of their inner operators, and launch nothing."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

BF = torch.bfloat16


def adapters(grad, device):
    from rocm_qlora.lora import adapters_add
    e = lambda *s, dtype=BF: torch.empty(*s, device=device, dtype=dtype)  # noqa: E731
    base, x, A, B, s = e(2, 3, 32), e(2, 3, 160), e(1, 160, 8), e(1, 32, 8), e(1, dtype=torch.float32)
    if not grad:
        return [(adapters_add(base, x, A, B, s), (2, 3, 32), BF)]
    leaves = [t.requires_grad_() for t in (base, x, A, B)]
    y = adapters_add(*leaves, s)
    return [(y, (2, 3, 32), BF)] + [(g, t.shape, BF) for g, t in zip(torch.autograd.grad(y.float().sum(), leaves), leaves)]


def activations(grad, device):
    from rocm_qlora.activation8 import pack_activation, swiglu8, unpack_activation
    gate, up = (torch.empty(2, 3, 200, device=device, dtype=BF, requires_grad=grad) for _ in range(2))
    h, packed = swiglu8(gate, up, pack_output=True)
    found = [(h, (2, 3, 200), BF), (packed.codes, (6, 256), torch.int8), (packed.scales, (6, 2), torch.float32),
             (unpack_activation(packed), (2, 3, 200), BF), (pack_activation(gate).codes, (6, 256), torch.int8),
             (swiglu8(gate, up), (2, 3, 200), BF)]
    if grad:
        found += [(g, (2, 3, 200), BF) for g in torch.autograd.grad(h.float().sum(), (gate, up))]
    return found


def preference(grad, device):
    from rocm_qlora.preference import preference_loss, token_logprobs
    logits = torch.empty(4, 3, 50, device=device, dtype=BF, requires_grad=grad)
    labels = torch.empty(4, 3, device=device, dtype=torch.int64)
    f32 = torch.float32
    out = preference_loss(logits, labels, torch.empty(4, 3, device=device))
    lp = token_logprobs(logits, labels)
    found = [(out.loss, (), f32), (out.logps, (4,), f32), (out.chosen_rewards, (2,), f32), (lp, (4, 3), f32)]
    if grad:
        found += [(torch.autograd.grad(out.loss, logits)[0], (4, 3, 50), BF),
                  (torch.autograd.grad(lp.sum(), logits)[0], (4, 3, 50), BF)]
    return found


# without a GPU autograd itself has no streams for fake CUDA tensors
@pytest.mark.parametrize("grad,device", [(False, "cuda"), (True, "meta"),
                                         pytest.param(True, "cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("which", [adapters, activations, preference])
def test_fake_tensors(which, grad, device):
    from torch._subclasses.fake_tensor import FakeTensor
    with FakeTensorMode(allow_non_fake_inputs=False):
        for value, shape, dtype in which(grad, device):
            assert isinstance(value, FakeTensor) and value.shape == tuple(shape) and value.dtype == dtype
            assert value.device.type == device


def test_graph():
    """make_fx sees the inner operators, so what it traces can run."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from rocm_qlora.activation8 import swiglu8
    from rocm_qlora.lora import adapters_add

    def f(base, x, A, B, s):
        return swiglu8(adapters_add(base, x, A, B, s), base)

    e = lambda *s, dtype=BF: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    graph = make_fx(f)(e(4, 32), e(4, 16), e(1, 16, 8), e(1, 32, 8), e(1, dtype=torch.float32))
    names = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    assert any("rocm_qlora.adapters" in n for n in names) and any("rocm_qlora.swiglu8" in n for n in names), names


@pytest.mark.gpu
def test_traced_graph_runs():
    """What make_fx traced on FakeTensors computes the operators' results."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from rocm_qlora.activation8 import pack_activation, swiglu8, unpack_activation
    from rocm_qlora.lora import adapters_add
    from rocm_qlora.preference import preference_loss

    def f(base, x, A, B, s, labels, ref):
        h = swiglu8(adapters_add(base, x, A, B, s), base)
        h = unpack_activation(pack_activation(h))
        return preference_loss(h.view(2, 2, 32), labels, ref).loss

    g = torch.Generator(device="cuda").manual_seed(0)
    draw = lambda *shape, dtype=BF: torch.randn(*shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    args = (draw(4, 32), draw(4, 16), draw(1, 16, 8), draw(1, 32, 8), draw(1, dtype=torch.float32),
            torch.tensor([[1, 5], [2, 7]], device="cuda"), draw(2, 2, dtype=torch.float32))
    graph = make_fx(f, tracing_mode="fake")(*args)
    assert torch.equal(graph(*args), f(*args))
