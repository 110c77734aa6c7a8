"""Inputs and upstream gradients that are one row for all rows (row stride 0),
as expand() and the backward of a sum over rows make them, and rows that
overlap: the results are those of a contiguous copy, bit for bit."""
import pytest
import torch

DTYPES = [torch.bfloat16, torch.float16]


def leaf(*shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype).requires_grad_()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(70,), (3, 20), (1, 9)])
@pytest.mark.parametrize("k,n,rank", [(64, 136, 16), (65, 131, 40)])
@pytest.mark.parametrize("packed", [False, True])
def test_adapters_upstream_of_a_sum_over_rows(shape, k, n, rank, packed, dtype):
    from rocm_qlora.activation8 import pack_activation
    from rocm_qlora.lora import adapters_add
    base, x = leaf(*shape, n, dtype=dtype, seed=1), leaf(*shape, k, dtype=dtype, seed=2)
    A, B = leaf(1, k, rank, dtype=dtype, seed=3), leaf(1, n, rank, dtype=dtype, seed=4)
    s, up = torch.full((1,), 0.7, device="cuda"), leaf(*shape[1:], n, dtype=dtype, seed=5).detach()
    y = adapters_add(base, x, A, B, s, packed_x=pack_activation(x) if packed else None)
    got = torch.autograd.grad(y.sum(0), (base, x, A, B), up, retain_graph=True)
    want = torch.autograd.grad(y, (base, x, A, B), up.expand(*shape, n).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(64, 136), (65, 131)])
def test_adapters_of_expanded_inputs(k, n, dtype):
    from rocm_qlora.activation8 import pack_activation
    from rocm_qlora.lora import AdapterPlan, adapters_add
    rows = 50
    x, base = leaf(1, k, dtype=dtype, seed=1), leaf(1, n, dtype=dtype, seed=2)
    A, B, dy = (leaf(3, k, 16, dtype=dtype, seed=3), leaf(3, n, 16, dtype=dtype, seed=4),
                leaf(rows, n, dtype=dtype, seed=5).detach())
    s, plan = torch.ones(3, device="cuda"), AdapterPlan(torch.arange(rows) % 3, 3)
    for packed in (None, pack_activation(x.expand(rows, k))):
        results = []
        for copy in (False, True):
            xe, be = x.expand(rows, k), base.expand(rows, n)
            if copy:
                xe, be = xe.contiguous(), be.contiguous()
            y = adapters_add(be, xe, A, B, s, plan, packed_x=packed)
            with torch.no_grad():
                assert torch.equal(adapters_add(be, xe, A, B, s, plan), y)
            results.append((y, *torch.autograd.grad(y, (base, x, A, B), dy)))
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, *DTYPES])
@pytest.mark.parametrize("rows,k", [(40, 256), (7, 131)])
def test_activations(rows, k, dtype):
    from rocm_qlora.activation8 import pack_activation, swiglu8
    gate, up, v = leaf(rows, k, dtype=dtype, seed=1), leaf(rows, k, dtype=dtype, seed=2), leaf(k, dtype=dtype, seed=3)
    h = swiglu8(gate, up)
    got = torch.autograd.grad(h.sum(0), (gate, up), v.detach(), retain_graph=True)
    want = torch.autograd.grad(h, (gate, up), v.detach().expand(rows, k).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    row = v.expand(rows, k)
    assert torch.equal(swiglu8(row, up), swiglu8(row.contiguous(), up))
    assert torch.equal(swiglu8(gate, row), swiglu8(gate, row.contiguous()))
    windows = torch.randn(rows + k, device="cuda").to(dtype).unfold(0, k, 1)[:rows]  # rows that overlap
    for part in (row, windows):
        p, q = pack_activation(part), pack_activation(part.contiguous())
        assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)


@pytest.mark.gpu
def test_layer():
    """The layer's backward after a sum over rows, with expanded inputs."""
    from rocm_qlora.lora import AdapterBank, MultiLoRALinear
    from rocm_qlora.quantization import QuantLinear
    torch.manual_seed(0)
    linear = torch.nn.Linear(256, 320, bias=False, device="cuda", dtype=torch.bfloat16)
    layer = MultiLoRALinear(QuantLinear.from_linear(linear, bits=4), AdapterBank(256, 320, 1, 16, device="cuda"))
    torch.nn.init.normal_(layer.bank.lora_A), torch.nn.init.normal_(layer.bank.lora_B)
    x = leaf(1, 256, dtype=torch.bfloat16, seed=1)
    y = layer(x.expand(30, 256))
    up = torch.randn(320, device="cuda").bfloat16()
    leaves = (x, layer.bank.lora_A, layer.bank.lora_B)
    got = torch.autograd.grad(y.sum(0), leaves, up, retain_graph=True)
    want = torch.autograd.grad(y, leaves, up.expand(30, 320).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
