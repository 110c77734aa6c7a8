"""The adapters' plan and packed inputs have to be on the device of the rows,
of the right types and sizes: refused before anything is launched.  Tensors
of the meta device stand for the GPU's here."""
import pytest
import torch

BF = torch.bfloat16


def made(device, rows=4, k=160, n=32, count=1, rank=8):
    e = lambda *s, dtype=BF: torch.empty(*s, device=device, dtype=dtype)  # noqa: E731
    return e(rows, n), e(rows, k), e(count, k, rank), e(count, n, rank), e(count, dtype=torch.float32)


def operators():
    from rocm_qlora import _native as nat
    return nat.loaded_ops()


def packed(device, rows=4, columns=256, blocks=2, code=torch.int8, scale=torch.float32, scale_device=None):
    return (torch.empty(rows, columns, device=device, dtype=code),
            torch.empty(rows, blocks, device=scale_device or device, dtype=scale))


def plan_words(rows=4, count=1, tile=16):
    from rocm_qlora import _native as nat
    return nat.load_library().rq_adapter_plan_words(rows, count, tile)


def add(device="meta", plan=None, codes=None, scales=None):
    return operators().adapters_add(*made(device), plan, 4, 1, 16, codes, scales)


def test_accepted():
    plan = torch.empty(plan_words(), device="meta", dtype=torch.int32)
    assert add(plan=plan).shape == (4, 32)
    base, x, A, B, s = made("meta")
    codes, scales = packed("meta")
    y = operators().adapters_add(base, x, A.requires_grad_(), B, s, plan, 4, 1, 16, codes, scales)
    grad, = torch.autograd.grad(y, A, torch.empty_like(y))
    assert grad.shape == A.shape


def test_plan_elsewhere():
    words = plan_words()
    with pytest.raises(Exception, match="device"):
        add(plan=torch.empty(words, dtype=torch.int32))
    with pytest.raises(Exception, match="plan"):
        add(plan=torch.empty(words, device="meta", dtype=torch.int64))
    with pytest.raises(Exception, match="plan"):
        add(plan=torch.empty(words, 2, device="meta", dtype=torch.int32)[:, 0])


@pytest.mark.parametrize("args", [
    dict(device="cpu"), dict(device="meta", scale_device="cpu"), dict(device="cpu", scale_device="meta")])
def test_packed_input_elsewhere(args):
    with pytest.raises(Exception, match="device"):
        operators().adapters_add(*made("meta"), None, 0, 0, 0, *packed(**args))


@pytest.mark.parametrize("args", [
    dict(code=torch.uint8), dict(code=torch.int16), dict(scale=torch.float64), dict(scale=BF), dict(blocks=1),
    dict(blocks=3), dict(columns=160), dict(rows=5)])
def test_packed_input_of_another_kind(args):
    """At the call, not in its backward."""
    base, x, A, B, s = made("meta")
    with pytest.raises(ValueError, match="packed_x"):
        operators().adapters_add(base, x, A.requires_grad_(), B, s, None, 0, 0, 0, *packed("meta", **args))
    codes, scales = packed("meta")
    with pytest.raises(ValueError, match="packed_x"):
        operators().adapters_add(base, x, A, B, s, None, 0, 0, 0, codes, scales.t().contiguous().t())
    with pytest.raises(ValueError, match="packed_x"):
        operators().adapters_add(base, x, A, B, s, None, 0, 0, 0, codes, None)


class Plan:
    """What adapters_add reads of an AdapterPlan."""

    def __init__(self, data, rows=4, count=1, tile=16):
        self.data, self.rows, self.count, self.tile = data, rows, count, tile


@pytest.mark.gpu
def test_on_the_gpu():
    """The public forms: a plan or a packed input that was moved to the host is refused."""
    from rocm_qlora.activation8 import PackedActivation, pack_activation
    from rocm_qlora.lora import AdapterBank, AdapterPlan, LoRALinear, MultiLoRALinear, adapters_add
    from rocm_qlora.quantization import QuantLinear
    base, x, A, B, s = made("cuda")
    x.zero_(), base.zero_()
    plan = AdapterPlan(torch.zeros(4, dtype=torch.int64), 1)
    there = Plan(plan.data.cpu(), tile=plan.tile)
    p = pack_activation(x)
    off = [PackedActivation(p.codes.cpu(), p.scales.cpu(), p.shape, p.dtype),
           PackedActivation(p.codes, p.scales.cpu(), p.shape, p.dtype)]
    linear = torch.nn.Linear(160, 32, bias=False, device="cuda", dtype=BF)
    quantized = QuantLinear.from_linear(linear, bits=4)
    layer, lora = MultiLoRALinear(quantized, AdapterBank(160, 32, 1, 8, device="cuda")), LoRALinear(quantized).cuda()
    for call in (lambda: adapters_add(base, x, A, B, s, there), lambda: adapters_add(base, x, A, B, s, there, out=base),
                 lambda: layer(x, there)):
        with pytest.raises(Exception, match="device"):
            call()
    for q in off:
        for call in (lambda: adapters_add(base, x, A, B, s, packed_x=q), lambda: layer(x, None, q), lambda: lora(x, q)):
            with pytest.raises(Exception, match="device"):
                call()


def test_inner_operators():
    """The operators below the differentiable ones check for themselves."""
    ops = operators()
    base, x, A, B, s = made("meta")
    cpu = made("cpu")
    plan = torch.empty(plan_words(), dtype=torch.int32)
    mid = torch.empty(4, 8, device="meta", dtype=torch.float32)
    codes, scales = packed("meta")
    bad = [lambda: ops.adapters_apply(x, A, B, s, base, plan, 16), lambda: ops.adapters_apply(x, cpu[2], B, s, base, None, 0),
           lambda: ops.adapters_apply(x, A, cpu[3], s, base, None, 0), lambda: ops.adapters_apply(x, A, B, cpu[4], base, None, 0),
           lambda: ops.adapters_apply(x, A, B, s, cpu[0], None, 0), lambda: ops.adapters_apply_(base, x, A, B, s, cpu[0], None, 0),
           lambda: ops.adapters_apply_(cpu[0], x, A, B, s, base, None, 0), lambda: ops.adapters_mid(x, A, B, s, plan, 16),
           lambda: ops.adapters_grad(x, None, mid, 160, 1, BF, plan, 16),
           lambda: ops.adapters_grad(x, None, mid.new_empty(4, 8, device="cpu"), 160, 1, BF, None, 0),
           lambda: ops.adapters_grad(codes, scales.new_empty(4, 2, device="cpu"), mid, 160, 1, BF, None, 0),
           lambda: ops.act8_unpack(codes, scales.new_empty(4, 2, device="cpu"), 160, BF)]
    gate = torch.empty(4, 160, device="meta")
    two = torch.empty(2, 4, 256, device="meta", dtype=torch.int8), torch.empty(2, 4, 2, device="meta")
    logits, labels = torch.empty(2, 3, 9, device="meta"), torch.empty(2, 3, device="meta", dtype=torch.int64)
    stats, slopes = torch.empty(2, 3, 4, device="meta"), torch.empty(2, device="meta")
    host = lambda t: torch.empty_like(t, device="cpu")  # noqa: E731
    bad += [lambda: ops.swiglu8_forward(gate, host(gate), 2), lambda: ops.swiglu8_backward(gate, host(two[0]), two[1]),
            lambda: ops.swiglu8_backward(gate, two[0], host(two[1])), lambda: ops.token_logprobs(logits, host(labels), -100),
            lambda: ops.preference_forward(logits, labels, host(stats[..., 0].contiguous()), -100, 0, 0.1, 0.0),
            lambda: ops.token_logprobs_grad(logits, labels, -100, host(stats), slopes, None),
            lambda: ops.token_logprobs_grad(logits, labels, -100, stats, host(slopes), None),
            lambda: ops.token_logprobs_grad(logits, labels, -100, stats, slopes, torch.empty(()))]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError, match="device"):
            call()
            pytest.fail(f"call {i} was accepted")
