"""What happens to the states of rocm_qlora.optim.AdamW from outside a step:
parameters that are written over, states and learning rates that are loaded,
groups without parameters, gradients that are views or not finite."""
import math

import pytest
import torch

from tests.test_optim import BF, F4, F8, HF, HALF, NUMBERS, TINY, formula, kept8, made


def stepped(values, bits, steps=3, seed=20):
    """A bf16 parameter with a remainder, after some steps."""
    from rocm_qlora.optim import AdamW
    g = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(values, generator=g).to(BF).cuda())
    opt = AdamW([p], **NUMBERS, state_bits=bits, remainder=True)
    for _ in range(steps):
        p.grad = (torch.randn(values, generator=g) * 0.1).to(BF).cuda()
        opt.step()
    return p, opt


def check_from(p, opt, start, t):
    """One step of p from the values `start`, to which a remainder of less than
    a unit in their last place may belong (2^-7 of them; nothing of it at 0 but
    2^-134): p is the formula's, rounded to bf16 once."""
    m, v = (x[:p.numel()].clone() for x in opt.moments())
    opt.step()
    want, _, _, _, step = formula(start, p.grad, m, v, t)
    slack = (2.0 ** -7 + 2.0 ** -22) * start.to(F8).abs() + 2.0 ** -18 * step + 2.0 ** -133
    bound = HALF[BF] * (want.abs() + slack) + slack + TINY[BF]
    off = (p.detach().to(F8) - want).abs()
    assert bool((off <= bound).all()), (int((~(off <= bound)).sum()), float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("write", ["zero", "negative zero", "negated", "half", "some zero"])
def test_a_parameter_written_over_goes_on_from_what_was_written(write, bits):
    p, opt = stepped(1000, bits)
    low = opt.state[p]["remainder"]
    assert bool((low < 0).any()) and bool((low > 0).any())
    with torch.no_grad():
        if write == "zero":
            p.zero_()
        elif write == "negative zero":
            p.fill_(-0.0)
        elif write == "negated":
            p.neg_()
        elif write == "half":
            p.fill_(0.5)
        else:
            p[::3] = 0.0
    check_from(p, opt, p.detach().clone(), 4)
    check_from(p, opt, p.detach().clone(), 5)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_infinities_written_into_a_parameter_stay(bits):
    p, opt = stepped(600, bits)
    start = p.detach().clone()
    start[:200], start[200:400] = float("inf"), float("-inf")
    with torch.no_grad():
        p.copy_(start)
    opt.step()
    assert torch.equal(p.detach()[:400], start[:400]) and bool(torch.isfinite(p.detach()[400:]).all())


@pytest.mark.gpu
def test_merged_and_reset_adapters_go_on():
    """merge_lora zeroes an adapter's matrices, set_adapter writes another one."""
    from rocm_qlora import LoRALinear, QuantLinear
    from rocm_qlora.lora import AdapterBank
    from rocm_qlora.optim import AdamW
    torch.manual_seed(21)
    layer = LoRALinear(QuantLinear.from_linear(torch.nn.Linear(128, 64, bias=False, dtype=BF, device="cuda"), bits=4),
                       r=8).cuda()
    layer.lora_A.data, layer.lora_B.data = layer.lora_A.data.to(BF), layer.lora_B.data.to(BF)
    bank = AdapterBank(128, 64, 2, 16, BF, torch.device("cuda"))
    torch.nn.init.normal_(bank.lora_A)
    torch.nn.init.normal_(bank.lora_B)
    params = [layer.lora_A, layer.lora_B, bank.lora_A, bank.lora_B]
    opts = [AdamW([p], **NUMBERS, remainder=True) for p in params]

    def gradients():
        for p in params:
            p.grad = torch.randn_like(p) * 0.1

    for _ in range(3):
        gradients()
        for o in opts:
            o.step()
    layer.merge_lora()
    layer.unmerge_lora()
    bank.set_adapter(1, torch.randn(8, 128, device="cuda"), torch.zeros(64, 8, device="cuda"), 1.0)
    gradients()
    for p, o in zip(params, opts):
        start = p.detach().clone()
        m, v = (x[:p.numel()].view(p.shape).clone() for x in o.moments())
        o.step()
        want, _, _, _, step = formula(start, p.grad, m, v, 4)
        slack = (2.0 ** -7 + 2.0 ** -22) * start.to(F8).abs() + 2.0 ** -18 * step + 2.0 ** -133
        assert bool(((p.detach().to(F8) - want).abs() <= HALF[BF] * (want.abs() + slack) + slack + TINY[BF]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F4, BF, HF])
@pytest.mark.parametrize("bits", [8, 32])
def test_first_step_from_zero_is_the_step_itself(bits, dtype):
    """lora_B begins at 0, where the step is all of the parameter.  From empty
    moments it is lr' m q with m = rest1 g, q = 1 / (sqrt(rest2 g g) y + eps):
    roundings of 2^-24 are two in m, one and a half in the root of three in v,
    one each in the root, y, the divisor, the quotient, lr', the two products and
    the sum; an approximate root and quotient are off by 2^-23 each.  14 of
    2^-24, and then the type's."""
    from rocm_qlora.optim import AdamW
    g = torch.Generator().manual_seed(22)
    p = torch.nn.Parameter(torch.zeros(5000, dtype=dtype, device="cuda"))
    p.grad = (torch.randn(5000, generator=g) * 10.0 ** (-3 * torch.rand(5000, generator=g))).to(dtype).cuda()
    AdamW([p], **NUMBERS, state_bits=bits).step()
    zero = torch.zeros(5000, device="cuda")
    want, _, _, _, step = formula(zero, p.grad, zero, zero, 1)
    slack = 14 * 2.0 ** -24 * step
    assert bool(((p.detach().to(F8) - want).abs() <= HALF[dtype] * (want.abs() + slack) + slack + TINY[dtype]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_that_are_not_finite_reach_no_other_value(bits):
    """In 32 bits a NaN or an infinity stays where it is; in 8 bits it takes the
    moments of its block, whose other parameters' step is the formula's."""
    from rocm_qlora.optim import AdamW
    g = torch.Generator().manual_seed(23)
    p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
    p.grad = (torch.randn(1024, generator=g) * 0.1).cuda()
    p.grad[300], p.grad[600] = float("nan"), float("inf")
    opt = AdamW([p], **NUMBERS, state_bits=bits)
    opt.step()
    bad = torch.zeros(1024, dtype=torch.bool, device="cuda")
    bad[[300, 600]] = True
    want = formula(torch.ones_like(p), p.grad, torch.zeros_like(p), torch.zeros_like(p), 1)[0]
    off = (p.detach().to(F8) - want).abs()
    assert bool((off[~bad] <= 2.0 ** -22).all()) and not bool(torch.isfinite(p.detach()[bad]).any())
    m, v = opt.moments()
    if bits == 32:
        assert torch.equal(torch.isfinite(m), ~bad) and torch.equal(torch.isfinite(v), ~bad)
        return
    assert bool(torch.isnan(m[256:768]).all()) and bool(torch.isnan(v[256:768]).all())
    f = torch.tensor(1 - 0.9), torch.tensor(1 - 0.999)
    x = p.grad.cpu()
    want = kept8((x * f[0]).numpy(), (x * x * f[1]).numpy())
    for got, w in zip((m, v), want):
        for part in (slice(0, 256), slice(768, 1024)):
            assert torch.equal(got[part].cpu(), torch.from_numpy(w[part]))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_a_gradient_with_a_lazy_sign(bits):
    """The imaginary part of a conjugate is a view whose values are stored with
    the other sign."""
    from rocm_qlora.optim import AdamW
    (p, q), g = made([(300,), (300,)], F4, seed=24), torch.Generator().manual_seed(24)
    q.data.copy_(p.data)
    p.grad = torch._neg_view(torch.randn(300, generator=g).cuda())
    assert p.grad.is_neg()
    q.grad = p.grad.clone()
    AdamW([p], state_bits=bits).step()
    AdamW([q], state_bits=bits).step()
    assert not q.grad.is_neg() and torch.equal(p, q)


# ------------------------------------------------------ loaded learning rates

def with_rate(lr, seed=25, **kw):
    from rocm_qlora.optim import AdamW
    (p,) = made([(300,)], F4, seed=seed)
    return p, AdamW([p], lr=lr, **kw)


def rate(value):
    return torch.full((), value, device="cuda")


@pytest.mark.gpu
def test_a_loaded_rate_is_seen_by_a_captured_step():
    own = rate(1e-2)
    p, opt = with_rate(own)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    q, other = with_rate(rate(0.25))
    other.load_state_dict(opt.state_dict())
    other.param_groups[0]["lr"].fill_(0.25)
    assert float(own) == float(torch.tensor(1e-2))      # each has a rate of its own
    q.data.copy_(p.data)
    opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] is own and float(own) == 0.25
    graph.replay()
    other.step()
    assert torch.equal(p, q) and int(opt.state[p]["step"]) == 2


@pytest.mark.gpu
def test_rates_loaded_from_the_cpu_and_from_numbers():
    p, opt = with_rate(rate(0.5))
    saved = torch.utils._pytree.tree_map(lambda x: x.cpu() if isinstance(x, torch.Tensor) else x, opt.state_dict())
    own = rate(1e-3)
    _, other = with_rate(own)
    other.load_state_dict(saved)
    assert other.param_groups[0]["lr"] is own and float(own) == 0.5
    other.step()
    q, number = with_rate(1e-3)
    number.load_state_dict(saved)                        # takes a tensor of its own, on its device
    lr = number.param_groups[0]["lr"]
    assert lr.is_cuda and lr is not saved["param_groups"][0]["lr"] and float(lr) == 0.5
    number.step()
    _, third = with_rate(0.125)
    other.load_state_dict(third.state_dict())            # a number into the tensor that is there
    assert other.param_groups[0]["lr"] is own and float(own) == 0.125
    other.step()


@pytest.mark.gpu
def test_groups_that_shared_a_rate_take_their_own():
    from rocm_qlora.optim import AdamW
    own = rate(1e-2)
    a, b = made([(300,), (40, 20)], F4, seed=26)
    opt = AdamW([dict(params=[a]), dict(params=[b])], lr=own)
    saved = opt.state_dict()
    opt.load_state_dict(saved)
    assert all(g["lr"] is own for g in opt.param_groups)
    saved["param_groups"][0]["lr"], saved["param_groups"][1]["lr"] = rate(0.5), rate(0.25)
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] is own and [float(g["lr"]) for g in opt.param_groups] == [0.5, 0.25]
    opt.step()


@pytest.mark.gpu
def test_load_state_dict_runs_its_hooks():
    _, opt = with_rate(1e-2)
    _, other = with_rate(1.0)
    called = []

    def before(o, state):
        called.append("before")
        return dict(state, param_groups=[dict(g, lr=0.5) for g in state["param_groups"]])

    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(lambda o: called.append("after"))
    other.load_state_dict(opt.state_dict())
    assert called == ["before", "after"] and other.param_groups[0]["lr"] == 0.5


# ------------------------------------------------------------- empty groups

@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("clip", [None, 0.05])
@pytest.mark.parametrize("place", ["first", "last", "added"])
def test_a_group_without_parameters(place, clip, bits):
    """A split into decayed and other parameters may leave one side empty."""
    from rocm_qlora.optim import AdamW
    (p,), (q,) = made([(300,)], F4, seed=27), made([(300,)], F4, seed=27)
    groups = [dict(params=[p]), dict(params=[], weight_decay=0.0)]
    opt = AdamW(groups[::-1] if place == "first" else groups if place == "last" else groups[:1], **NUMBERS,
                state_bits=bits, max_grad_norm=clip)
    if place == "added":
        opt.add_param_group(groups[1])
    plain = AdamW([q], **NUMBERS, state_bits=bits, max_grad_norm=clip)
    for _ in range(2):
        opt.step()
        plain.step()
    assert torch.equal(p, q) and len(opt.param_groups) == 2
    if clip:
        assert torch.equal(opt.grad_norm, plain.grad_norm)
    empty = 0 if place == "first" else 1
    assert all(x.shape == (0,) and x.dtype == F4 for x in opt.moments(empty))
    opt.set_moments(*opt.moments(empty), 2, empty)
    opt.load_state_dict(opt.state_dict())
    opt.step()
    plain.step()
    assert torch.equal(p, q)


@pytest.mark.gpu
def test_only_empty_groups_and_a_first_parameter_later():
    from rocm_qlora.optim import AdamW
    opt = AdamW([dict(params=[])], **NUMBERS, max_grad_norm=0.5)
    opt.step()
    (p,), (q,) = made([(300,)], F4, seed=28), made([(300,)], F4, seed=28)
    opt.add_param_group(dict(params=[p]))
    opt.step()
    plain = AdamW([q], **NUMBERS, max_grad_norm=0.5)
    plain.step()
    assert torch.equal(p, q) and torch.equal(opt.grad_norm, plain.grad_norm)


@pytest.mark.gpu
def test_a_refused_group_leaves_the_others():
    from rocm_qlora.optim import AdamW
    (p,) = made([(300,)], F4, seed=29)
    opt = AdamW([p], **NUMBERS)
    for group, error in ((dict(params=[torch.nn.Parameter(torch.zeros(8, device="cuda", dtype=F8))]), TypeError),
                         (dict(params=[torch.nn.Parameter(torch.zeros(8, device="cuda"))], lr=-1.0), ValueError)):
        with pytest.raises(error):
            opt.add_param_group(group)
        assert len(opt.param_groups) == 1
        opt.step()
    assert int(opt.state[p]["step"]) == 2 and math.isfinite(float(p.detach().sum()))


def test_empty_groups_need_no_gpu():
    from rocm_qlora.optim import AdamW
    for bits in (8, 32):
        opt = AdamW([dict(params=[]), dict(params=[], lr=0.5)], state_bits=bits, max_grad_norm=1.0)
        assert opt.step() is None and opt.step(lambda: 2.5) == 2.5
        assert len(opt.param_groups) == 2 and opt.moments(1)[0].shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_an_eps_below_the_normal_range_keeps_untouched_values(bits):
    """A value that never had a gradient has a step of 0 / eps."""
    from rocm_qlora.optim import AdamW
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.zeros_like(p)
    p.grad[5] = 0.1
    AdamW([p], lr=1e-2, eps=1e-40, weight_decay=0.0, state_bits=bits).step()
    assert bool((p.detach()[torch.arange(300, device="cuda") != 5] == 1.0).all())
    assert abs(float(p.detach()[5]) - 0.99) <= 2.0 ** -22
