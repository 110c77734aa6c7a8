"""AdamW over many tensors (rocm_qlora.optim): the update and the norm against
the formula in 64 bits, the 8-bit moments bit for bit against their definition
in numpy fp32, and what is refused."""
import math

import numpy as np
import pytest
import torch

F8 = torch.float64
BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32
HALF = {F4: 2.0 ** -24, BF: 2.0 ** -8, HF: 2.0 ** -11}
TINY = {F4: 2.0 ** -150, BF: 2.0 ** -134, HF: 2.0 ** -25}
NUMBERS = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def made(shapes, dtype, seed=0, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).cuda()) for s in shapes]
    for p in params:
        p.grad = (torch.randn(p.shape, generator=g) * scale * torch.exp(torch.randn(p.shape[:1] or (1,), generator=g))
                  .view(-1, *[1] * max(0, p.dim() - 1))).to(dtype).cuda().view(p.shape)
    return params


def formula(p, g, m, v, t, c=1.0, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1):
    """p, m, v after step t in 64 bits, and the size of the terms that the update sums."""
    p, g, m, v = (x.to(F8) for x in (p, g, m, v))
    b1, b2 = betas
    g = g * c
    size = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    by = lr / (1 - b1 ** t) / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lr * weight_decay) - by * m, m, v, size, by * size


def check_params(got, p, step):
    """32-bit values: the decay and its product, the sum, each off by 2^-24 of
    p; fewer than 30 roundings of 2^-24 and an approximate quotient of 2^-22 in
    the step; then one rounding to the type."""
    dt = got.dtype
    slack = 3 * 2.0 ** -24 * p.abs() + 2.0 ** -18 * step
    bound = HALF[dt] * (p.abs() + slack) + slack + TINY[dt]
    off = (got.detach().to(F8) - p).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


SHAPES = [(1,), (255,), (256,), (257,), (7, 33), (16, 1000), (3, 5, 17), (0, 4), (2048,), ()]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F4, BF, HF])
def test_steps_with_32_bit_moments(dtype):
    from rocm_qlora.optim import AdamW
    params = made(SHAPES, dtype)
    opt = AdamW(params, **NUMBERS)
    state = [(torch.zeros_like(p, dtype=F4), torch.zeros_like(p, dtype=F4)) for p in params]
    for t in range(1, 4):
        before = [p.detach().clone() for p in params]
        versions = [p._version for p in params]
        opt.step()
        assert all(p._version > n for p, n in zip(params, versions))
        for i, p in enumerate(params):
            want, m, v, size, step = formula(before[i], p.grad, *state[i], t)
            check_params(p, want, step)
            s = opt.state[p]
            assert int(s["step"]) == t
            # two products and their sum
            assert bool(((s["exp_avg"] - m).abs() <= 3 * 2.0 ** -24 * size + 2.0 ** -148).all())
            assert bool(((s["exp_avg_sq"] - v).abs() <= 5 * 2.0 ** -24 * v + 2.0 ** -148).all())
            state[i] = (s["exp_avg"].clone(), s["exp_avg_sq"].clone())
            p.grad.mul_(-0.7)


def e4m3(t):
    return torch.from_numpy(t).to(torch.float8_e4m3fn).float().numpy()


def root8(t):
    """The codes' values of numbers in [0, 507904]: whole numbers up to 31, then
    16 steps to a power of two, ties to even."""
    step = np.ldexp(np.float32(1), np.maximum(np.frexp(t)[1] - 5, 0)).astype(np.float32)
    return (np.rint(t / step) * step).astype(np.float32)


def kept8(m, v):
    """The values that the 8-bit form of moments [blocks, 256] (fp32) stands for."""
    m, r = m.reshape(-1, 256), np.sqrt(v.reshape(-1, 256))
    with np.errstate(all="ignore"):
        out = []
        for x, most in ((m, np.float32(448)), (r, np.float32(507904))):
            top = np.abs(x).max(-1, keepdims=True)
            bad, live = ~np.isfinite(x).all(-1, keepdims=True), top >= np.float32(2.0 ** -100)
            code = np.where(live & ~bad, x * (most / np.where(live, top, 1)), 0).astype(np.float32)
            code = e4m3(code) if most == 448 else np.where((x > 0) & live, np.maximum(root8(code), 1), 0).astype(np.float32)
            scale = np.where(bad, np.float32("nan"), np.where(live, top / most, 0)).astype(np.float32)
            out.append(code * scale)
        return out[0].reshape(-1), (out[1] * out[1]).reshape(-1)


def arena(tensors, like):
    """Values of tensors at the starts of whole blocks."""
    out = np.zeros(sum(-(-t.numel() // 256) for t in tensors) * 256, np.float32)
    at = 0
    for t in tensors:
        out[at:at + t.numel()] = t.detach().float().cpu().numpy().reshape(-1)
        at += -(-t.numel() // 256) * 256
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F4, BF, HF])
@pytest.mark.parametrize("clip", [None, 0.05])
def test_steps_with_8_bit_moments(dtype, clip):
    """Codes are those of the formula in fp32, each product and sum rounded."""
    from rocm_qlora.optim import AdamW
    params = made(SHAPES, dtype, seed=1)
    opt = AdamW(params, **NUMBERS, state_bits=8, max_grad_norm=clip)
    f = np.float32
    m, v = opt.moments()
    assert not bool(m.any()) and not bool(v.any())
    m, v = m.cpu().numpy(), v.cpu().numpy()
    for t in range(1, 5):
        before = [p.detach().clone() for p in params]
        g = arena([p.grad for p in params], m)
        c = f(1)
        if clip:
            norm = f(math.sqrt(np.square(g.astype(np.float64)).sum()))
            c = min(f(1), (f(1) / (norm + f(1e-6))) * f(clip))
        opt.step()
        if clip:
            assert abs(float(opt.grad_norm) - float(norm)) <= 2.0 ** -23 * float(norm)
        g = g * c
        rest1, rest2 = f(1 - 0.9), f(1 - 0.999)
        new_m, new_v = m * f(0.9) + g * rest1, v * f(0.999) + (g * g) * rest2
        at = 0
        for i, p in enumerate(params):
            part = slice(at, at + p.numel())
            old = [torch.from_numpy(x[part].copy()).cuda().view(p.shape) for x in (m, v)]
            want, _, _, _, step = formula(before[i], p.grad, *old, t, float(c))
            check_params(p, want, step)
            at += -(-p.numel() // 256) * 256
        m, v = kept8(new_m, new_v)
        got_m, got_v = (x.cpu().numpy() for x in opt.moments())
        assert np.array_equal(got_m, m) and np.array_equal(got_v, v)
        for p in params:
            p.grad.mul_(-1.5)


@pytest.mark.gpu
def test_set_moments_takes_values_and_keeps_what_is_not_zero():
    from rocm_qlora.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(1000, device="cuda"))
    opt = AdamW([p], state_bits=8)
    g = torch.Generator().manual_seed(2)
    m = torch.zeros(1024)
    m[:1000] = torch.randn(1000, generator=g) * 10.0 ** torch.randint(-12, 3, (1000,), generator=g)
    v = m.square()
    v[5], v[6] = 2.0 ** -149, 1e30
    opt.set_moments(m.cuda(), v.cuda(), 7)
    got = opt.moments()
    want = kept8(m.numpy(), v.numpy())
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(got, want))
    assert bool((got[1].cpu()[v > 0] > 0).all()) and int(opt.state[p]["step"]) == 7
    assert opt.state[p]["exp_avg"].dtype == torch.uint8


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_infinities_and_nans_stay_in_their_block(bits):
    from rocm_qlora.optim import AdamW
    p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
    p.grad = torch.full_like(p, 0.1)
    p.grad[300], p.grad[600], p.grad[1023] = float("nan"), float("inf"), 0.0
    opt = AdamW([p], state_bits=bits)
    for _ in range(2):
        opt.step()
    ok = torch.isfinite(p.detach())
    assert not bool(ok[300]) and not bool(ok[600])
    first = torch.ones(256, dtype=torch.bool, device="cuda")
    assert bool(ok[:256].all()) and bool(ok[768:].all()) and bool(first.all())
    m, v = opt.moments()
    assert bool(torch.isnan(m[256:512]).any()) and bool(torch.isfinite(m[768:]).all())
    assert float(v[1023]) == 0.0 and float(p.detach()[1023]) < 1.0   # decayed, not moved


@pytest.mark.gpu
def test_remainder_holds_a_32_bit_value():
    """Steps too small for bf16 add up; the parameter is the 32-bit value
    rounded, half away from zero."""
    from rocm_qlora.optim import AdamW
    g = torch.Generator().manual_seed(3)
    start = torch.randn(700, generator=g).to(BF).cuda()
    grad = (torch.randn(700, generator=g) * 1e-3).to(BF).cuda()
    p = torch.nn.Parameter(start.clone())
    p.grad = grad
    full = torch.nn.Parameter(start.float())
    full.grad = grad.float()
    numbers = dict(lr=1e-5, weight_decay=0.01)
    opt, ref = AdamW([p], remainder=True, **numbers), AdamW([full], **numbers)
    for _ in range(20):
        opt.step()
        ref.step()
    low = opt.state[p]["remainder"]
    bits = (p.detach().view(torch.int16).int() << 16) + low.int()
    assert torch.equal(bits.view(F4), full.detach())
    away = ((full.detach().view(torch.int32) + 0x8000) >> 16).to(torch.int16)
    assert torch.equal(p.detach().view(torch.int16), away) and bool((p.detach() != start).any())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_one_launch_takes(bits):
    """1300 tensors of mixed types, some without a gradient, unaligned views
    and strided gradients among them, as each one alone."""
    from rocm_qlora.optim import AdamW
    g = torch.Generator().manual_seed(4)
    params, alone = [], []
    for i in range(1300):
        dt = (F4, BF, HF)[i % 3]
        base = torch.randn(1 + (i * 37) % 600 + 3, generator=g).to(dt).cuda()
        t = base[i % 4:]                                              # starts anywhere
        p = torch.nn.Parameter(t)
        q = torch.nn.Parameter(t.clone())
        if i % 7:
            grad = (torch.randn(2, p.numel(), generator=g) * 0.1).to(dt).cuda()
            p.grad = grad.t()[:, 0] if i % 5 == 0 else grad[0]
            q.grad = grad[0].clone()
        params.append(p)
        alone.append(q)
    many = AdamW(params, **NUMBERS, state_bits=bits)
    ones = [AdamW([q], **NUMBERS, state_bits=bits) for q in alone]
    for _ in range(2):
        many.step()
        for o in ones:
            o.step()
    for i, (p, q) in enumerate(zip(params, alone)):
        assert torch.equal(p, q), i
        assert int(many.state[p]["step"]) == (2 if i % 7 else 0)
        assert torch.equal(many.state[p]["exp_avg"], ones[i].state[q]["exp_avg"])


@pytest.mark.gpu
def test_groups_closure_and_learning_rates_on_the_device():
    from rocm_qlora.optim import AdamW
    a, b = made([(300,), (40, 20)], F4, seed=5)
    before = [a.detach().clone(), b.detach().clone()]
    rate = torch.full((), 3e-2, device="cuda")
    opt = AdamW([dict(params=[a], lr=rate), dict(params=[b], weight_decay=0.0, betas=(0.0, 0.5), eps=1e-3)], **NUMBERS,
                max_grad_norm=1e-3)
    loss = opt.step(lambda: torch.full((), 2.5))
    assert float(loss) == 2.5
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in (a, b)))
    assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
    c = 1e-3 / (norm + 1e-6)
    for p, old, kw in ((a, before[0], dict(NUMBERS, lr=3e-2)),
                       (b, before[1], dict(lr=1e-2, weight_decay=0.0, betas=(0.0, 0.5), eps=1e-3))):
        want, _, _, _, step = formula(old, p.grad, torch.zeros_like(p), torch.zeros_like(p), 1, c, **kw)
        check_params(p, want, step)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_count_on(bits):
    from rocm_qlora.optim import AdamW
    params, same = made([(300,), (70, 9)], BF, seed=6), made([(300,), (70, 9)], BF, seed=6)
    rate = torch.full((), 1e-2, device="cuda")
    kw = dict(weight_decay=0.1, state_bits=bits, max_grad_norm=0.1, remainder=True)
    opt, eager = AdamW(params, lr=rate, **kw), AdamW(same, lr=1e-2, **kw)
    opt.step()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for t in range(3):
        if t == 2:
            rate.fill_(5e-3)
            eager.param_groups[0]["lr"] = float(torch.tensor(5e-3))
        for p, q in zip(params, same):
            p.grad.mul_(0.9)
            q.grad.mul_(0.9)
        graph.replay()
        eager.step()
    for p, q in zip(params, same):
        assert int(opt.state[p]["step"]) == 4
        # the rate on the device is the float32 nearest to 1e-2
        assert torch.equal(opt.state[p]["exp_avg"], eager.state[q]["exp_avg"])
        assert bool(((p - q).abs().float() <= 2.0 ** -7 * q.detach().abs().float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict_round_trip(bits, tmp_path):
    from rocm_qlora.optim import AdamW
    params, same = made([(300,), (70, 9)], BF, seed=7), made([(300,), (70, 9)], BF, seed=7)
    kw = dict(state_bits=bits, remainder=True)
    opt = AdamW(params, **NUMBERS, **kw)
    for _ in range(2):
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "state.pt")
    other = AdamW(same, lr=1.0, **kw)
    other.load_state_dict(torch.load(tmp_path / "state.pt"))
    for p, q in zip(params, same):
        q.data.copy_(p.data)
    opt.step()
    other.step()
    for p, q in zip(params, same):
        assert torch.equal(p, q) and other.state[q]["exp_avg"].dtype == opt.state[p]["exp_avg"].dtype
    with pytest.raises(ValueError):
        AdamW(same, state_bits=40 - bits, remainder=True).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        AdamW(same[:1], **kw).load_state_dict(opt.state_dict())


@pytest.mark.gpu
def test_other_stream_and_later_groups():
    from rocm_qlora.optim import AdamW
    a, b = made([(513,), (9, 9)], F4, seed=8)
    c, d = made([(513,), (9, 9)], F4, seed=8)
    one, two = AdamW([a], **NUMBERS), AdamW([c], **NUMBERS)
    one.add_param_group(dict(params=[b]))
    two.add_param_group(dict(params=[d]))
    side = torch.cuda.Stream()
    for _ in range(3):
        one.step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            two.step()
        torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F4, BF, HF])
def test_grad_norm(dtype):
    from rocm_qlora.optim import grad_norm
    g = torch.Generator().manual_seed(9)
    for shapes in ([(1,)], [(5, 7), (0,), (1000, 301)], [(i % 300 + 1,) for i in range(1100)]):
        ts = [(torch.randn(s, generator=g) * 3).to(dtype).cuda() for s in shapes]
        want = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
        assert abs(float(grad_norm(ts)) - want) <= 2.0 ** -23 * want
    t = torch.randn(64, 300, generator=g).to(dtype).cuda()
    want = math.sqrt(float(t.double().square().sum()))
    for view in (t.t(), t[:, 1:], t.view(-1)[3:]):
        want = math.sqrt(float(view.double().square().sum()))
        assert abs(float(grad_norm([view])) - want) <= 2.0 ** -23 * want
    big = torch.full((300,), torch.finfo(dtype).max, device="cuda", dtype=dtype)[:1 if dtype != HF else 300]
    assert abs(float(grad_norm([big])) / (float(big[0]) * math.sqrt(big.numel())) - 1) <= 2.0 ** -22
    small = torch.full((300,), 2.0 ** -100 if dtype != HF else 2.0 ** -24, device="cuda", dtype=dtype)
    assert abs(float(grad_norm([small])) / (float(small[0]) * math.sqrt(300)) - 1) <= 2.0 ** -22
    small[7] = float("nan")
    assert math.isnan(float(grad_norm([small]))) and float(grad_norm([t[:0]])) == 0.0


@pytest.mark.gpu
def test_refused_parameters():
    from rocm_qlora.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(8, 8, device="cuda"))
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.zeros(8, device="cuda", dtype=F8))])
    with pytest.raises(TypeError):
        AdamW([p], remainder=True)
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(8, 8, device="cuda").t()[:, :4])])
    opt = AdamW([p])
    p.grad = torch.zeros(8, 8, device="cuda")
    opt.param_groups[0]["betas"] = (1.0, 0.9)
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[0]["betas"] = (0.9, 0.9)
    opt.param_groups[0]["lr"] = torch.zeros(())
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-3
    p.data = torch.zeros(30, 30, device="cuda")
    p.grad = None
    p.grad = torch.zeros(30, 30, device="cuda")
    with pytest.raises(ValueError, match="size"):
        opt.step()


@pytest.mark.gpu
def test_a_refused_step_changes_nothing_and_clipping_may_come_later():
    from rocm_qlora.optim import AdamW
    a, b = made([(300,), (20, 20)], F4, seed=12)
    opt = AdamW([dict(params=[a]), dict(params=[b], lr=torch.zeros(()))], lr=1e-2, weight_decay=0)
    before = a.detach().clone()
    with pytest.raises(ValueError):
        opt.step()  # the second group's learning rate is on the CPU
    assert torch.equal(a.detach(), before) and int(opt.state[a]["step"]) == 0
    opt.param_groups[1]["lr"] = 1e-2
    opt.max_grad_norm = -1.0
    with pytest.raises(ValueError):
        opt.step()
    opt.max_grad_norm = 0.5
    opt.step()
    norm = math.sqrt(sum(float(p.grad.to(F8).square().sum()) for p in (a, b)))
    assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm and int(opt.state[a]["step"]) == 1


@pytest.mark.gpu
def test_hooks_schedulers_and_profiler_ranges():
    from rocm_qlora.optim import AdamW
    (p,) = made([(300,)], F4, seed=10)
    opt = AdamW([p], lr=1, weight_decay=0)
    called = []
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda t: 0.5 ** t)
    opt.step()
    schedule.step()
    assert opt.param_groups[0]["lr"] == 0.5
    before = opt.register_step_pre_hook(lambda *a: called.append("before"))
    after = opt.register_step_post_hook(lambda *a: called.append("after"))
    opt.step()
    before.remove(), after.remove()
    opt.step()
    assert called == ["before", "after"] and int(opt.state[p]["step"]) == 3
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as seen:
        opt.step()
    assert any(e.key.startswith("Optimizer.step#AdamW") for e in seen.key_averages())
    with pytest.raises(TypeError, match="state_dict"):
        import copy
        copy.deepcopy(opt)


@pytest.mark.gpu
def test_half_precision_with_a_gradient_scaler():
    """GradScaler skips a step whose gradients overflow and takes the others."""
    from rocm_qlora.optim import AdamW
    (p,) = made([(600,)], F4, seed=11)
    opt = AdamW([p], lr=1e-2, state_bits=8, max_grad_norm=1.0)
    scaler = torch.amp.GradScaler("cuda", init_scale=4.0)
    start = p.detach().clone()
    for scale, steps in ((float("inf"), 0), (4.0, 1)):
        scaler.scale(torch.zeros((), device="cuda", requires_grad=True))  # the scale's own lazy start
        p.grad = torch.ones_like(p) * scale
        scaler.step(opt)
        scaler.update()
        assert int(opt.state[p]["step"]) == steps and bool((p == start).all()) == (steps == 0)


# ------------------------------------------------------------- refused, CPU

def test_refused_numbers():
    from rocm_qlora.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(8))
    for kw in (dict(state_bits=16), dict(max_grad_norm=0.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
               dict(lr=-1.0), dict(lr=float("nan")), dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(ValueError):
        AdamW([])


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate")
def test_refused_parameters_that_share_memory():
    """One launch updates a group's tensors side by side."""
    from rocm_qlora.optim import AdamW
    p, whole = torch.nn.Parameter(torch.zeros(8)), torch.zeros(40)
    for params in ([p, p], [torch.nn.Parameter(whole[:21]), torch.nn.Parameter(whole[20:])]):
        with pytest.raises(ValueError, match="share memory"):
            AdamW(params)


def test_refused_devices():
    from rocm_qlora import _native as nat
    from rocm_qlora.optim import AdamW, grad_norm
    with pytest.raises(nat.NativeUnavailable):
        AdamW([torch.nn.Parameter(torch.zeros(8))])
    with pytest.raises(nat.NativeUnavailable):
        grad_norm([torch.zeros(8)])
    with pytest.raises(ValueError):
        grad_norm([])
    with pytest.raises(TypeError):
        grad_norm([torch.zeros(8, dtype=torch.int32)])


def test_meta_gives_shapes():
    from rocm_qlora import _native as nat
    assert nat.loaded_ops().grad_norm([torch.zeros(8, device="meta")]).shape == ()
    codes = torch.empty(512, dtype=torch.uint8, device="meta")
    m, v = nat.loaded_ops().adam_unpack(codes, codes, torch.empty(2, 2, device="meta"))
    assert m.shape == v.shape == (512,)
    with pytest.raises(RuntimeError):
        nat.loaded_ops().adam_unpack(codes, codes[:256], torch.empty(2, 2, device="meta"))
