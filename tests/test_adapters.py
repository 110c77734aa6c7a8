"""Adapters of many requests (rocm_qlora.lora.adapter_bank) against the
formula in 64 bits.

Bounds, per output, derived from how it is computed: the result is rounded
once to 16 bits (half an ulp, HALF of its magnitude, and half the smallest
subnormal), and everything before is fp32 accumulation.  A sum of n products
in fp32 errs by at most n * 2^-22 of the sum of their magnitudes (tensor
cores truncate, hence one bit more than rounding), and the low-rank
intermediate enters its second product with 16 bits, 2^-16 of its magnitude.
"""
import pytest
import torch

F8 = torch.float64
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def make(rows, k, n, rank, count, dtype, seed=0, none=0.15, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, count, (rows,), generator=g)
    ids[torch.rand(rows, generator=g) < none] = -1
    t = dict(base=torch.randn(rows, n, generator=g), x=torch.randn(rows, k, generator=g),
             A=torch.randn(count, k, rank, generator=g) / k ** 0.5, B=torch.randn(count, n, rank, generator=g) * 0.3,
             dy=torch.randn(rows, n, generator=g))
    t = {name: v.to(dtype).to(device) for name, v in t.items()}
    t["scaling"] = (0.5 + torch.rand(count, generator=g)).to(device)
    t["ids"] = ids.to(device)
    return t


def formula(t, z=None):
    """y, dx, dA, dB in 64 bits and the bound of each (z: what stands for x in dA)."""
    x, base, dy, dt = t["x"].to(F8), t["base"].to(F8), t["dy"].to(F8), t["x"].dtype
    z = x if z is None else z
    y, dx = base.clone(), torch.zeros_like(x)
    dA, dB = torch.zeros_like(t["A"], dtype=F8), torch.zeros_like(t["B"], dtype=F8)
    ey, ex, eA, eB = (torch.zeros_like(v) for v in (y, dx, dA, dB))
    k, n, r = x.shape[1], base.shape[1], t["A"].shape[2]
    acc = 2.0 ** -22
    for a in range(t["A"].shape[0]):
        at = (t["ids"] == a).nonzero()[:, 0]
        if not len(at):
            continue
        A, B, s = t["A"][a].to(F8), t["B"][a].to(F8), t["scaling"][a].to(F8)
        u, v = s * (x[at] @ A), s * (dy[at] @ B)
        mu, mv = s * (x[at].abs() @ A.abs()), s * (dy[at].abs() @ B.abs())
        eu, ev = (k + 4) * acc * mu, (n + 4) * acc * mv   # error of the intermediate as stored
        su, sv = eu + 2.0 ** -16 * u.abs(), ev + 2.0 ** -16 * v.abs()  # and as multiplied
        y[at] += u @ B.t()
        ey[at] = su @ B.abs().t() + (r + 4) * acc * (mu @ B.abs().t() + base[at].abs())
        dx[at] = v @ A.t()
        ex[at] = sv @ A.abs().t() + (r + 4) * acc * (mv @ A.abs().t())
        m = len(at) + 4
        dA[a] = z[at].t() @ v
        eA[a] = z[at].abs().t() @ sv + m * acc * (z[at].abs().t() @ mv)
        dB[a] = dy[at].t() @ u
        eB[a] = dy[at].abs().t() @ su + m * acc * (dy[at].abs().t() @ mu)
    # the rounding is of the value that carries the error
    return [(v, HALF[dt] * (v.abs() + e) + e + TINY[dt]) for v, e in ((y, ey), (dx, ex), (dA, eA), (dB, eB))]


def check(got, want, name):
    value, bound = want
    assert got.shape == value.shape
    off = (got.to(F8) - value).abs()
    assert bool((off <= bound).all()), f"{name}: {float((off - bound).max()):.3g} over its bound"


def run(t, packed_x=None, ids=None):
    from rocm_qlora.lora import AdapterPlan, adapters_add
    plan = AdapterPlan(t["ids"] if ids is None else ids, t["A"].shape[0])
    leaves = [t[n].detach().clone().requires_grad_() for n in ("base", "x", "A", "B")]
    y = adapters_add(*leaves, t["scaling"], plan, packed_x=packed_x)
    return y, torch.autograd.grad(y, leaves, t["dy"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n,rank,count", [
    (1, 64, 64, 8, 1), (1, 4096, 4096, 16, 8), (3, 1, 1, 8, 2), (5, 65, 127, 16, 3), (16, 256, 136, 24, 1),
    (17, 1088, 200, 32, 4), (33, 130, 4098, 64, 40), (64, 1024, 1000, 128, 5), (129, 333, 1024, 64, 2),
    (300, 520, 264, 16, 2), (300, 264, 520, 40, 64), (1025, 264, 72, 128, 3), (1500, 72, 264, 8, 1)])
def test_forward_and_gradients(rows, k, n, rank, count, dtype):
    t = make(rows, k, n, rank, count, dtype, seed=rows + k)
    y, grads = run(t)
    want = formula(t)
    assert torch.equal(grads[0], t["dy"])
    for got, w, name in zip((y, *grads[1:]), want, ("y", "dx", "dA", "dB")):
        check(got, w, f"{name} {rows}x{k}x{n} r{rank} of {count}")


@pytest.mark.gpu
def test_long_rows_of_large_layers():
    t = make(2050, 4096, 11008, 16, 2, torch.bfloat16)
    y, grads = run(t)
    for got, w, name in zip((y, *grads[1:]), formula(t), ("y", "dx", "dA", "dB")):
        check(got, w, name)


@pytest.mark.gpu
@pytest.mark.parametrize("spread", ["even", "half", "one", "two"])
@pytest.mark.parametrize("rows,k,n,rank,count,dtype", [
    (90, 2048, 4099, 16, 40, torch.bfloat16), (1500, 2048, 1027, 16, 40, torch.bfloat16),
    (1500, 2048, 1032, 32, 40, torch.float16), (1200, 2056, 1027, 64, 70, torch.bfloat16),
    (2500, 512, 264, 16, 300, torch.float16)])
def test_many_adapters(rows, k, n, rank, count, dtype, spread):
    """Banks of many adapters, their rows spread evenly or most of them on one or two."""
    from rocm_qlora.activation8 import pack_activation
    t = make(rows, k, n, rank, count, dtype, seed=rows)
    g = torch.Generator().manual_seed(1)
    some = torch.rand(rows, generator=g).to(t["ids"].device)
    if spread == "half":
        t["ids"][some < 0.5] = count - 1
    elif spread == "one":
        t["ids"][:] = count // 2
    elif spread == "two":
        t["ids"][:] = torch.where(some < 0.6, 0, count - 2)
    packed = pack_activation(t["x"])
    y, grads = run(t)
    for got, w, name in zip((y, *grads[1:]), formula(t), ("y", "dx", "dA", "dB")):
        check(got, w, f"{name} {spread}")
    again = run(t)[1]
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    codes = packed.codes[:, :k].to(F8) * packed.scales.to(F8).repeat_interleave(128, 1)[:, :k]
    check(run(t, packed_x=packed)[1][2], formula(t, z=codes)[2], f"dA of codes {spread}")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [7, 200])
def test_rows_without_an_adapter(rows):
    t = make(rows, 264, 136, 16, 3, torch.bfloat16, none=1.1)
    y, grads = run(t)
    assert torch.equal(y, t["base"])
    assert all(int(torch.count_nonzero(g)) == 0 for g in grads[1:])
    # a bank of which one adapter alone is used: the others' gradients are zero
    t["ids"][:] = 1
    _, grads = run(t)
    for g in grads[2:]:
        assert int(torch.count_nonzero(g[0])) == 0 and int(torch.count_nonzero(g[2])) == 0
        assert int(torch.count_nonzero(g[1])) > 0


@pytest.mark.gpu
def test_ids_that_name_no_adapter_give_nan():
    t = make(40, 136, 72, 16, 3, torch.bfloat16, none=0.0)
    good = run(t)
    ids = t["ids"].clone()
    ids[5], ids[11], ids[12] = 3, -2, 2 ** 40
    y, grads = run(t, ids=ids)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[5, 11, 12]] = True
    assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], good[0][~bad])
    assert bool(torch.isnan(grads[1][bad]).all()) and torch.equal(grads[1][~bad], good[1][1][~bad])
    assert bool(torch.isfinite(grads[2]).all()) and bool(torch.isfinite(grads[3]).all())


@pytest.mark.gpu
def test_strides_int32_ids_and_outputs():
    from rocm_qlora.lora import AdapterPlan, adapters_add
    t = make(50, 128, 96, 16, 4, torch.bfloat16)
    want = formula(t)[0]
    wide_x = torch.zeros(50, 301, dtype=torch.bfloat16, device="cuda")
    wide_b = torch.zeros(50, 240, dtype=torch.bfloat16, device="cuda")
    wide_x[:, 3:131], wide_b[:, 104:200] = t["x"], t["base"]
    plan = AdapterPlan(t["ids"].int(), 4)
    y = adapters_add(wide_b[:, 104:200], wide_x[:, 3:131], t["A"], t["B"], t["scaling"], plan)
    check(y, want, "strided")
    base = t["base"].clone()
    assert adapters_add(base, t["x"], t["A"], t["B"], t["scaling"], plan, out=base) is base
    assert torch.equal(base, y)
    three = adapters_add(t["base"].view(5, 10, 96), t["x"].view(5, 10, 128), t["A"], t["B"], t["scaling"], plan)
    assert three.shape == (5, 10, 96) and torch.equal(three.view(50, 96), y)
    cpu = AdapterPlan(t["ids"].cpu(), 4)
    assert torch.equal(adapters_add(t["base"], t["x"], t["A"], t["B"], t["scaling"], cpu), y)
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        other = adapters_add(t["base"], t["x"], t["A"], t["B"], t["scaling"], plan)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(other, y)


@pytest.mark.gpu
def test_transposed_gradient_and_broadcast_upstream():
    t = make(70, 136, 72, 16, 2, torch.float16)
    want = formula(t)
    from rocm_qlora.lora import AdapterPlan, adapters_add
    plan = AdapterPlan(t["ids"], 2)
    x, A, B = (t[n].clone().requires_grad_() for n in ("x", "A", "B"))
    y = adapters_add(t["base"], x, A, B, t["scaling"], plan)
    grads = torch.autograd.grad(y, (x, A, B), t["dy"].t().contiguous().t())
    for got, w, name in zip(grads, want[1:], ("dx", "dA", "dB")):
        check(got, w, name)
    y = adapters_add(t["base"], x, A, B, t["scaling"], plan)
    t["dy"] = torch.ones_like(t["dy"])
    grads = torch.autograd.grad(y.sum(), (x, A, B))
    for got, w, name in zip(grads, formula(t)[1:], ("dx", "dA", "dB")):
        check(got, w, name)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,count", [(24, 3), (260, 2)])
def test_gradients_against_differences(rows, count):
    """Along random directions: y is linear in each of x, A, B, so the central
    difference of <dy, y> in 64 bits is its derivative but for rounding."""
    t = make(rows, 72, 40, 16, count, torch.bfloat16)
    _, grads = run(t)
    want = dict(zip(("x", "A", "B"), formula(t)[1:]))
    g = torch.Generator(device="cuda").manual_seed(5)

    def f(**moved):
        s = {**t, **moved}
        total = 0.0
        for a in range(count):
            at = s["ids"] == a
            u = s["scaling"][a].to(F8) * (s["x"].to(F8)[at] @ s["A"][a].to(F8))
            total = total + (s["dy"].to(F8)[at] * (u @ s["B"][a].to(F8).t())).sum()
        return total

    for name, grad in zip(("x", "A", "B"), grads[1:]):
        way = torch.randn(t[name].shape, generator=g, device="cuda", dtype=F8)
        slope = (f(**{name: t[name].to(F8) + 0.5 * way}) - f(**{name: t[name].to(F8) - 0.5 * way}))
        bound = (want[name][1] * way.abs()).sum()
        assert abs(float((grad.to(F8) * way).sum() - slope)) <= float(bound) + 1e-9 * abs(float(slope)), name


@pytest.mark.gpu
def test_infinite_and_nan_rows_stay_in_their_rows():
    t = make(40, 136, 72, 16, 2, torch.bfloat16, none=0.0)
    clean = run(t)[0]
    t["x"][3, 7], t["x"][20, 0] = float("inf"), float("nan")
    y = run(t)[0]
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[3, 20]] = False
    assert torch.equal(y[keep], clean[keep])
    assert bool(torch.isnan(y[20]).all()) and not bool(torch.isfinite(y[3]).any())


@pytest.mark.gpu
def test_results_repeat_bit_for_bit():
    t = make(700, 264, 136, 64, 5, torch.bfloat16)
    y, grads = run(t)
    for _ in range(3):
        y2, g2 = run(t)
        assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, g2))


@pytest.mark.gpu
def test_empty_batch():
    t = make(0, 64, 32, 8, 2, torch.bfloat16)
    y, grads = run(t)
    assert y.shape == (0, 32) and all(int(torch.count_nonzero(g)) == 0 for g in grads[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,count", [(1, 1), (5, 3), (1000, 1), (1000, 7), (3000, 4096)])
def test_plan(rows, count):
    """The plan's rows are sorted by adapter, each adapter's in batch order."""
    from rocm_qlora.lora import AdapterPlan
    ids = torch.randint(-1, count, (rows,), generator=torch.Generator().manual_seed(rows))
    plan = AdapterPlan(ids, count)
    data = plan.data.cpu()
    key = torch.where(ids < 0, count, ids)
    order = torch.sort(key, stable=True).indices
    assert torch.equal(data[-rows:].long(), order)
    sizes = torch.bincount(key, minlength=count + 2)
    first = torch.cat([torch.zeros(1, dtype=torch.long), sizes.cumsum(0)])
    assert torch.equal(data[1:count + 4].long(), first)
    tiles = (sizes + plan.tile - 1) // plan.tile
    assert int(data[0]) == int(tiles.sum())
    at = (count + 4 + 3) // 4 * 4
    table = data[at:at + 4 * int(data[0])].view(-1, 4)
    assert torch.equal(torch.bincount(table[:, 0].long(), minlength=count + 2), tiles)
    assert torch.equal(torch.zeros(count + 2, dtype=torch.long).index_add(0, table[:, 0].long(), table[:, 2].long()),
                       sizes)
    assert int(table[:, 2].max()) <= plan.tile and int(table[:, 2].min()) >= 1


@pytest.mark.gpu
def test_bank_layer_and_lora_layer():
    """MultiLoRALinear gives the single layers' outputs and gradients up to
    their 16-bit roundings: at most three more per output than the bank's one."""
    import torch.nn as nn
    from rocm_qlora import LoRALinear, QuantLinear
    from rocm_qlora.activation8 import pack_activation
    from rocm_qlora.lora import AdapterBank, AdapterPlan, MultiLoRALinear
    torch.manual_seed(0)
    k, n, rows, dt = 256, 192, 90, torch.bfloat16
    ql = QuantLinear.from_linear(nn.Linear(k, n, bias=True, device="cuda", dtype=dt), bits=4)
    singles = []
    for r in (4, 12):
        lora = LoRALinear(ql, r=r, lora_alpha=16).cuda()
        nn.init.normal_(lora.lora_B, std=0.05)
        singles.append(lora)
    bank = AdapterBank.from_lora_layers(singles, dt)
    assert bank.lora_A.shape == (2, k, 16) and bank.rank == 12
    layer = MultiLoRALinear(ql, bank)
    x = torch.randn(rows, k, device="cuda", dtype=dt, requires_grad=True)
    ids = torch.arange(rows) % 3 - 1
    plan = AdapterPlan(ids, 2)
    y = layer(x, plan)
    dy = torch.randn_like(y)
    dx, dA, dB = torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), dy)
    with torch.no_grad():
        assert torch.equal(layer(x, plan), y)
        assert torch.equal(y[ids.cuda() == -1], ql(x)[ids.cuda() == -1])
    for a, lora in enumerate(singles):
        at = ids.cuda() == a
        xa = x[at].detach().requires_grad_()
        ya = lora(xa)
        ga = torch.autograd.grad(ya, (xa, lora.lora_A, lora.lora_B), dy[at])
        for got, want in ((y[at], ya), (dx[at], ga[0]), (dA[a, :, :lora.r].t(), ga[1]), (dB[a, :, :lora.r], ga[2])):
            top = want.float().abs().max()
            assert float((got.float() - want.float()).abs().max()) <= 4 * 2.0 ** -8 * float(top)
        assert int(torch.count_nonzero(dA[a, :, lora.r:])) == 0 and int(torch.count_nonzero(dB[a, :, lora.r:])) == 0
    # the single layer with its input packed: the same up to the packing (half a step of a block's
    # largest value, 1/254, on the values of dA's sums)
    lora = singles[1]
    for packed in (None, pack_activation(x.detach())):
        y = lora(x, packed_x=packed) if packed is not None else lora(x)
        g = torch.autograd.grad(y, (x, lora.lora_A, lora.lora_B), dy)
        if packed is None:
            first = (y, *g)
    step = x.detach().float().abs().amax() / 254
    slack = (dy.float() @ lora.lora_B.float()).abs().sum(0).max() * lora.scaling * step
    for i, (got, want) in enumerate(zip((y, *g), first)):
        top = float(want.float().abs().max())
        more = float(slack) if i == 2 else 0.0
        assert got.dtype == want.dtype
        assert float((got.float() - want.float()).abs().max()) <= 4 * 2.0 ** -8 * top + more


# ------------------------------------------------------------- refusals (CPU)

def test_refusals():
    from rocm_qlora import _native as nat
    from rocm_qlora.lora import AdapterBank, AdapterPlan, adapters_add
    t = make(4, 16, 24, 8, 2, torch.bfloat16, device="cpu")
    args = [t[n] for n in ("base", "x", "A", "B", "scaling")]
    with pytest.raises(ValueError, match="needs a plan"):
        adapters_add(*args)
    with pytest.raises(ValueError, match="between -1 and 1"):
        AdapterPlan(torch.tensor([0, 2]), 2)
    with pytest.raises(ValueError, match="1-D int64 or int32"):
        AdapterPlan(torch.zeros(3), 2)
    with pytest.raises(ValueError, match="count"):
        AdapterPlan(torch.zeros(3, dtype=torch.long), 0)
    one = [args[0], args[1], args[2][:1], args[3][:1], args[4][:1]]
    with pytest.raises(nat.NativeUnavailable):
        adapters_add(*one)
    for i, bad, error in ((1, args[1].float(), TypeError), (0, args[0].half(), TypeError),
                          (2, args[2][:1, :, :6], ValueError), (2, args[2][:1].half(), TypeError),
                          (4, args[4][:1].double(), ValueError), (0, args[0][:, :9], ValueError),
                          (1, args[1][:3], ValueError)):
        with pytest.raises(error):
            adapters_add(*[bad if j == i else v for j, v in enumerate(one)])
    with pytest.raises(ValueError, match="rank"):
        AdapterBank(8, 8, 1, 129)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        AdapterBank(8, 8, 1, 8, torch.float32)
    bank = AdapterBank(16, 24, 2, 5)
    assert bank.lora_A.shape == (2, 16, 8) and bank.lora_B.shape == (2, 24, 8)
    with pytest.raises(IndexError):
        bank.set_adapter(2, torch.zeros(5, 16), torch.zeros(24, 5), 1.0)
    with pytest.raises(ValueError, match="do not fit"):
        bank.set_adapter(0, torch.zeros(6, 16), torch.zeros(24, 6), 1.0)
    bank.set_adapter(1, torch.ones(3, 16), torch.ones(24, 3), 2.0)
    assert int(torch.count_nonzero(bank.lora_A)) == 48 and float(bank.scaling[1]) == 2.0


@pytest.mark.gpu
def test_c_entry_refuses_bad_arguments():
    """Every refusal comes from the host checks, before a launch."""
    from rocm_qlora import _native as nat
    L = nat.lib()
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    u = torch.zeros(1, 64, 16, dtype=torch.bfloat16, device="cuda")
    s, mid = torch.ones(1, device="cuda"), torch.zeros(4, 16, device="cuda")
    plan = torch.zeros(4096, dtype=torch.int32, device="cuda")

    def apply(**k):
        a = dict(x=x.data_ptr(), ldx=64, u=u.data_ptr(), v=u.data_ptr(), s=s.data_ptr(), base=None, ldb=0, m=4, d1=64,
                 d2=64, r=16, count=1, dt=nat.BF16, plan=None, words=0, tile=16, mid=mid.data_ptr(), out=x.data_ptr(),
                 ldo=64)
        a.update(k)
        return L.rq_adapters_apply(*a.values(), nat.stream_ptr(x.device))

    assert apply(r=12) == -1 and apply(r=136) == -1 and apply(count=0) == -1 and apply(ldx=63) == -1
    assert apply(dt=nat.F32) == -3 and apply(u=u.data_ptr() + 2) == -2 and apply(x=x.data_ptr() + 1) == -2
    assert apply(plan=plan.data_ptr(), words=5) == -5 and apply(plan=plan.data_ptr(), words=4096, tile=17) == -1
    assert apply(s=None) == -1 and apply(out=None) == -1 and apply(m=-1) == -1
    assert L.rq_adapter_plan_words(10, 0, 16) == -1 and L.rq_adapter_plan_words(10, 2, 20) == -1
    assert L.rq_adapter_plan(None, 1, 4, 2, 16, plan.data_ptr(), 4096, None) == -1
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_row_offsets_past_32_bits():
    """Rows of x, base and dy that lie over 2^31 elements apart."""
    from rocm_qlora.lora import AdapterPlan, adapters_add
    t = make(18, 136, 72, 16, 2, torch.bfloat16)
    wide = torch.empty(18 << 27, dtype=torch.bfloat16, device="cuda")
    far = {n: wide[at:].as_strided((18, t[n].shape[1]), (1 << 27, 1)) for n, at in (("x", 0), ("base", 256), ("dy", 512))}
    for n, v in far.items():
        v.copy_(t[n])
    plan = AdapterPlan(t["ids"], 2)
    out = []
    for src in (t, far):
        x, A, B = src["x"].detach().requires_grad_(), t["A"].clone().requires_grad_(), t["B"].clone().requires_grad_()
        y = adapters_add(src["base"], x, A, B, t["scaling"], plan)
        out.append((y, *torch.autograd.grad(y, (x, A, B), src["dy"])))
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.gpu
def test_graph_replay_follows_its_inputs():
    from rocm_qlora.lora import AdapterPlan, adapters_add
    t = make(40, 264, 136, 16, 3, torch.bfloat16)
    ids, x = t["ids"].clone(), t["x"].clone()
    call = lambda: adapters_add(t["base"], x, t["A"], t["B"], t["scaling"], AdapterPlan(ids, 3))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for seed in (1, 2):
        other = make(40, 264, 136, 16, 3, torch.bfloat16, seed=seed)
        ids.copy_(other["ids"])
        x.copy_(other["x"])
        graph.replay()
        assert torch.equal(y, call())


@pytest.mark.gpu
def test_small_float16_gradients_keep_their_precision():
    """fp16 with gradients near 1e-6, as without loss scaling: the intermediate
    is brought into fp16's range by a power of two, so A's gradient errs by
    its own rounding (subnormal here) and no more."""
    t = make(200, 264, 136, 16, 2, torch.float16)
    t["dy"] = (t["dy"].float() * 1e-3).half()
    t["x"] = (t["x"].float() * 30.0).half()
    t["B"] = (t["B"].float() * 1e-2).half()
    y, grads = run(t)
    for got, w, name in zip((y, *grads[1:]), formula(t), ("y", "dx", "dA", "dB")):
        check(got, w, name)


@pytest.mark.gpu
def test_create_graph_is_refused():
    from rocm_qlora.lora import AdapterPlan, adapters_add
    t = make(8, 64, 32, 8, 1, torch.bfloat16)
    x = t["x"].requires_grad_()
    y = adapters_add(t["base"], x, t["A"], t["B"], t["scaling"], AdapterPlan(t["ids"], 1))
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y, x, t["dy"], create_graph=True)


@pytest.mark.gpu
def test_empty_dimensions():
    from rocm_qlora.activation8 import pack_activation, swiglu8, unpack_activation
    for shape in ((0, 5), (3, 0), (2, 0, 7), (2, 3, 0)):
        x = torch.zeros(shape, device="cuda", dtype=torch.bfloat16)
        assert unpack_activation(pack_activation(x)).shape == shape and swiglu8(x, x).shape == shape
