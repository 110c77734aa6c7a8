"""Microscaled 4-bit values (rocm_qlora.mx4): the form bit for bit against its
definition, products and the input gradient against the formula in 64 bits,
and what is refused."""
import math

import pytest
import torch

F8 = torch.float64
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=F8)
BF, HF = torch.bfloat16, torch.float16


def definition(x):
    """(codes [rows, Kp], scale bytes [rows, Kp / 32]) of rows on the CPU, in 64 bits."""
    m, k = x.shape
    v = torch.zeros(m, -(-k // 128) * 128, dtype=F8)
    v[:, :k] = x.to(F8)
    v = v.view(m, -1, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    e = torch.frexp(torch.where(bad, 1.0, top)).exponent - 1 - 2   # floor(log2 top) - 2
    e = torch.where(top == 0, -127, e).clamp(min=-127)
    a = torch.ldexp(v, -e[..., None]).abs()
    code = torch.zeros(v.shape, dtype=torch.long)
    for i, between in enumerate((LEVELS[1:] + LEVELS[:-1]) / 2):
        code += (a > between) | ((a == between) & (i % 2 == 1))     # a tie goes to the even code
    code += 8 * torch.signbit(v).long()
    return code.view(m, -1), torch.where(bad, 255, e + 127)


def values(codes, scales, k):
    """What codes and scale bytes stand for, in 64 bits."""
    v = LEVELS[codes & 7] * torch.where(codes >= 8, -1.0, 1.0)
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.to(F8) - 127))
    return (v.view(v.shape[0], -1, 32) * s[..., None]).view(v.shape)[:, :k]


def kept(x):
    return values(*definition(x.detach().cpu().reshape(-1, x.shape[-1])), x.shape[-1]).to(x.device)


def check_form(x, p):
    codes, scales = definition(x.cpu())
    got = p.codes.cpu().long()
    got = torch.stack([got & 15, got >> 4], -1).view(got.shape[0], -1)
    live = (scales != 255).repeat_interleave(32, 1)
    assert torch.equal(got[live], codes[live])
    assert torch.equal(p.scale_rows().cpu().long(), scales)


# a block's largest value on every edge of the rule: powers of two, just below,
# saturating, and ties between levels
def edges(dtype):
    x = torch.zeros(24, 64, dtype=F8)
    for r in range(12):
        x[r, 0] = 2.0 ** (r - 6)
        x[12 + r, 0] = 2.0 ** (r - 6) * 1.75
        between = torch.cat([LEVELS, (LEVELS[1:] + LEVELS[:-1]) / 2])
        x[r, 1:16] = between * 2.0 ** (r - 8)
        x[r, 16:31] = -between * 2.0 ** (r - 8)
        x[12 + r, 32:47] = between * 2.0 ** (r - 8)
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 31), (5, 32), (2, 33), (127, 128), (129, 200), (40, 1093), (300, 136)])
def test_pack_is_the_definition(rows, k, dtype):
    from rocm_qlora.mx4 import pack_mx4, unpack_mx4
    g = torch.Generator().manual_seed(rows * k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    p = pack_mx4(x.cuda())
    check_form(x, p)
    out = unpack_mx4(p)
    assert out.dtype == dtype and torch.equal(out.cpu(), kept(x).to(dtype))
    assert torch.equal(unpack_mx4(p, torch.float32).cpu(), kept(x).float())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
def test_pack_edges(dtype):
    from rocm_qlora.mx4 import pack_mx4, unpack_mx4
    x = edges(dtype)
    p = pack_mx4(x.cuda())
    check_form(x, p)
    assert torch.equal(unpack_mx4(p).cpu(), kept(x).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
def test_pack_zeros_tiny_huge_infinite_and_nan_blocks(dtype):
    from rocm_qlora.mx4 import pack_mx4, unpack_mx4
    x = torch.ones(6, 160, dtype=dtype)
    x[0, :32] = 0
    x[0, 32:64] = -0.0
    x[1, :] = torch.finfo(dtype).smallest_normal
    x[1, 64] = torch.finfo(dtype).smallest_normal / 2
    x[2, :] = torch.finfo(dtype).max
    x[2, 40:50] = torch.finfo(dtype).min
    x[3, 70] = float("inf")
    x[4, 159] = float("nan")
    x[5, 0] = float("-inf")
    p = pack_mx4(x.cuda())
    check_form(x, p)
    out = unpack_mx4(p, torch.float32).cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(kept(x)))
    fine = ~torch.isnan(out)
    assert torch.equal(out[fine], kept(x).float()[fine])


@pytest.mark.gpu
def test_pack_strides_and_shapes():
    from rocm_qlora.mx4 import pack_mx4, unpack_mx4
    x = torch.randn(6, 700, device="cuda", dtype=BF)
    for part in (x[:, 8:400], x[:, 3:402], x[::2], x.view(2, 3, 700), x.t(), x[:1].expand(5, 700), x[0]):
        p, want = pack_mx4(part), pack_mx4(part.contiguous())
        assert torch.equal(p.codes, want.codes) and torch.equal(p.scales, want.scales)
        assert unpack_mx4(p).shape == part.shape
    empty = pack_mx4(x[:0])
    assert unpack_mx4(empty).shape == (0, 700)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("first", [0, 4, 8, 16])
@pytest.mark.parametrize("rows,widths", [(131, (16, 144, 400, 1040, 1048)), (999, (1040, 1048, 2064))])
def test_pack_rows_at_every_alignment(rows, widths, first, dtype):
    """Rows that lie at multiples of 32, 16 and 8 bytes, in widths of whole and of part pieces."""
    from rocm_qlora.mx4 import pack_mx4, unpack_mx4
    g = torch.Generator().manual_seed(first)
    x = torch.randn(rows, 2080, generator=g).to(dtype)
    for k in widths:
        part = x.cuda()[:, first:first + k]
        p = pack_mx4(part)
        check_form(x[:, first:first + k], p)
        assert torch.equal(unpack_mx4(p).cpu(), kept(x[:, first:first + k]).to(dtype))


def close(got, want, slack):
    """One rounding to the type, and `slack` before it."""
    dt = got.dtype
    bound = HALF[dt] * (want.abs() + slack) + slack + TINY[dt]
    off = (got.to(F8) - want).abs()
    assert got.shape == want.shape and bool((off <= bound).all()), float((off / bound).max())


def sums(a, b, k):
    """What summing k products in 32 bits can be off by: at most 2^-23 of the
    magnitudes at each of the k / 64 steps, and for each term of a step."""
    return (k / 64 + 64) * 2.0 ** -23 * (a.abs() @ b.abs().t())


SIZES = [(1, 1, 1), (1, 128, 16), (1, 4096, 130), (3, 33, 257), (16, 1024, 384), (5, 12801, 40), (9, 12800, 20000),
         (16, 2500, 1000), (17, 500, 128), (33, 300, 100),
         (64, 2048, 1088), (100, 128, 64), (128, 640, 129), (129, 1093, 70), (200, 256, 512), (256, 1280, 96),
         (257, 200, 300), (300, 1093, 1089), (513, 1024, 640), (1000, 64, 255),
         (2500, 300, 1000), (1300, 640, 2049), (6000, 1093, 2600)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_product_and_its_gradient(rows, k, n, dtype):
    from rocm_qlora.mx4 import mx4_linear, mx4_matmul, pack_mx4
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w, dy = normal(rows, k).to(dtype), (normal(n, k) * 0.05).to(dtype), (normal(rows, n) * 0.1).to(dtype)
    bias = normal(n).to(dtype)
    packed = pack_mx4(w)
    xk, wk = kept(x), kept(w)
    want, slack = xk @ wk.t(), sums(xk, wk, k)
    y = mx4_matmul(pack_mx4(x), packed, dtype=dtype)
    close(y, want, slack)
    close(mx4_matmul(pack_mx4(x), packed, bias, dtype), want + bias.to(F8), slack + 2.0 ** -24 * (want.abs() + bias.abs().to(F8)))
    x.requires_grad_()
    out = mx4_linear(x, packed)
    assert torch.equal(out, y)
    dx, = torch.autograd.grad(out, x, dy)
    close(dx, dy.to(F8) @ wk, sums(dy.to(F8), wk.t(), n))
    with torch.no_grad():
        assert torch.equal(mx4_linear(x, packed), y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,k,n", [(4096, 4096, 4096), (2047, 11008, 4096), (300, 4096, 11008), (4096, 1024, 8200)])
def test_long_runs_of_tiles_and_stages(rows, k, n, dtype):
    """Many tiles a CTA and many rounds of its rings, several times over: every
    call gives the same values, near the product in 32 bits (whose own sums are
    off by less than 2^-20 of the terms' root sum of squares)."""
    from rocm_qlora import _native as nat
    from rocm_qlora.mx4 import mx4_matmul, pack_mx4, unpack_mx4
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    w = pack_mx4((torch.randn(n, k, generator=g, device="cuda") * 0.02).to(dtype))
    x = pack_mx4(torch.randn(rows, k, generator=g, device="cuda").to(dtype))
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    wide = unpack_mx4(w, torch.float32)
    for f, a, b in ((lambda: mx4_matmul(x, w, dtype=dtype), unpack_mx4(x, torch.float32), wide.t()),
                    (lambda: nat.loaded_ops().mx4_dx(dy, w.codes, w.scales, k), dy.float(), wide)):
        want = a @ b
        bound = HALF[dtype] * want.abs() + 2.0 ** -16 * (a.square() @ b.square()).sqrt() + TINY[dtype]
        first = f()
        assert bool(((first.float() - want).abs() <= bound).all())
        for _ in range(6):
            assert torch.equal(f(), first)


@pytest.mark.gpu
def test_gradient_against_differences():
    """On inputs that the 4-bit form holds exactly the product is linear in x."""
    from rocm_qlora.mx4 import mx4_linear, pack_mx4
    g = torch.Generator(device="cuda").manual_seed(5)
    x = LEVELS.cuda()[torch.randint(0, 6, (4, 64), generator=g, device="cuda")].to(HF)
    x[:, ::32] = 6.0                                                   # every block has the scale 1
    packed = pack_mx4(torch.randn(24, 64, generator=g, device="cuda", dtype=HF))
    x.requires_grad_()
    grad, = torch.autograd.grad(mx4_linear(x, packed).float().sum(), x)
    y = mx4_linear(x.detach(), packed).double()
    for i, j in ((0, 1), (1, 40), (3, 63)):
        moved = x.detach().clone()
        moved[i, j] = 4.0 if moved[i, j] != 4.0 else 0.0
        step = float(moved[i, j] - x[i, j])
        slope = float((mx4_linear(moved, packed).double() - y).sum()) / step
        # 24 outputs rounded to fp16 twice, the gradient once
        assert abs(slope - float(grad[i, j])) <= 2 * 2.0 ** -11 * float(y[i].abs().sum() + 24) / abs(step) + 2.0 ** -10 * abs(slope)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,scale", [(HF, 2.0 ** -30), (HF, 2.0 ** -12), (HF, 2.0 ** 12), (BF, 2.0 ** -118),
                                         (BF, 2.0 ** -30), (BF, 2.0 ** 12), (BF, 2.0 ** 120)])
def test_gradient_of_small_and_large_weights(dtype, scale):
    from rocm_qlora.mx4 import mx4_linear, pack_mx4
    g = torch.Generator(device="cuda").manual_seed(6)
    w = torch.randn(96, 128, generator=g, device="cuda") * scale   # in fp16 2^-30 is below what the type holds
    w[:, 32:64] *= 2.0 ** -4
    packed = pack_mx4(w)
    x = torch.zeros(40, 128, device="cuda", dtype=dtype, requires_grad=True)
    dy = (torch.randn(40, 96, generator=g, device="cuda") * min(1.0, 0.1 / scale)).to(dtype)
    dx, = torch.autograd.grad(mx4_linear(x, packed), x, dy)
    wk = kept(w)
    close(dx, dy.to(F8) @ wk, sums(dy.to(F8), wk.t(), 96))


@pytest.mark.gpu
def test_linear_strides_shapes_and_empties():
    from rocm_qlora.mx4 import mx4_linear, pack_mx4
    w = torch.randn(72, 192, device="cuda", dtype=BF)
    packed = pack_mx4(w)
    x = torch.randn(2, 5, 200, device="cuda", dtype=BF)
    for part in (x[..., :192], x[..., 3:195], x[0, :, 8:], x[:, ::2, :192], x[0, 0, :192]):
        y = mx4_linear(part, packed)
        assert y.shape == (*part.shape[:-1], 72) and torch.equal(y, mx4_linear(part.contiguous(), packed))
    e = x[..., :192].detach().requires_grad_()
    y = mx4_linear(e, packed)
    a, = torch.autograd.grad(y, e, torch.ones_like(y), retain_graph=True)
    b, = torch.autograd.grad(y.sum(), e)                              # a gradient of stride 0
    assert a.shape == e.shape and torch.equal(a, b)
    empty = x[:0, :, :192].requires_grad_()
    y = mx4_linear(empty, packed)
    assert y.shape == (0, 5, 72) and torch.autograd.grad(y.sum(), empty)[0].shape == empty.shape
    none = pack_mx4(w[:0])
    y = mx4_linear(e, none)
    assert y.shape == (2, 5, 0) and not bool(torch.autograd.grad(y.sum(), e)[0].any())


@pytest.mark.gpu
def test_a_row_of_nan_or_infinity_stays_in_its_row():
    from rocm_qlora.mx4 import mx4_linear, pack_mx4
    packed = pack_mx4(torch.randn(130, 300, device="cuda", dtype=BF))
    x = torch.randn(20, 300, device="cuda", dtype=BF)
    want = mx4_linear(x, packed)
    bad = x.clone()
    bad[3, 299], bad[7, 0] = float("nan"), float("inf")
    got = mx4_linear(bad, packed)
    keep = torch.ones(20, dtype=torch.bool, device="cuda")
    keep[[3, 7]] = False
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[~keep]).all())


@pytest.mark.gpu
def test_other_streams_and_graphs():
    from rocm_qlora.mx4 import mx4_linear, pack_mx4
    packed = pack_mx4(torch.randn(256, 512, device="cuda", dtype=BF))
    xs = [torch.randn(24, 512, device="cuda", dtype=BF) for _ in range(2)]
    want = [mx4_linear(x, packed) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mx4_linear(x, packed) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    hold = xs[0].clone().requires_grad_()
    dy = torch.randn(24, 256, device="cuda", dtype=BF)
    graphs, outs = [], []
    for _ in range(2):                                                # two graphs replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mx4_linear(hold, packed)
            dx, = torch.autograd.grad(y, hold, dy)
        graphs.append(graph)
        outs.append((y, dx))
    dx = torch.autograd.grad(mx4_linear(hold, packed), hold, dy)[0]
    for x, w in zip(xs, want):
        hold.data.copy_(x)
        for graph, (y, d) in zip(graphs, outs):
            graph.replay()
            assert torch.equal(y, w) and torch.equal(d, dx)


@pytest.mark.gpu
def test_module():
    from rocm_qlora.mx4 import Mx4Linear, mx4_linear
    torch.manual_seed(0)
    linear = torch.nn.Linear(200, 96, dtype=BF, device="cuda")
    m = Mx4Linear.from_linear(linear)
    x = torch.randn(3, 4, 200, device="cuda", dtype=BF)
    y = m(x)
    assert y.shape == (3, 4, 96) and torch.equal(y, mx4_linear(x, m.weight, linear.bias.detach()))
    assert torch.equal(m.dequantized(), kept(linear.weight).to(BF)) and not list(m.parameters())
    other = Mx4Linear(200, 96, bias=True, device="cuda")
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), y)
    assert m(x.half()).dtype == HF


# ------------------------------------------------------------- refused, CPU

def operators():
    from rocm_qlora import _native as nat
    return nat.loaded_ops()


def meta(rows=4, k=160, device="meta"):
    pitch = -(-k // 128) * 128
    e = lambda *s, dtype=torch.uint8: torch.empty(*s, device=device, dtype=dtype)  # noqa: E731
    return e(rows, pitch // 2), e(-(-rows // 128), pitch // 128, 512)


def test_meta_gives_shapes():
    x = torch.empty(2, 3, 160, device="meta", dtype=BF, requires_grad=True)
    y = operators().mx4_linear(x, *meta(72), 160, None)
    assert y.shape == (2, 3, 72) and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    codes, scales = operators().pack_mx4(x)
    assert codes.shape == (6, 128) and scales.shape == (1, 2, 512)


def test_refused_types_and_sizes():
    ops = operators()
    x = torch.empty(4, 160, device="meta", dtype=BF)
    with pytest.raises(TypeError):
        ops.pack_mx4(x.double())
    with pytest.raises(ValueError):
        ops.pack_mx4(x[:, :0])
    with pytest.raises(TypeError):
        ops.mx4_linear(x.float(), *meta(72), 160, None)
    with pytest.raises(ValueError):
        ops.mx4_linear(x[:, :150], *meta(72), 160, None)
    with pytest.raises(ValueError):
        ops.mx4_linear(x, *meta(72, 300), 160, None)
    with pytest.raises(ValueError):
        ops.mx4_linear(x, *meta(72), 160, torch.empty(71, device="meta", dtype=BF))
    with pytest.raises(TypeError):
        ops.mx4_linear(x, *meta(72), 160, torch.empty(72, device="meta"))
    with pytest.raises(ValueError, match="gradient"):
        ops.mx4_linear(x, *meta(72), 160, torch.empty(72, device="meta", dtype=BF, requires_grad=True))
    codes, scales = meta(72)
    with pytest.raises(TypeError):
        ops.mx4_matmul(codes, scales, codes, scales, 160, None, torch.float32)
    with pytest.raises(ValueError):
        ops.mx4_matmul(codes, scales, codes, scales, 500, None, BF)
    with pytest.raises(ValueError):
        ops.mx4_matmul(codes, scales[:, :1], codes, scales, 160, None, BF)


def test_refused_devices():
    from rocm_qlora import _native as nat
    from rocm_qlora.mx4 import Mx4Linear, mx4_linear, mx4_matmul, pack_mx4, PackedMx4, unpack_mx4
    with pytest.raises(nat.NativeUnavailable):
        pack_mx4(torch.randn(4, 64))
    cpu = PackedMx4(*meta(4, 64, "cpu"), (4, 64), BF)
    with pytest.raises(nat.NativeUnavailable):
        unpack_mx4(cpu)
    with pytest.raises(nat.NativeUnavailable):
        mx4_linear(torch.randn(2, 64, dtype=BF), cpu)
    with pytest.raises(nat.NativeUnavailable):
        Mx4Linear(64, 4)(torch.randn(2, 64, dtype=BF))
    with pytest.raises(Exception, match="device"):
        mx4_linear(torch.empty(2, 64, dtype=BF, device="meta"), cpu)
    with pytest.raises(ValueError):
        mx4_matmul(cpu, PackedMx4(*meta(4, 96, "cpu"), (4, 96), BF))


def test_refused_at_the_c_boundary():
    from rocm_qlora import _native as nat
    L = nat.load_library()
    assert L.rq_mx4_scale_bytes(130, 129) == 2 * 2 * 512 and L.rq_mx4_scale_bytes(-1, 5) == -1
    assert L.rq_mx4_linear_workspace_bytes(3, 5, 100) == 0                # packed on the way
    assert L.rq_mx4_linear_workspace_bytes(30, 5, 100) == 30 * 64 + 128 + 512


def test_differentiable_once_and_no_forward_derivatives():
    x = torch.empty(4, 160, device="meta", dtype=BF, requires_grad=True)
    y = operators().mx4_linear(x, *meta(72), 160, None)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(Exception):
        operators().mx4_linear(fw.make_dual(x.detach(), torch.empty_like(x)), *meta(72), 160, None)


def traced(device, grad):
    from rocm_qlora.mx4 import mx4_linear, mx4_matmul, pack_mx4, unpack_mx4
    x = torch.empty(2, 3, 200, device=device, dtype=BF, requires_grad=grad)
    packed = pack_mx4(torch.empty(72, 200, device=device, dtype=BF))
    y = mx4_linear(x, packed)
    found = [(y, (2, 3, 72), BF), (mx4_matmul(pack_mx4(x), packed, dtype=HF), (2, 3, 72), HF),
             (unpack_mx4(packed), (72, 200), BF), (packed.codes, (72, 128), torch.uint8)]
    if grad:
        found.append((torch.autograd.grad(y.float().sum(), x)[0], (2, 3, 200), BF))
    return found


# without a GPU autograd itself has no streams for fake CUDA tensors
@pytest.mark.parametrize("grad,device", [(False, "cuda"), (True, "meta"),
                                         pytest.param(True, "cuda", marks=pytest.mark.gpu)])
def test_fake_tensors(grad, device):
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=False):
        for value, shape, dtype in traced(device, grad):
            assert isinstance(value, FakeTensor) and value.shape == tuple(shape) and value.dtype == dtype
            assert value.device.type == device


@pytest.mark.gpu
def test_traced_graph_runs():
    from torch.fx.experimental.proxy_tensor import make_fx
    from rocm_qlora.mx4 import mx4_linear, pack_mx4, unpack_mx4
    packed = pack_mx4(torch.randn(72, 200, device="cuda", dtype=BF))
    f = lambda x: unpack_mx4(pack_mx4(mx4_linear(x, packed)))  # noqa: E731
    x = torch.randn(20, 200, device="cuda", dtype=BF)
    graph = make_fx(f)(x)
    names = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    assert any("rocm_qlora.mx4_forward" in n for n in names), names
    assert torch.equal(graph(x), f(x))
