"""Activations in 8 bits (rocm_qlora.activation8): the format bit for bit
against its definition in numpy fp32, swiglu8 against the formula in 64 bits,
and the adapters' gradient from packed inputs."""
import numpy as np
import pytest
import torch

from tests.test_adapters import F8, HALF, TINY, check, formula, make, run

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF8 = {**HALF, torch.float32: 2.0 ** -24}
TINY8 = {**TINY, torch.float32: 0.0}


def packed_numpy(x):
    """(codes, scales) of fp32 rows by the definition."""
    m, k = x.shape
    nb = -(-k // 128)
    v = np.zeros((m, nb * 128), np.float32)
    v[:, :k] = x
    v = v.reshape(m, nb, 128)
    with np.errstate(all="ignore"):
        top = np.abs(v).max(-1)
        bad = ~np.isfinite(v).all(-1)
        live = ~bad & (top >= np.float32(2.0 ** -100))
        scale = np.where(live, top / np.float32(127), np.where(bad, np.float32("nan"), np.float32(0))).astype(np.float32)
        by = np.where(live, np.float32(127) / np.where(live, top, 1), 0).astype(np.float32)
        codes = np.where(live[..., None], np.rint((v * by[..., None]).astype(np.float32)), 0).astype(np.int8)
    return codes.reshape(m, -1), scale


def dequantized(x):
    codes, scale = packed_numpy(x.float().cpu().numpy())
    m = x.shape[0]
    v = codes.reshape(m, -1, 128).astype(np.float64) * scale[..., None].astype(np.float64)
    return torch.from_numpy(v.reshape(m, -1)[:, :x.shape[1]].copy()).to(x.device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 127), (5, 128), (7, 129), (2, 1000), (33, 1088), (300, 130)])
def test_pack_is_the_definition(rows, k, dtype):
    from rocm_qlora.activation8 import pack_activation, unpack_activation
    g = torch.Generator().manual_seed(rows * k)
    x = torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    x = x.to(dtype)
    p = pack_activation(x.cuda())
    codes, scale = packed_numpy(x.float().numpy())
    assert np.array_equal(p.codes.cpu().numpy(), codes)
    assert np.array_equal(p.scales.cpu().numpy(), scale)
    want = torch.from_numpy((codes.reshape(rows, -1, 128).astype(np.float32) * scale[..., None]).reshape(rows, -1))
    out = unpack_activation(p)
    assert out.shape == x.shape and torch.equal(out.cpu(), want[:, :k].to(dtype))
    assert torch.equal(unpack_activation(p, torch.float32).cpu(), want[:, :k])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_zeros_tiny_infinite_and_nan_blocks(dtype):
    from rocm_qlora.activation8 import pack_activation, unpack_activation
    x = torch.ones(4, 512, dtype=dtype)
    x[0, :128] = 0
    x[0, 128:256] = -0.0
    if dtype != torch.float16:
        x[0, 256:384] = 2.0 ** -101
        x[1, :128] = 2.0 ** -100
    x[1, 200] = float("inf")
    x[2, 300] = float("nan")
    x[3, 400] = float("-inf")
    x[3, 20] = torch.finfo(dtype).min
    p = pack_activation(x.cuda())
    codes, scale = packed_numpy(x.float().numpy())
    assert np.array_equal(p.codes.cpu().numpy(), codes)
    assert np.array_equal(p.scales.cpu().numpy(), scale, equal_nan=True)
    out = unpack_activation(p).cpu()
    assert bool(torch.isnan(out[1, 128:256]).all()) and bool(torch.isnan(out[2, 256:384]).all())
    assert bool(torch.isfinite(out[0]).all()) and int(torch.count_nonzero(out[0, :256])) == 0


@pytest.mark.gpu
def test_pack_strided_rows_and_shapes():
    from rocm_qlora.activation8 import pack_activation, unpack_activation
    x = torch.randn(6, 700, device="cuda", dtype=torch.bfloat16)
    for part in (x[:, 8:400], x[:, 3:402], x[::2], x.view(2, 3, 700), x.t()):
        p = pack_activation(part)
        want = pack_activation(part.contiguous())
        assert torch.equal(p.codes, want.codes) and torch.equal(p.scales, want.scales)
        assert unpack_activation(p).shape == part.shape
    assert unpack_activation(pack_activation(x[:0])).shape == (0, 700)


def swiglu_formula(gate, up, dh):
    """h, dgate, dup in 64 bits with their bounds: one rounding to the type, and
    the few fp32 operations before it.  The exponential errs by 2^-20 at most
    here (|gate| < 40), so p and 1 - p do by as much, and so does the sum in
    dgate relative to the sum of its terms' magnitudes."""
    dt = gate.dtype
    g, u, d = gate.to(F8), up.to(F8), dh.to(F8)
    h = g * torch.sigmoid(g) * u
    g, u = dequantized(gate), dequantized(up)
    p = torch.sigmoid(g)
    dg, du = d * u * p * (1 + g * (1 - p)), d * g * p
    eps = 2.0 ** -18
    eh, eg, eu = eps * h.abs(), eps * (d * u * p).abs() * (1 + g.abs()), eps * du.abs()
    return [(v, HALF8[dt] * (v.abs() + e) + e + TINY8[dt]) for v, e in ((h, eh), (dg, eg), (du, eu))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (4, 127), (61, 384), (9, 1001), (130, 1088)])
def test_swiglu8(rows, k, dtype):
    from rocm_qlora.activation8 import pack_activation, swiglu8
    g = torch.Generator(device="cuda").manual_seed(k)
    both = (3 * torch.randn(rows, 2 * k, generator=g, device="cuda")).to(dtype)
    dh = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    gate, up = both[:, :k].detach().requires_grad_(), both[:, k:].detach().requires_grad_()
    h, packed = swiglu8(gate, up, pack_output=True)
    grads = torch.autograd.grad(h, (gate, up), dh)
    for got, want, name in zip((h, *grads), swiglu_formula(gate.detach(), up.detach(), dh), ("h", "dgate", "dup")):
        check(got, want, f"{name} {rows}x{k} {dtype}")
    again = pack_activation(h.detach())
    assert torch.equal(packed.codes, again.codes) and torch.equal(packed.scales, again.scales)
    assert torch.equal(swiglu8(gate, up), h)


@pytest.mark.gpu
def test_swiglu8_against_differences():
    """Central differences in 64 bits at the packed point, where the backward is taken."""
    from rocm_qlora.activation8 import swiglu8
    g = torch.Generator(device="cuda").manual_seed(1)
    gate, up, dh = (torch.randn(40, 200, generator=g, device="cuda", dtype=torch.float32) for _ in range(3))
    a, b = gate.requires_grad_(), up.requires_grad_()
    da, db = torch.autograd.grad(swiglu8(a, b), (a, b), dh)
    qa, qb = dequantized(gate.detach()), dequantized(up.detach())
    f = lambda s, t: (dh.to(F8) * torch.nn.functional.silu(s) * t).sum()  # noqa: E731
    for grad, move in ((da, (1.0, 0.0)), (db, (0.0, 1.0))):
        way = torch.randn(40, 200, generator=g, device="cuda", dtype=F8)
        e = 1e-5
        slope = (f(qa + e * move[0] * way, qb + e * move[1] * way) - f(qa - e * move[0] * way, qb - e * move[1] * way))
        slope = float(slope / (2 * e))
        # the difference's own error is e^2 times third derivatives (< 1 here) and 1e-16 / e of the sum
        scale = float((dh.to(F8) * (1 + qb.abs()) * (1 + qa.abs()) * way).abs().sum())
        assert abs(float((grad.to(F8) * way).sum()) - slope) <= scale * (2.0 ** -18 + 1e-10 + 1e-11)


@pytest.mark.gpu
def test_swiglu8_extreme_gates():
    from rocm_qlora.activation8 import swiglu8
    gate = torch.tensor([[-300.0, 300.0, 0.0, -88.0, float("inf")]], device="cuda", dtype=torch.bfloat16)
    up = torch.full_like(gate, 2.0)
    h = swiglu8(gate, up)
    assert torch.equal(h[0, [0, 1, 2, 4]].float().cpu(), torch.tensor([0.0, 600.0, 0.0, float("inf")]))
    assert abs(float(h[0, 3])) < 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k,n,rank,count", [
    (1, 64, 64, 8, 1), (5, 127, 129, 16, 3), (33, 1088, 72, 64, 2), (260, 300, 136, 16, 1), (700, 520, 40, 128, 3)])
def test_adapter_gradients_from_packed_inputs(rows, k, n, rank, count, dtype):
    """dA is of the packed values; everything else is as without packing."""
    from rocm_qlora.activation8 import pack_activation
    t = make(rows, k, n, rank, count, dtype, seed=k)
    t["x"][:, ::50] *= 8
    y, grads = run(t, packed_x=pack_activation(t["x"]))
    plain_y, plain = run(t)
    assert torch.equal(y, plain_y) and torch.equal(grads[1], plain[1]) and torch.equal(grads[3], plain[3])
    value, bound = formula(t, z=dequantized(t["x"]))[2]
    # code * scale enters as fp32: one more rounding, 2^-24 of the sums' magnitudes, inside the accumulation's
    check(grads[2], (value, bound), f"dA {rows}x{k} r{rank}")


@pytest.mark.gpu
def test_packed_nan_block_reaches_the_gradient():
    from rocm_qlora.activation8 import pack_activation
    t = make(20, 256, 64, 16, 1, torch.bfloat16, none=0.0)
    t["x"][4, 130] = float("nan")
    packed = pack_activation(t["x"])
    t["x"][4, 130] = 0.0
    _, grads = run(t, packed_x=packed)
    assert bool(torch.isfinite(grads[2][0, :128].float()).all()) and bool(torch.isnan(grads[2][0, 128:]).all())


def test_refusals():
    from rocm_qlora import _native as nat
    from rocm_qlora.activation8 import pack_activation, swiglu8
    with pytest.raises(nat.NativeUnavailable):
        pack_activation(torch.zeros(2, 3))
    with pytest.raises(TypeError, match="unsupported dtype"):
        pack_activation(torch.zeros(2, 3, dtype=torch.float64))
    with pytest.raises(ValueError):
        pack_activation(torch.zeros(()))
    with pytest.raises(ValueError, match="differ"):
        swiglu8(torch.zeros(2, 3), torch.zeros(2, 4))
    with pytest.raises(ValueError, match="differ"):
        swiglu8(torch.zeros(2, 3), torch.zeros(2, 3).half())
    with pytest.raises(nat.NativeUnavailable):
        swiglu8(torch.zeros(2, 3), torch.zeros(2, 3))


@pytest.mark.gpu
def test_packed_input_of_another_shape_is_refused():
    from rocm_qlora.activation8 import pack_activation
    t = make(20, 256, 64, 16, 1, torch.bfloat16)
    for other in (t["x"][:, :128], t["x"][:10]):
        with pytest.raises(ValueError, match="packed_x"):
            run(t, packed_x=pack_activation(other))
