"""The adapters' low-rank intermediate keeps its 32 bits in the products that
follow it.

Row 0's intermediates are 1 + 2^-9 + 2^-18 and 1 + 2^-9 (three and two of its
inputs sum to them exactly), and the weights or rows after them take their
difference, so every result is 2^-18, exact in each type.  From 8-bit codes
the intermediate is multiplied by a scale first: two roundings of 2^-24.
"""
import pytest
import torch

SMALL = 2.0 ** -18


def parts(width, dtype):
    """A row of `width` whose first three values sum to 1 + 2^-9 + 2^-18, and two ranks: of all three, of two."""
    row = torch.zeros(width, device="cuda", dtype=dtype)
    row[:3] = torch.tensor([1.0, 2.0 ** -9, SMALL])
    ranks = torch.zeros(width, 2, device="cuda", dtype=dtype)
    ranks[:3, 0] = 1
    ranks[:2, 1] = 1
    return row, ranks


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("rows,k,n", [(2, 40, 48), (70, 131, 264), (4500, 136, 40)])
def test_row_products(rows, k, n, rank, dtype):
    from rocm_qlora import _native as nat
    ops = nat.loaded_ops()
    row, ranks = parts(k, dtype)
    U = torch.zeros(1, k, rank, device="cuda", dtype=dtype)
    U[0, :, rank - 2:] = ranks
    V = torch.zeros(1, n, rank, device="cuda", dtype=dtype)
    V[0, :, rank - 2], V[0, :, rank - 1] = 1, -1
    out, mid = ops.adapters_apply(row.expand(rows, k).contiguous(), U, V, torch.ones(1, device="cuda"), None, None, 0)
    assert bool((mid[:, rank - 2] == 1 + 2.0 ** -9 + SMALL).all()) and bool((mid[:, rank - 1] == 1 + 2.0 ** -9).all())
    assert bool((out == SMALL).all()), float(out.max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("rows,k,count", [(2, 40, 1), (300, 131, 1), (300, 136, 1), (640, 136, 40)])
def test_bank_gradients(rows, k, count, rank, dtype):
    from rocm_qlora import _native as nat
    from rocm_qlora.activation8 import pack_activation
    from rocm_qlora.lora import AdapterPlan
    ops = nat.loaded_ops()
    z = torch.zeros(rows, k, device="cuda", dtype=dtype)
    z[0], z[1] = 1, -1
    mid = torch.zeros(rows, rank, device="cuda")
    mid[0], mid[1] = 1 + 2.0 ** -9 + SMALL, 1 + 2.0 ** -9
    ids = torch.arange(rows, device="cuda") % count
    ids[1] = 0
    plan = AdapterPlan(ids, count)
    got = ops.adapters_grad(z, None, mid, k, count, dtype, plan.data, plan.tile)
    assert bool((got[0] == SMALL).all()) and int(torch.count_nonzero(got[1:])) == 0
    p = pack_activation(z)
    got = ops.adapters_grad(p.codes, p.scales, mid, k, count, dtype, plan.data, plan.tile)
    # each row's 127 * (mid / 127) rounds twice: the scale, the product
    assert bool(((got[0].double() - SMALL).abs() <= 2.0 ** -21).all()), float(got[0].max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("rows,k", [(4200, 22016), (4200, 22015), (1000, 22016)])
def test_sums_of_long_rows_are_not_shifted(rows, k, rank, dtype):
    """Positive products: a tensor core cuts its sum off at each step, half of 2^-23 of it on average at most, and
    a run of 16 steps between two rounded additions therefore shifts it by 2^-20 at most."""
    from rocm_qlora import _native as nat
    ops = nat.loaded_ops()
    g = torch.Generator(device="cuda").manual_seed(rank)
    x = torch.rand(rows, k, generator=g, device="cuda").to(dtype)
    U = torch.rand(1, k, rank, generator=g, device="cuda").div(64).to(dtype)
    mid = ops.adapters_mid(x, U, torch.zeros(1, 8, rank, device="cuda", dtype=dtype), torch.ones(1, device="cuda"), None, 0)
    shift = []
    for at in range(0, rows, 700):
        want = x[at:at + 700].double() @ U[0].double()
        shift.append(((mid[at:at + 700].double() - want) / want).mean())
    assert abs(float(torch.stack(shift).mean())) <= 2.0 ** -20
