"""A bank of several adapters without a plan: every row uses adapter 0, and an
adapter without rows gets a zero gradient."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,d,rank,count", [(5, 40, 8, 2), (300, 264, 16, 3), (1500, 136, 16, 64), (1500, 264, 64, 70),
                                               (1500, 131, 128, 64)])
def test_rows_are_adapter_0s(rows, d, rank, count, dtype):
    from rocm_qlora import _native as nat
    ops = nat.loaded_ops()
    g = torch.Generator(device="cuda").manual_seed(rows)
    z = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
    mid = torch.randn(rows, rank, generator=g, device="cuda")
    torch.full((count, d, rank), float("nan"), device="cuda", dtype=dtype)  # what the result's memory held
    got = ops.adapters_grad(z, None, mid, d, count, dtype, None, 0)
    want = ops.adapters_grad(z, None, mid, d, 1, dtype, None, 0)
    # sums of `rows` fp32 products in one order or another, each rounded once to dtype
    bound = (rows + 4) * 2.0 ** -22 * (z.double().abs().t() @ mid.double().abs()) + \
        2.0 ** (-8 if dtype == torch.bfloat16 else -11) * want[0].double().abs() + 2.0 ** -24
    assert bool(((got[0].double() - want[0].double()).abs() <= 2 * bound).all())
    assert int(torch.count_nonzero(got[1:])) == 0
    # the row products' side of it
    U, V = (torch.randn(count, d, rank, generator=g, device="cuda").to(dtype) for _ in range(2))
    s = torch.ones(count, device="cuda")
    y, _ = ops.adapters_apply(z, U, V, s, None, None, 0)
    one, _ = ops.adapters_apply(z, U[:1], V[:1], s[:1], None, None, 0)
    assert torch.equal(y, one)
