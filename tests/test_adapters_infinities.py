"""Infinities among the adapters' weights and the rows: where the formula in
64 bits has an infinity, or a finite value, so have the kernels, in its place;
NaN where it has NaN."""
import pytest
import torch

F8 = torch.float64
INF = float("inf")


def same_kind(got, want):
    got, want = got.to(F8), want.to(got.dtype).to(F8)  # a value past the type's range is an infinity of it
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isposinf(got), torch.isposinf(want)) and torch.equal(torch.isneginf(got), torch.isneginf(want))


def inputs(rows, k, n, rank, dtype):
    """Values that are short binary fractions, so that the intermediates have no remainder beside their first
    16-bit piece in some places, and others that have one."""
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    draw = lambda *s: torch.randint(1, 9, s, generator=g, device="cuda").div(8).to(dtype)  # noqa: E731
    x, U, V, base = draw(rows, k), draw(1, k, rank), draw(1, n, rank), draw(rows, n)
    x[1::2] = (x[1::2].float() * 1.3).to(dtype)
    return x, U, V, base


SIZES = [(1, 64, 64), (5, 4096, 136), (33, 1093, 131), (300, 260, 264), (4500, 520, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("where", ["u first", "u last", "u many", "v", "v nan", "x", "base"])
def test_row_products(rows, k, n, rank, where, dtype):
    from rocm_qlora import _native as nat
    ops = nat.loaded_ops()
    x, U, V, base = inputs(rows, k, n, rank, dtype)
    if where == "u first":
        U[0, 0, 1] = INF
    elif where == "u last":
        U[0, k - 1, 0] = -INF
    elif where == "u many":
        U[0, k // 3: k // 2, 2] = INF
    elif where == "v":
        V[0, n // 2, 3], V[0, 1, rank - 1] = INF, -INF
    elif where == "v nan":
        V[0, n // 2, 3] = float("nan")
    elif where == "x":
        x[rows // 2, k // 2] = INF
    else:
        base[rows // 2, n // 2] = -INF
    s = torch.full((1,), 0.5, device="cuda")
    out, mid = ops.adapters_apply(x, U, V, s, base, None, 0)
    want_mid = 0.5 * (x.to(F8) @ U[0].to(F8))
    want = base.to(F8) + want_mid @ V[0].to(F8).t()
    same_kind(mid, want_mid)
    same_kind(out, want)
    same_kind(ops.adapters_apply_(base.clone(), x, U, V, s, base, None, 0), want_mid)
    again = base.clone()
    ops.adapters_apply_(again, x, U, V, s, again, None, 0)
    assert torch.equal(again.isnan(), out.isnan()) and torch.equal(again.nan_to_num(), out.nan_to_num())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("rows,d,count", [(3, 64, 1), (300, 131, 1), (300, 264, 1), (1500, 136, 1), (640, 136, 40),
                                          (1500, 264, 64)])
@pytest.mark.parametrize("where", ["z", "z many", "z nan", "mid", "mid and z"])
def test_bank_gradients(rows, d, rank, count, where, dtype):
    from rocm_qlora import _native as nat
    from rocm_qlora.lora import AdapterPlan
    ops = nat.loaded_ops()
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    z = torch.randint(1, 9, (rows, d), generator=g, device="cuda").div(8).to(dtype)
    mid = torch.randint(1, 9, (rows, rank), generator=g, device="cuda").div(8)
    mid[1::2] *= 1.0 + 2.0 ** -12
    ids = torch.arange(rows, device="cuda") % count
    if count == 64:
        ids[: rows // 2] = 5  # most of the rows are one adapter's
    if where.startswith("z"):
        z[rows // 2, 3] = float("nan") if where == "z nan" else INF
    if where == "z many":
        z[0, d // 2:] = -INF
        z[rows - 1, d - 1] = INF
    if "mid" in where:
        mid[rows // 3, rank - 1] = -INF
    if where == "mid and z":
        z[rows // 2, 3], z[rows // 3, 1] = INF, -INF
    plan = AdapterPlan(ids, count)
    got = ops.adapters_grad(z, None, mid, d, count, dtype, plan.data, plan.tile)
    for a in range(count):
        at = (ids == a).nonzero()[:, 0]
        same_kind(got[a], z[at].to(F8).t() @ mid[at].to(F8))
