"""Log-probabilities of rows of any finite magnitude: masked whole with the
type's lowest value, partly with a large negative one, or with its largest
value among them.  Against log_softmax in 64 bits.

Bounds: as everywhere, a log-probability errs by 2^-17 absolutely and 2^-23 of
itself, a probability by 2^-17 of itself, and a gradient is rounded once.
"""
import pytest
import torch

F8 = torch.float64
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rows_of(kind, vocab, dtype, g):
    """One row [vocab] of a kind; None where the type has no such value."""
    info = torch.finfo(dtype)
    x = 3 * torch.randn(vocab, generator=g, device="cuda")
    if kind == "lowest":
        return torch.full((vocab,), info.min, device="cuda", dtype=dtype)
    if kind == "largest":
        return torch.full((vocab,), info.max, device="cuda", dtype=dtype)
    x = x.to(dtype)
    if kind == "one largest":
        x[vocab // 3] = info.max
    elif kind == "two scales":
        x[:] = info.min
        x[vocab // 2:] = info.min / 2
    elif kind == "lowest but one":
        x[:] = info.min
        x[vocab - 2] = 1.5
    else:  # a magnitude: the first half masked with -it, the whole row shifted down or up by it
        value, how = kind
        if value > info.max:
            return None
        if how == "first half":
            x[: vocab // 2] = -value
        elif how == "last half":
            x[vocab // 2:] = -value
        else:
            x = (x.to(F8) + (value if how == "up" else -value)).clamp(info.min, info.max).to(dtype)
    return x


KINDS = ["lowest", "largest", "one largest", "two scales", "lowest but one"] + [
    (v, how) for v in (6e4, 1e7, 1e9, 1e10, 3e20, 1e30, 2.5e38) for how in ("first half", "last half", "up", "down")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 5, 1000, 32001])
@pytest.mark.parametrize("copies", [1, 300])  # few rows, and enough of them for the small blocks
def test_rows_of_any_magnitude(vocab, copies, dtype):
    from rocm_qlora.preference import token_logprobs
    if vocab == 32001 and copies == 300:
        copies = 40
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows = [r for r in (rows_of(k, vocab, dtype, g) for k in KINDS) if r is not None]
    logits = torch.stack(rows + [rows[0]])[None].expand(copies, -1, -1).contiguous()
    length = logits.shape[1]
    labels = torch.randint(0, vocab, (copies, length), generator=g, device="cuda")
    labels[:, 3] = vocab - vocab // 3 - 1
    leaf = logits.clone().requires_grad_()
    got = token_logprobs(leaf, labels)
    up = torch.randn(copies, length, generator=g, device="cuda")
    grad, = torch.autograd.grad(got, leaf, up)
    for i in range(0, copies, 37):
        x, y = logits[i, :-1].to(F8), labels[i, 1:]
        lp = torch.log_softmax(x, -1)
        want = lp.gather(1, y[:, None])[:, 0]
        off = (got[i, 1:].to(F8) - want).abs()
        assert bool((off <= 2.0 ** -17 + 2.0 ** -23 * want.abs()).all()), (got[i, 1:][off > 1e-3], want[off > 1e-3])
        c = up[i, 1:].to(F8)
        hot = torch.zeros_like(x).scatter_(1, y[:, None], 1.0)
        d = c[:, None] * (hot - lp.exp())
        err = 2.0 ** -17 * c.abs()[:, None] * (lp.exp() + hot * 2.0 ** -6)
        bound = HALF[dtype] * (d.abs() + err) + err + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)
        off = (grad[i, :-1].to(F8) - d).abs()
        assert bool((off <= bound).all()), float((off - bound).max())
    assert int(torch.count_nonzero(grad[:, -1])) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", ["sigmoid", "ipo"])
def test_loss_with_a_masked_row(form, dtype):
    """A counted row at the type's lowest value is uniform: -log V, not NaN."""
    from rocm_qlora.preference import preference_loss
    g = torch.Generator(device="cuda").manual_seed(0)
    logits = torch.randn(2, 6, 500, generator=g, device="cuda").to(dtype)
    logits[0, 2] = torch.finfo(dtype).min
    labels = torch.randint(0, 500, (2, 6), generator=g, device="cuda")
    leaf = logits.clone().requires_grad_()
    out = preference_loss(leaf, labels, torch.zeros(2, 6, device="cuda"), form=form)
    lp = torch.log_softmax(logits[:, :-1].to(F8), -1).gather(-1, labels[:, 1:, None])[..., 0].sum(1)
    assert bool(((out.logps.to(F8) - lp).abs() <= 5 * 2.0 ** -17 + 2.0 ** -22 * lp.abs()).all())
    grad, = torch.autograd.grad(out.loss, leaf)
    assert bool(torch.isfinite(grad.float()).all()) and bool(torch.isfinite(out.loss))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_distribution(dtype):
    """A row of -inf alone, or with +inf or NaN in it, is no distribution: NaN."""
    from rocm_qlora.preference import token_logprobs
    logits = torch.full((1, 5, 700), torch.finfo(dtype).min, device="cuda", dtype=dtype)
    logits[0, 0] = -float("inf")
    logits[0, 1, 600] = float("inf")
    logits[0, 2, 3] = float("nan")
    logits[0, 3, 10:] = -float("inf")
    got = token_logprobs(logits, torch.full((1, 5), 5, device="cuda"))[0].cpu()
    assert bool(torch.isnan(got[1:4]).all())
    assert abs(float(got[4]) + 2.302585092994046) <= 2.0 ** -17
