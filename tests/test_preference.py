"""Token log-probabilities and the preference loss (rocm_qlora.preference)
against their definitions in 64 bits.

Bounds: a row's normaliser is a sum of V exponentials in fp32, summed in
blocks, so log s errs by well under 2^-18, and x - m by half an ulp of fp32
(exact for most 16-bit logits); a probability therefore errs by 2^-17 of
itself at most, a log-probability by 2^-17 absolutely plus 2^-23 of itself.
"""
import pytest
import torch

F8 = torch.float64
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
LOGP = 2.0 ** -17
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(pairs, length, vocab, dtype, seed=0, masked=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b = 2 * pairs
    logits = (3 * torch.randn(b, length, vocab, generator=g, device="cuda")).to(dtype)
    labels = torch.randint(0, vocab, (b, length), generator=g, device="cuda")
    labels[torch.rand(b, length, generator=g, device="cuda") < masked] = -100
    ref = exact_logps(logits, labels).float() + 0.2 * torch.randn(b, length, generator=g, device="cuda")
    return logits, labels, ref


def target_of(labels):
    return torch.nn.functional.pad(labels[:, 1:], (0, 1), value=-100)


def exact_logps(logits, labels):
    """At each label's place its log-probability, 0 where none counts (64 bits)."""
    t = target_of(labels)
    lp = torch.log_softmax(logits.to(F8), -1).gather(-1, t.clamp(min=0)[..., None])[..., 0]
    lp = torch.where(t != -100, lp, 0.0)
    return torch.nn.functional.pad(lp[:, :-1], (1, 0))


def exact_loss(logps, labels, ref, beta, smooth, form):
    counts = target_of(labels) != -100
    n = counts.sum(1).clamp(min=1)
    counted = torch.nn.functional.pad(counts[:, :-1], (1, 0))
    R = torch.where(counted, logps - ref.to(F8), 0.0).sum(1)
    h = len(n) // 2
    if form == "ipo":
        return ((R[:h] / n[:h] - R[h:] / n[h:] - 0.5 / beta) ** 2).mean(), R
    z = beta * (R[:h] - R[h:])
    ls = torch.nn.functional.logsigmoid
    return (-(1 - smooth) * ls(z) - smooth * ls(-z)).mean(), R


CASES = [(1, 1, 5), (1, 2, 1), (1, 7, 33), (2, 17, 1000), (3, 5, 4097), (1, 9, 32000), (2, 3, 32001), (1, 3, 131073),
         (40, 3, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairs,length,vocab", CASES)
def test_logprobs_and_gradient(pairs, length, vocab, dtype):
    from rocm_qlora.preference import token_logprobs
    logits, labels, _ = make(pairs, length, vocab, dtype, seed=vocab)
    x = logits.clone().requires_grad_()
    got = token_logprobs(x, labels)
    want = exact_logps(logits, labels)
    assert got.dtype == torch.float32
    assert bool(((got.to(F8) - want).abs() <= LOGP + 2.0 ** -23 * want.abs()).all())
    g = torch.randn(got.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    d, = torch.autograd.grad(got, x, g)
    t = target_of(labels)
    slope = torch.where(t != -100, torch.nn.functional.pad(g[:, 1:], (0, 1)), 0.0).to(F8)[..., None]
    p = torch.softmax(logits.to(F8), -1)
    one = torch.zeros_like(p).scatter_(-1, t.clamp(min=0)[..., None], 1.0)
    want = slope * (one - p)
    e = slope.abs() * (2.0 ** -16 * p + 2.0 ** -22 * one)
    assert bool(((d.to(F8) - want).abs() <= HALF[dtype] * (want.abs() + e) + e + TINY[dtype]).all())
    assert int(torch.count_nonzero(d[t == -100])) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form,smooth", [("sigmoid", 0.0), ("sigmoid", 0.2), ("ipo", 0.0)])
@pytest.mark.parametrize("pairs,length,vocab", CASES)
def test_preference_loss(pairs, length, vocab, form, smooth):
    from rocm_qlora.preference import preference_loss
    dtype, beta = torch.float32, 0.3
    logits, labels, ref = make(pairs, length, vocab, dtype, seed=vocab + 1)
    x = logits.clone().requires_grad_()
    out = preference_loss(x, labels, ref, beta=beta, label_smoothing=smooth, form=form)
    d, = torch.autograd.grad(out.loss, x, torch.tensor(-1.5, device="cuda"))

    y = logits.to(F8).requires_grad_()
    logps = exact_logps(y, labels)
    loss, R = exact_loss(logps, labels, ref, beta, smooth, form)
    want, = torch.autograd.grad(loss, y)
    n = float((target_of(labels) != -100).sum(1).max())
    off = n * LOGP + 2.0 ** -22 * float(logps.detach().abs().sum(1).max())  # of a sequence's sum
    assert bool(((out.logps.to(F8) - logps.sum(1).detach()).abs() <= 2 * off).all())
    rewards = torch.cat([out.chosen_rewards, out.rejected_rewards]).to(F8)
    assert bool(((rewards - beta * R.detach()).abs() <= 2 * beta * off + 2.0 ** -22 * R.detach().abs()).all())
    # the loss moves by at most its slope's bound times the error of the two sums (per token for ipo)
    if form == "ipo":
        size = float((torch.sqrt(loss.detach()) * pairs ** 0.5 + LOGP) * 2)
        dloss, curve = size * 2 * (LOGP + 2.0 ** -22 * float(logps.detach().abs().max())), 2.0 / pairs
        slope_off = curve * 2 * LOGP * 2
    else:
        dloss, slope_off = 2 * beta * off, beta * beta * 0.25 * 2 * off / pairs
    assert abs(float(out.loss) - float(loss)) <= dloss + 2.0 ** -22 * float(loss)
    assert out.loss.dtype == torch.float32
    p = torch.softmax(logits.to(F8), -1)
    one = torch.zeros_like(p).scatter_(-1, target_of(labels).clamp(min=0)[..., None], 1.0)
    bound = 1.5 * (want.abs() * 2.0 ** -15 + (slope_off + 2.0 ** -20 * beta) * (one + p) * 2 + 2.0 ** -22 * (one + p))
    assert bool(((d.to(F8) + 1.5 * want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["sigmoid", "ipo"])
def test_gradient_against_differences(form):
    from rocm_qlora.preference import preference_loss
    logits, labels, ref = make(2, 9, 50, torch.float32)
    x = logits.clone().requires_grad_()
    d, = torch.autograd.grad(preference_loss(x, labels, ref, beta=0.2, form=form).loss, x)
    g = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(4):
        way = torch.randn(logits.shape, generator=g, device="cuda", dtype=F8)
        way /= way.norm()
        e = 1e-4
        f = lambda s: exact_loss(exact_logps(logits.to(F8) + s * way, labels), labels, ref, 0.2, 0.0, form)[0]  # noqa: E731
        slope = float(f(e) - f(-e)) / (2 * e)
        # second-order differences: e^2 times a third derivative of order 10; the gradient's own error 2^-15
        assert abs(float((d.to(F8) * way).sum()) - slope) <= 1e-6 + 2.0 ** -15 * float(d.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lift", [0.0, 12.0])
def test_log_probabilities_are_not_biased(lift, dtype):
    """Sums over thousands of tokens add a common error up, so the mean over
    1600 rows is held to 2^-25 (a quarter of an ulp of 1): flat rows, and rows
    that one token dominates (lift), where the others' sum is what remains."""
    from rocm_qlora.preference import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(4)
    logits = 2 * torch.randn(4, 401, 8000, generator=g, device="cuda")
    labels = torch.randint(0, 8000, (4, 401), generator=g, device="cuda")
    logits[:, :-1].scatter_add_(2, labels[:, 1:, None], torch.full((4, 400, 1), lift, device="cuda"))
    logits = logits.to(dtype)
    got = token_logprobs(logits, labels).double()
    off = (got - exact_logps(logits, labels))[:, 1:]
    # what token_logprobs returns is rounded to fp32: up to 2^-21 each, without a bias
    assert abs(float(off.mean())) <= 2.0 ** -25 + 2.0 ** -21 / 1600 ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_logits(dtype):
    """A slice of a padded vocabulary, sequences apart and an odd start."""
    from rocm_qlora.preference import preference_loss, token_logprobs
    wide = torch.randn(4, 13, 259, device="cuda").to(dtype)
    part = wide[:, 2:11, 5:206]
    labels = torch.randint(0, 201, (4, 9), device="cuda")
    whole = part.contiguous()
    ref = token_logprobs(whole, labels) * 0.9
    got = [preference_loss(v.detach().requires_grad_(), labels, ref) for v in (part, whole)]
    assert all(torch.allclose(a, b, rtol=0, atol=2 * 9 * LOGP) for a, b in zip(got[0], got[1]))
    swapped = whole.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(token_logprobs(swapped, labels), token_logprobs(whole, labels))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_counts(dtype):
    from rocm_qlora.preference import preference_loss, token_logprobs
    logits = torch.randn(4, 6, 100, device="cuda").to(dtype).requires_grad_()
    labels = torch.full((4, 6), -100, device="cuda")
    out = preference_loss(logits, labels, torch.zeros(4, 6, device="cuda"))
    assert abs(float(out.loss.detach()) - 0.6931471805599453) < 1e-6
    assert int(torch.count_nonzero(out.logps)) == 0 and int(torch.count_nonzero(out.chosen_rewards)) == 0
    d, = torch.autograd.grad(out.loss, logits)
    assert int(torch.count_nonzero(d)) == 0
    assert int(torch.count_nonzero(token_logprobs(logits, labels))) == 0
    # masked rows are not read: NaN in them stays there
    labels[:, 3] = 7
    bad = logits.detach().clone()
    bad[:, [0, 1, 3, 4, 5]] = float("nan")
    bad.requires_grad_()
    out = preference_loss(bad, labels, torch.zeros(4, 6, device="cuda"))
    d, = torch.autograd.grad(out.loss, bad)
    assert bool(torch.isfinite(out.loss)) and bool(torch.isfinite(d).all())
    # an ignored label may be inside the vocabulary
    same = preference_loss(bad, torch.where(labels == -100, 9, labels), torch.zeros(4, 6, device="cuda"), ignore_index=9)
    assert torch.equal(same.loss, out.loss)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_lowest_values_and_infinities(dtype):
    """Vocabulary entries masked with the type's lowest value or -inf take no
    probability; a label among them has log-probability -inf; +inf and NaN and
    rows without any finite logit give NaN, in their own row alone."""
    from rocm_qlora.preference import token_logprobs
    logits = torch.randn(2, 8, 300, device="cuda").to(dtype)
    labels = torch.randint(0, 100, (2, 8), device="cuda")
    logits[:, :, 150:220] = torch.finfo(dtype).min
    logits[:, :, 220:] = float("-inf")
    short = token_logprobs(logits[:, :, :150].contiguous(), labels)
    x = logits.clone().requires_grad_()
    got = token_logprobs(x, labels)
    assert torch.allclose(got, short, rtol=0, atol=2 * LOGP)
    d, = torch.autograd.grad(got.sum(), x)
    assert bool(torch.isfinite(d).all()) and int(torch.count_nonzero(d[:, :, 150:])) == 0
    labels[0, 3], labels[0, 6] = 250, 300
    logits[1, 1, 4], logits[1, 3, 5] = float("inf"), float("nan")
    logits[1, 5] = float("-inf")
    got = token_logprobs(logits, labels)
    assert float(got[0, 3]) == float("-inf") and bool(torch.isnan(got[0, 6]))
    assert bool(torch.isnan(got[1, [2, 4, 6]]).all())
    fine = torch.ones(2, 8, dtype=torch.bool, device="cuda")
    fine[0, [3, 6]] = False
    fine[1, [2, 4, 6]] = False
    assert torch.allclose(got[fine], short[fine], rtol=0, atol=2 * LOGP)


@pytest.mark.gpu
def test_label_outside_the_vocabulary():
    from rocm_qlora.preference import preference_loss
    logits = torch.randn(2, 4, 30, device="cuda", requires_grad=True)
    for bad in (30, -1, 2 ** 40):
        labels = torch.randint(0, 30, (2, 4), device="cuda")
        labels[0, 2] = bad
        out = preference_loss(logits, labels, torch.zeros(2, 4, device="cuda"))
        d, = torch.autograd.grad(out.loss, logits)
        assert bool(torch.isnan(out.loss)) and bool(torch.isnan(d[0, 1]).all())


@pytest.mark.gpu
def test_saturated_pairs_and_other_stream():
    from rocm_qlora.preference import preference_loss, token_logprobs
    logits, labels, _ = make(2, 20, 64, torch.float32, masked=0.0)
    ref = token_logprobs(logits, labels)
    ref[:2] += 900.0   # z = -beta * 900 * 19: the loss is linear there
    out = preference_loss(logits.requires_grad_(), labels, ref, beta=1.0)
    assert abs(float(out.loss) / (900.0 * 19) - 1) < 1e-4
    d, = torch.autograd.grad(out.loss, logits)
    assert bool(torch.isfinite(d).all())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = preference_loss(logits, labels, ref, beta=1.0)
        e, = torch.autograd.grad(again.loss, logits)
    s.synchronize()
    assert torch.equal(again.loss, out.loss) and torch.equal(d, e)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows whose first element lies over 2^32 bytes and 2^31 elements in."""
    from rocm_qlora.preference import token_logprobs
    logits = torch.zeros(2, 36, 32768, device="cuda", dtype=torch.bfloat16)
    big = torch.empty(2 ** 31 + 2 ** 26, device="cuda", dtype=torch.bfloat16)
    far = big.as_strided((2, 36, 32768), (2 ** 31, 32768, 1))
    logits.normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    far.copy_(logits)
    labels = torch.randint(0, 32768, (2, 36), device="cuda")
    assert torch.equal(token_logprobs(far, labels), token_logprobs(logits, labels))


def test_refusals():
    from rocm_qlora import _native as nat
    from rocm_qlora.preference import preference_loss, token_logprobs
    logits, labels, ref = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    with pytest.raises(nat.NativeUnavailable):
        preference_loss(logits, labels, ref)
    with pytest.raises(nat.NativeUnavailable):
        token_logprobs(logits, labels)
    for kw, match in ((dict(form="hinge"), "form"), (dict(beta=0.0), "beta"), (dict(label_smoothing=0.6), "smoothing")):
        with pytest.raises(ValueError, match=match):
            preference_loss(logits, labels, ref, **kw)
    with pytest.raises(ValueError, match="pairs"):
        preference_loss(logits[:1], labels[:1], ref[:1])
    with pytest.raises(ValueError, match="ref_logps"):
        preference_loss(logits, labels, torch.zeros(2))
    with pytest.raises(ValueError, match="logits must be"):
        token_logprobs(logits[0], labels)
    with pytest.raises(TypeError, match="int64"):
        token_logprobs(logits, labels.int())
    with pytest.raises(TypeError, match="unsupported dtype"):
        token_logprobs(logits.double(), labels)
