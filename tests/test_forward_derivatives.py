"""Forward-mode derivatives are not implemented: every differentiable operator
refuses a dual tensor, none drops its tangent.  Meta tensors stand for the
GPU's."""
import pytest
import torch
import torch.autograd.forward_ad as fw


def operands():
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    return [e(4, 32), e(4, 16), e(1, 16, 8), e(1, 32, 8), e(1, dtype=torch.float32)]


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("grad", [False, True])
def test_adapters_add(which, grad):
    from rocm_qlora.lora import adapters_add
    t = operands()
    with torch.set_grad_enabled(grad):
        assert adapters_add(*t).shape == (4, 32)
        with fw.dual_level():
            assert adapters_add(*t).shape == (4, 32)  # no tangent: nothing to refuse
            t[which] = fw.make_dual(t[which], torch.empty_like(t[which]))
            with pytest.raises(RuntimeError, match="jvp|forward"):
                adapters_add(*t)


@pytest.mark.parametrize("which", range(4))
def test_functional_transform(which):
    from rocm_qlora.lora import adapters_add
    t = operands()

    def f(v):
        return adapters_add(*t[:which], v, *t[which + 1:])

    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.jvp(f, (t[which],), (t[which],))


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(5))
def test_out(which):
    """The form that writes in place; without a tangent it runs."""
    from rocm_qlora.lora import adapters_add
    t = [torch.zeros(v.shape, device="cuda", dtype=v.dtype) for v in operands()]
    out = torch.zeros_like(t[0])
    with torch.no_grad(), fw.dual_level():
        adapters_add(*t, out=out)
        t[which] = fw.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="differentiation|jvp|forward"):
            adapters_add(*t, out=out)


def test_others_refuse():
    from rocm_qlora.activation8 import swiglu8
    from rocm_qlora.preference import preference_loss, token_logprobs
    logits, labels = torch.empty(2, 3, 9, device="meta"), torch.empty(2, 3, device="meta", dtype=torch.int64)
    with fw.dual_level():
        dual = fw.make_dual(logits, torch.empty_like(logits))
        for call in (lambda: swiglu8(dual, logits), lambda: swiglu8(logits, dual), lambda: token_logprobs(dual, labels),
                     lambda: preference_loss(dual, labels, torch.empty(2, 3, device="meta"))):
            with pytest.raises(RuntimeError, match="jvp|forward"):
                call()
