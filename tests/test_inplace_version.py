"""adapters_add(out=...) writes in place: autograd's version counter of the
output counts it, so that a node that saved the tensor before refuses its
backward instead of using what is there now."""
import pytest
import torch


def test_counter():
    from rocm_qlora import _native as nat
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    out = e(4, 32)
    args = (e(4, 16), e(1, 16, 8), e(1, 32, 8), e(1, dtype=torch.float32), e(4, 32), None, 0)
    before = out._version
    nat.loaded_ops().adapters_apply_(out, *args)
    assert out._version == before + 1 and all(t._version == 0 for t in args[:5])
    nat.loaded_ops().adapters_apply_(out.view(2, 64).view(4, 32), *args)
    assert out._version == before + 2
    with torch.inference_mode():
        held = e(4, 32)
        nat.loaded_ops().adapters_apply_(held, *args)  # has no counter


@pytest.mark.gpu
def test_saved_output_is_refused():
    from rocm_qlora.lora import adapters_add
    base, x = torch.ones(4, 32, device="cuda").bfloat16(), torch.ones(4, 16, device="cuda").bfloat16()
    A, B, s = torch.ones(1, 16, 8, device="cuda").bfloat16(), torch.ones(1, 32, 8, device="cuda").bfloat16(), torch.ones(1, device="cuda")
    w = torch.ones(4, 32, device="cuda").bfloat16().requires_grad_()
    product = w * base  # saves base
    with torch.no_grad():
        got = adapters_add(base, x, A, B, s, out=base)
    assert got is base and float(base[0, 0]) == 129.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
