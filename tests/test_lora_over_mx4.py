"""LoRALinear over a base in microscaled 4 bits: activations of either 16-bit
type whatever was packed, and the refusal to merge."""
import pytest
import torch

BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [F4, BF, HF])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_layer_over_weights_of_any_type(packed, dtype):
    """A base packed from 32-bit weights takes 16-bit activations as they are;
    one packed from 16 bits takes them in its own type."""
    from rocm_qlora import LoRALinear
    from rocm_qlora.mx4 import Mx4Linear
    torch.manual_seed(0)
    base = Mx4Linear.from_linear(torch.nn.Linear(96, 64, dtype=packed, device="cuda"))
    layer = LoRALinear(base, r=4).cuda()
    x = torch.randn(5, 96, device="cuda", dtype=dtype, requires_grad=True)
    y = layer(x)                                             # lora_B is 0
    want = base(x if packed == F4 else x.to(packed))
    assert y.dtype == want.dtype and torch.equal(y, want)
    torch.nn.init.normal_(layer.lora_B)
    grads = torch.autograd.grad(layer(x).float().square().sum(), (x, layer.lora_A, layer.lora_B))
    assert all(bool(torch.isfinite(g).all()) and bool(g.any()) for g in grads)


def test_merging_is_refused_and_changes_nothing():
    from rocm_qlora import LoRALinear
    from rocm_qlora.mx4 import Mx4Linear
    layer = LoRALinear(Mx4Linear(64, 32), r=4)
    torch.nn.init.normal_(layer.lora_B)
    before = layer.lora_B.detach().clone()
    with pytest.raises(TypeError, match="Mx4Linear"):
        layer.merge_lora()
    assert not layer.merged and torch.equal(layer.lora_B, before)
    with pytest.raises(RuntimeError):
        layer.unmerge_lora()
