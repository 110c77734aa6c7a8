"""Products in microscaled 4 bits where CTAs of a cluster meet: results that
must not depend on who is first, and waits that run out."""
import pytest
import torch

from tests.test_mx4 import BF, F8, HF, close, kept, sums


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,k,n", [(1, 1024, 2048), (130, 200, 1537), (257, 640, 385), (700, 2049, 900)])
def test_gradient_is_the_same_every_time(rows, k, n, dtype):
    """Both CTAs of a pair widen the weight, and one issues the MMAs: tiles of
    128 and 256 columns, rings that go round several times, 50 calls."""
    from rocm_qlora import _native as nat
    from rocm_qlora.mx4 import pack_mx4
    g = torch.Generator(device="cuda").manual_seed(rows)
    w = (torch.randn(n, k, generator=g, device="cuda") * 0.05).to(dtype)
    dy = (torch.randn(rows, n, generator=g, device="cuda") * 0.1).to(dtype)
    packed, wk = pack_mx4(w), kept(w)
    got = [nat.loaded_ops().mx4_dx(dy, packed.codes, packed.scales, k) for _ in range(50)]
    close(got[0], dy.to(F8) @ wk, sums(dy.to(F8), wk.t(), n))
    assert all(torch.equal(x, got[0]) for x in got)
