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


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 4096, 4096), (8, 1024, 130), (16, 4096, 2048), (33, 2048, 1000),
                                      (64, 4096, 2048), (200, 4096, 512), (20, 200, 100)])
def test_a_wait_that_runs_out_leaves_no_partial_sums(rows, k, n):
    """Without time for a wait no product has its sums, whether one CTA or a
    cluster makes them: outputs are NaN, the timeouts are counted, and the next
    call is as ever."""
    import ctypes
    from rocm_qlora import _native as nat
    from rocm_qlora.mx4 import mx4_linear, pack_mx4
    L = nat.load_library()
    x, bias = torch.randn(rows, k, device="cuda", dtype=BF), torch.randn(n, device="cuda", dtype=BF)
    w = pack_mx4(torch.randn(n, k, device="cuda", dtype=BF))
    want = mx4_linear(x, w, bias)
    out = torch.full((rows, n), 7.0, device="cuda", dtype=BF)
    need = L.rq_mx4_linear_workspace_bytes(rows, n, k)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    count = ctypes.c_uint(0)

    def call():
        torch.cuda.synchronize()
        rc = L.rq_mx4_linear(x.data_ptr(), 1, k, rows, w.codes.data_ptr(), w.scales.data_ptr(), n, k, bias.data_ptr(),
                             out.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and L.rq_take_kernel_timeouts(ctypes.byref(count)) == 0
        return count.value

    assert L.rq_take_kernel_timeouts(ctypes.byref(count)) == 0
    try:
        assert L.rq_mx4_set_wait(0) == 0
        assert call() > 0 and bool(torch.isnan(out).all())
    finally:
        assert L.rq_mx4_set_wait(-1) == 0
    assert call() == 0 and torch.equal(out, want)


def test_the_limit_of_a_wait_takes_any_number():
    from rocm_qlora import _native as nat
    L = nat.load_library()
    for ns in (0, 1, 2 ** 62, -2 ** 63, -1):
        assert L.rq_mx4_set_wait(ns) == 0


def test_unpacking_into_another_number_of_rows_is_refused():
    from rocm_qlora import _native as nat
    from tests.test_mx4 import meta
    ops, (codes, scales) = nat.loaded_ops(), meta(6, 160)
    assert ops.unpack_mx4(codes, scales, [2, 3, 160], BF).shape == (2, 3, 160)
    for shape in ([5, 160], [7, 160], [2, 2, 160], [160]):
        with pytest.raises(ValueError, match="rows"):
            ops.unpack_mx4(codes, scales, shape, BF)
    one = meta(1, 160)
    assert ops.unpack_mx4(*one, [160], BF).shape == (160,)
