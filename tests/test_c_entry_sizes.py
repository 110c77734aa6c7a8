"""C entries of the log-probabilities: sizes whose product leaves 64 bits are refused."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("b,l", [(1 << 62, 4), (4, 1 << 62), (1 << 32, 1 << 32), ((1 << 62) + 2, 4), (1 << 20, 1 << 20)])
def test_batch_times_length(b, l):
    from rocm_qlora import _native as nat
    L = nat.lib()
    t = torch.zeros(64, device="cuda")
    labels = torch.zeros(16, device="cuda", dtype=torch.int64)
    st = nat.stream_ptr(t.device)
    p, y = t.data_ptr(), labels.data_ptr()
    assert L.rq_token_logprobs(p, nat.F32, 4, 1, b, l, 1, y, -100, p, None, st) == -1
    assert L.rq_token_logprobs_grad(p, nat.F32, 4, 1, b, l, 1, y, -100, p, p, 0, None, p, st) == -1
    assert L.rq_preference_loss(b, l, y, -100, p, p, 0, 0.1, 0.0, p, p, p, p, st) == -1
