"""The fused cross-entropy scorer after an expired wait."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab,k", [(40, 1000, 64), (700, 50257, 128), (2100, 8000, 2112)])
def test_expired_wait_leaves_no_numbers(rows, vocab, k):
    """What a call whose wait ran out could not compute is NaN and counts as wrong, not what the
    workspace held: here the good result of the call before."""
    from zotitan_b200 import kernels as K
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, k, device="cuda", generator=g).bfloat16()
    w = torch.randn(vocab, k, device="cuda", generator=g).bfloat16()
    t = (x.float() @ w.float().t()).argmax(1)      # nearly every row correct
    t[3::7] = -100
    want = K.linear_xent(x, w, t)
    assert K.linear_xent_take_error() == 0 and torch.isfinite(want[0]).all() and bool(want[2].any())
    loss, lse, correct = K.linear_xent(x, w, t, test_stall_loads=True, test_wait_cycles=2_000_000)
    assert K.linear_xent_take_error() != 0
    for out in (loss, lse):
        assert torch.isnan(out[t >= 0]).all() and not out[t < 0].any()
    assert not correct.any()
    again = K.linear_xent(x, w, t)
    assert K.linear_xent_take_error() == 0 and all(torch.equal(a, b) for a, b in zip(again, want))
