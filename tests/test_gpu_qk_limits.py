"""Per-head q/k norms with rotation at the largest number of positions a call takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [16, 2])     # 16 bytes a lane, single elements
def test_most_positions(hd):
    """2^25 positions: the same heads as in calls on the first and the last sequences, forward and
    backward; one more position is refused."""
    from zotitan_b200 import _lib as L
    from zotitan_b200 import kernels as K
    B, T = 1 << 13, 1 << 12
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, gq = (torch.randn(B, T, 1, hd, device="cuda", generator=gen).bfloat16() for _ in range(2))
    k = torch.randn(B, T, 1, hd, device="cuda", generator=gen).bfloat16()
    w = torch.rand(hd, device="cuda", generator=gen).bfloat16()
    cos, sin = (torch.rand(T, hd, device="cuda", generator=gen).bfloat16() for _ in range(2))
    leaf = q.requires_grad_()
    qo, ko = K.qk_norm_rope(leaf, k, w, w, cos, sin)
    dq, = torch.autograd.grad(qo, leaf, gq)
    for part in (slice(0, 3), slice(B - 3, B)):
        some = q.detach()[part].contiguous().requires_grad_()
        a, b = K.qk_norm_rope(some, k[part], w, w, cos, sin)
        assert torch.equal(a, qo[part]) and torch.equal(b, ko[part])
        assert torch.equal(torch.autograd.grad(a, some, gq[part])[0], dq[part])
    del qo, ko, dq
    more = torch.zeros((1 << 25) + 1, 1, 2, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(L.ZtError, match="2\\^25"):
        K.qk_norm_rope(more, more, w[:2], w[:2], more[:, 0], more[:, 0])
