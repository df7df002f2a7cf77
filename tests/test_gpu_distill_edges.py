"""Distillation from a teacher's top logits, where a call must not look better than it is: an
expired wait, numbers that are none, long K, small probabilities, and the C entry points' options that
no wrapper passes."""
import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

from test_gpu_distill import DTYPES, U, Exact, close, make, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,V,k,top", [(40, 1000, 64, 4), (700, 50257, 128, 33), (2100, 8000, 2112, 16)])
def test_expired_wait_leaves_no_numbers(R, V, k, top):
    """What a call whose wait ran out could not compute is NaN, not what its workspace held: here the
    good result of the call before."""
    from zotitan_b200 import kernels as K
    x, w, idx, val = operands(R, V, k, top, seed=21)
    has = ((idx >= 0) & (val != -math.inf)).any(1)
    want = K.linear_distill(x, w, idx, val)
    assert K.linear_distill_take_error() == 0 and all(torch.isfinite(t).all() for t in want)
    got = K.linear_distill(x, w, idx, val, test_stall_loads=True, test_wait_cycles=2_000_000)
    assert K.linear_distill_take_error() != 0
    for t in got:
        assert torch.isnan(t[has]).all() and not t[~has].any()
    again = K.linear_distill(x, w, idx, val)
    assert K.linear_distill_take_error() == 0
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dt,vocab,copies", [("f32", 5001, 1), ("bf16", 1501, 200), ("f16", 40001, 1)])
def test_teacher_that_is_not_a_number(dt, vocab, copies, bad):
    """A NaN or +inf among a teacher's values makes the whole row NaN: loss, lse and every element of
    the gradient. Beside a negative index it is not looked at."""
    from zotitan_b200 import kernels as K
    z, idx, val = make(6, vocab, 40, DTYPES[dt], seed=22, empty=False)
    z, idx, val = (t.repeat(copies, 1) for t in (z, idx, val))
    ones = torch.ones(6 * copies, device="cuda")

    def both_ways():
        leaf = z.detach().requires_grad_()
        loss, lse = K.distill_rows(leaf, idx, val)
        return ((loss.detach(), lse.detach(), *torch.autograd.grad(loss, leaf, ones)), K.distill_rows_grad(z, idx, val, ones))

    clean = both_ways()
    val[1::6, 35] = bad
    val[4::6, 0] = bad
    val[3::6, 7], idx[3::6, 7] = bad, -1
    rest = torch.ones(6 * copies, dtype=torch.bool, device="cuda")
    rest[1::6] = rest[3::6] = rest[4::6] = False
    for (lo, ls, gr), was in zip(both_ways(), clean):
        for r in (1, 4):
            assert torch.isnan(lo[r::6]).all() and torch.isnan(ls[r::6]).all() and torch.isnan(gr[r::6]).all()
        assert torch.isfinite(lo[3::6]).all() and torch.equal(ls[3::6], was[1][3::6]) and torch.isfinite(gr[3::6]).all()
        assert all(torch.equal(a[rest], b[rest]) for a, b in zip((lo, ls, gr), was))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_teacher_that_is_not_a_number_in_the_head(bad):
    from zotitan_b200 import kernels as K
    x, w, idx, val = operands(300, 1537, 128, 40, seed=23, empty=False)
    clean = K.linear_distill(x, w, idx, val)
    val[5, 39] = bad
    val[299, 0] = bad
    val[7, 3], idx[7, 3] = bad, -1
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[5] = keep[7] = keep[299] = False
    for got, was in zip(K.linear_distill(x, w, idx, val), clean):
        assert torch.isnan(got[5]) and torch.isnan(got[299]) and torch.isfinite(got[7])
        assert torch.equal(got[keep], was[keep])
