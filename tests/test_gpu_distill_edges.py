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
