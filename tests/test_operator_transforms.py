"""Calls that a kernel launch would answer wrongly without a word are refused: inputs with a forward-mode
tangent, which the results would lose (and a tensor written in place keep), and traces, which would
hold the allocation of the outputs and no launch (CPU only: refused before any CUDA work)."""
import types

import pytest
import torch
import torch.autograd.forward_ad as fw

from zotitan_b200 import kernels as K

Q, KEY, W, TAB = torch.rand(2, 3, 4, 8), torch.rand(2, 3, 2, 8), torch.ones(8), torch.rand(3, 8)
Z, IDX, VAL, ONES = torch.rand(4, 10), torch.zeros(4, 2, dtype=torch.int64), torch.rand(4, 2), torch.ones(4)
X, HEAD = torch.rand(4, 64), torch.rand(10, 64)

CALLS = {
    "qk_norm_rope": (K.qk_norm_rope, [Q, KEY, W, W, TAB, TAB], (0, 1, 2, 3, 4, 5)),
    "qk_norm_rope_": (K.qk_norm_rope_, [Q, KEY, W, W, TAB, TAB], (0, 1, 2, 3, 4, 5)),
    "distill_rows": (K.distill_rows, [Z, IDX, VAL], (0, 2)),
    "distill_rows_grad": (lambda z, i, v, w, out: K.distill_rows_grad(z, i, v, w, out=out), [Z, IDX, VAL, ONES, Z.clone()], (0, 2, 3, 4)),
    "linear_distill": (K.linear_distill, [X, HEAD, IDX, VAL], (0, 1, 3)),
    "eggroll_rope_": (lambda q, k, c, s: K.eggroll_rope_(q, k, c, s, 3, 8), [Q.flatten(2).flatten(0, 1), KEY.flatten(2).flatten(0, 1), TAB, TAB],
                      (0, 1, 2, 3)),
}


@pytest.mark.parametrize("name,which", [(n, i) for n, c in CALLS.items() for i in c[2]])
@pytest.mark.parametrize("no_grad", [False, True])
def test_forward_mode_tangents_are_refused(name, which, no_grad):
    fn, args, _ = CALLS[name]
    with fw.dual_level(), torch.set_grad_enabled(not no_grad):
        dual = [fw.make_dual(a, torch.ones_like(a)) if i == which else a for i, a in enumerate(args)]
        with pytest.raises(ValueError, match="forward-mode"):
            fn(*dual)


@pytest.mark.parametrize("name", CALLS)
def test_a_level_without_tangents_is_no_obstacle(name):
    """What is refused there is these CPU tensors, as always."""
    fn, args, _ = CALLS[name]
    with fw.dual_level(), pytest.raises(ValueError) as e:
        fn(*args)
    assert "forward-mode" not in str(e.value)


@pytest.mark.parametrize("name", CALLS)
def test_traces_are_refused(name):
    fn, args, _ = CALLS[name]
    with torch.no_grad(), pytest.raises(ValueError, match="traced"):
        torch.jit.trace(lambda *a: fn(*a)[0], tuple(a.clone() for a in args), check_trace=False)


def test_backward_passes_refuse_tangents():
    """Forward over reverse: the upstream gradient carries the tangent."""
    qk = types.SimpleNamespace(saved_tensors=(Q, KEY, W, W, TAB, TAB), rest=(1e-6, False), needs_input_grad=(True,) * 8)
    rows = types.SimpleNamespace(saved_tensors=(Z, IDX, VAL, torch.rand(4, 2)), temperature=1.0)
    with fw.dual_level():
        for g in ((fw.make_dual(Q, Q), KEY), (Q, fw.make_dual(KEY, KEY))):
            with pytest.raises(ValueError, match="forward-mode"):
                K._qk_backward(qk, *g)
        for g in ((fw.make_dual(ONES, ONES), None), (None, fw.make_dual(ONES, ONES))):
            with pytest.raises(ValueError, match="forward-mode"):
                K._distill_backward(rows, *g)
