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


def test_frozen_head_keeps_small_probabilities():
    """Gradients through a frozen fp16 head: hidden rows that pick single columns make the logits exact.
    One token stands far above the others, whose probabilities of about 2e-9 are below fp16's
    smallest number, and the teacher agrees; the upstream gradient (a loss scale) makes up for it.
    The logits' gradient times 2^14 is rounded to fp16: 2^-11 of itself, or 2^-25, half a subnormal
    step, of 2^-14; the product adds V / 16 + 16 terms of 2 u (tensor cores, as in test_gpu_distill);
    the result, times g, is rounded once."""
    from zotitan_b200.losses import head_distill
    V, d, T = 4096, 64, 1.0
    gen = torch.Generator(device="cuda").manual_seed(26)
    w = torch.randn(V, 2 * d, device="cuda", generator=gen) * 0.5     # the first half makes the logits,
    w[:, :d] -= 5
    w[:, d:] += 1                                                     # the second sees their gradient,
    w[17, :d], w[17, d:] = 15.0, 0.0                                  # but for the high token's
    w = w.half()
    x = torch.eye(d, 2 * d, device="cuda").half().requires_grad_()
    idx = torch.tensor([[17, -1]], device="cuda").expand(d, 2)
    val = torch.zeros(d, 2, device="cuda")
    g = torch.full((d,), 32768.0, device="cuda")
    e = Exact(w[:, :d].t(), idx, val, T)
    dz, tol = e.grad(g)
    assert float(e.q.median()) < 3e-9
    want = dz @ w.double()
    wa = w.double().abs()
    tol = (tol + 2 ** -11 * dz.abs() + 2 ** -25 * 2 ** -14 * g.double()[:, None]) @ wa
    tol = tol + (V / 16 + 16) * 2 * U * (dz.abs() @ wa)
    assert float((tol / want.abs())[:, d:].max()) < 1e-2              # the second half tells
    loss, _ = head_distill(x, idx, val, w, chunk_rows=48)
    got, = torch.autograd.grad(loss, x, g)
    close(got, want, tol, torch.float16)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_frozen_head_rounds_the_result_once(dt):
    """Upstream gradients that are no powers of two: the hidden gradient is the fp32 product of the
    logits' rounded gradient with the head (1000 terms: (V / 16 + 16) 2 u on tensor cores, V u
    elsewhere), times g (u, and u of the product's own store), rounded once to the hidden type."""
    from zotitan_b200 import kernels as K
    from zotitan_b200.losses import head_distill
    dtype, V = DTYPES[dt], 1000
    x, w, idx, val = operands(300, V, 128, 16, seed=27)
    x, w = x.to(dtype), w.to(dtype)
    g = torch.rand(300, device="cuda") + 0.5
    leaf = x.detach().requires_grad_()
    loss, _ = head_distill(leaf, idx, val, w, chunk_rows=128)
    got, = torch.autograd.grad(loss, leaf, g)
    dz = torch.cat([K.distill_rows_grad(F.linear(c, w), i, v, torch.ones(len(c), device="cuda"))[2]
                    for c, i, v in zip(x.split(128), idx.split(128), val.split(128))]).double()
    want = dz @ w.double() * g.double()[:, None]
    terms = dz.abs() @ w.double().abs() * g.double()[:, None]
    adds = V * U if dt == "f32" else (V / 16 + 16) * 2 * U
    close(got, want, adds * terms + 2 * U * want.abs(), dtype)


@pytest.mark.parametrize("how", ["bias", "autocast"])
def test_z_loss_where_the_logits_are_kept(how):
    """The z-loss is refused only where the frozen head drops the logits: with a trained bias, and under
    autocast, it has its gradient."""
    from test_gpu_distill import model_with_head_norms, teacher_batch
    from zotitan_b200.losses import distill_xentropy
    m = model_with_head_norms(seed=30, layers=1).float()
    for p in m.parameters():
        p.requires_grad_(False)
    wq = m.model.layers[0].self_attn.q_norm.weight.requires_grad_(True)
    batch = teacher_batch(2, 16, 10, seed=31)
    params = [wq]
    if how == "bias":
        head = torch.nn.Linear(256, 1000, device="cuda")
        head.weight.data.copy_(m.lm_head.weight)
        head.weight.requires_grad_(False)
        m.lm_head = head
        params.append(head.bias)
    import contextlib
    with torch.autocast("cuda", torch.bfloat16) if how == "autocast" else contextlib.nullcontext():
        loss, z, _ = distill_xentropy(m, batch, 1.0, z_loss_weight=1e-2)
        grads = torch.autograd.grad(loss + z, params)
        alone = torch.autograd.grad(distill_xentropy(m, batch, 1.0)[0], params)
    assert all(torch.isfinite(t).all() for t in grads) and not torch.equal(grads[-1], alone[-1])
    frozen = m.lm_head
    if how == "bias":
        frozen.bias.requires_grad_(False)
    with pytest.raises(NotImplementedError):
        distill_xentropy(m, batch, 1.0, z_loss_weight=1e-2)


# an odd and an even number of accumulators a tile, whole and partial last ones, several row tiles
@pytest.mark.parametrize("R,V,k,top,T", [(300, 1537, 1088, 40, 1.0), (300, 1537, 2112, 64, 2.0), (600, 4097, 3136, 16, 1.0),
                                         (257, 700, 2048, 256, 0.7)])
def test_head_of_several_accumulators(R, V, k, top, T):
    """Tolerances as in test_gpu_distill.test_linear."""
    from zotitan_b200 import kernels as K
    x, w, idx, val = operands(R, V, k, top, seed=24)
    loss, lse = K.linear_distill(x, w, idx, val, T)
    assert K.linear_distill_take_error() == 0
    e = Exact(x.double() @ w.double().t(), idx, val, T)
    ez = (k / 16 + 16) * 2 * U * (x.double().abs() @ w.double().abs().t()).amax(1)
    close(loss, e.loss, e.tol_loss + 2 * T * ez, torch.float32)
    close(lse, e.lse, e.tol_lse + ez / T, torch.float32)


def test_pieces_of_k_are_added_in_fp32():
    """A logit of K 8192 is the sum of its eight pieces of 1024, rounded to nearest as they are added:
    with a vocabulary of one, lse is the logit. Each lse is rounded four times (the base's product with
    log2 e, that with ln 2, both constants: 4 u of it) and seven adds round once: (4 + 4 + 7) u of the
    logit, u = 2^-24. One accumulator for all of K would truncate at each of its 512 steps, a third of
    u of the logit every time, where the pieces lose an eighth of that: 150 u apart."""
    from zotitan_b200 import kernels as K
    g = torch.Generator(device="cuda").manual_seed(25)
    R, k = 300, 8192
    x = (torch.rand(R, k, device="cuda", generator=g) + 0.5).bfloat16()
    w = (torch.rand(1, k, device="cuda", generator=g) + 0.5).bfloat16()
    idx, val = torch.zeros(R, 1, dtype=torch.int64, device="cuda"), torch.zeros(R, 1, device="cuda")
    whole = K.linear_distill(x, w, idx, val)[1].double()
    pieces = sum(K.linear_distill(x[:, j:j + 1024].contiguous(), w[:, j:j + 1024].contiguous(), idx, val)[1].double()
                 for j in range(0, k, 1024))
    assert float(((whole - pieces).abs() / pieces).max()) <= 15 * U


def c_args(z, idx, val, T, grad, weight=None, weight_lse=None, loss=None, lse=None, stats=None):
    from zotitan_b200 import _lib as L
    a = L.ZtDistillArgs()
    a.logits, a.grad, a.top_idx, a.top_logits = z.data_ptr(), grad.data_ptr(), idx.data_ptr(), val.data_ptr()
    for name, t in (("weight", weight), ("weight_lse", weight_lse), ("loss", loss), ("lse", lse), ("stats", stats)):
        if t is not None:
            setattr(a, name, t.data_ptr())
    a.rows, a.vocab, a.ld, a.ld_grad = *z.shape, z.stride(0), grad.stride(0)
    a.dtype = {torch.float32: L.ZT_F32, torch.bfloat16: L.ZT_BF16, torch.float16: L.ZT_F16}[z.dtype]
    a.top, a.idx_bits, a.top_dtype, a.temperature = idx.shape[1], 64, L.ZT_F32, T
    return a


# a warp a row, a CTA a row (narrow and wide), a cluster of CTAs a row
@pytest.mark.parametrize("dt,rows,vocab,shift", [("bf16", 1500, 1003, 1), ("f32", 700, 8192, 0), ("f16", 320, 70001, 1), ("bf16", 9, 50257, 3)])
def test_c_entry_points_beyond_the_wrappers(dt, rows, vocab, shift):
    """zt_distill_rows_grad with a gradient of lse and with stats for a later backward, and
    zt_distill_rows_backward in place."""
    from zotitan_b200 import _lib as L
    lib, dtype, T = L.load(), DTYPES[dt], 2.0
    z, idx, val = make(rows, vocab, 33, dtype, T, ld=vocab + 5, seed=28, shift=shift)
    idx, val = idx.contiguous(), val.contiguous()
    gen = torch.Generator(device="cuda").manual_seed(29)
    g, gl = (torch.rand(rows, device="cuda", generator=gen) * 64 + 0.5 for _ in range(2))
    stream = torch.cuda.current_stream().cuda_stream
    e = Exact(z, idx, val, T)
    want, tol = e.grad(g, gl)
    loss, lse = (torch.empty(rows, device="cuda") for _ in range(2))
    stats = torch.empty(rows, 2, device="cuda")
    one = torch.empty_like(z)
    assert lib.zt_distill_rows_grad(ctypes.byref(c_args(z, idx, val, T, one, g, gl, loss, lse, stats)), stream) == L.ZT_OK
    close(one, want, tol, dtype)
    close(loss, e.loss, e.tol_loss, torch.float32)
    close(lse, e.lse, e.tol_lse, torch.float32)
    two = torch.empty_like(z)
    assert lib.zt_distill_rows_backward(ctypes.byref(c_args(z, idx, val, T, two, g, gl, stats=stats)), stream) == L.ZT_OK
    close(two, want, tol, dtype)
    gap = torch.as_strided(z, (rows - 1, 5), (z.stride(0), 1), z.storage_offset() + vocab).clone()
    assert lib.zt_distill_rows_backward(ctypes.byref(c_args(z, idx, val, T, z, g, gl, stats=stats)), stream) == L.ZT_OK
    close(z, want, tol, dtype)
    assert torch.equal(torch.as_strided(z, (rows - 1, 5), (z.stride(0), 1), z.storage_offset() + vocab), gap)   # behind each row
    # a gradient of lse alone
    z2, _, _ = make(rows, vocab, 33, dtype, T, ld=vocab + 5, seed=28, shift=shift)
    want, tol = e.grad(None, gl)
    assert lib.zt_distill_rows_backward(ctypes.byref(c_args(z2, idx, val, T, two, None, gl, stats=stats)), stream) == L.ZT_OK
    close(two, want, tol, dtype)
