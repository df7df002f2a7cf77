"""Distillation from a teacher's top logits on the GPU: zt_distill_rows and its backward,
zt_distill_rows_grad, zt_linear_distill, losses.head_distill and the scorer on a model.

Against the formula in 64 bits on the same inputs. With u = 2^-24, T the temperature,
s = (z - max) / T, terms t_k = log p_k - log q_k, and V/256 + 64 a bound on the longest chain
of adds in the row's sum (a thread of 256 adds V/256 values in two chains, then the merges):

- log of the row's sum: (V/256 + 64) u, exponentials (2^-22 each, 4 u) included;
- loss: T^2 u ((V/256 + 64) + 32 sum p (|log p| + |s| + |log S|) + (64 + K) sum p (1 + |log p|) |t|):
  the second part rounds each term's pieces (products by log2 e / T, logs: at most 16 u twice),
  the third p itself (its exponent's 2 u |t_k - t_max| / T, its sum's K u, its division);
- lse: (V/256 + 64) u + 8 u |lse|;
- gradient: half a step of its type, plus u |g| T (q (V/256 + 64 + 16 (1 + |s|)) + p (K + 64) (1 + |log p|))
  (for d lse the same with |g| q / T). fp16 may be subnormal: 2^-25; fp32 exponentials below 2^-126 flush to 0.

Tensor-core logits: each of the k / 16 accumulations rounds or truncates its fp32 sum once
(2 u of at most sum |x w|), and the 16 products inside align to the largest (16 u): every
logit is within e = (k / 16 + 16) 2 u sum |x w|; loss moves by at most T (sum q e + sum p e)
<= 2 T max e, lse by max e / T.
"""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class Exact:
    """The formula in 64 bits, with the sizes the tolerances are made of."""

    def __init__(self, z, idx, val, T):
        z = z.detach().double()
        R, V = z.shape
        idx = idx.long()
        use = (idx >= 0) & (val != -math.inf)
        t = val.double().masked_fill(~use, -math.inf) / T
        self.has = use.any(1)
        t = t - t.amax(1, keepdim=True)
        p = torch.where(use, t.exp(), 0.0)
        p = torch.where(self.has[:, None], p / p.sum(1, keepdim=True), 0.0)
        logp = torch.where(p > 0, torch.log_softmax(t.masked_fill(~use, -math.inf), 1), 0.0)
        s = z / T
        m = s.amax(1, keepdim=True)
        logS = (s - m).exp().sum(1, keepdim=True).log()   # a row of the lowest values would lose it beside m
        lse = (m + logS)[:, 0]
        at = idx.clamp(0, V - 1)
        sk = (s - m).gather(1, at)
        lq = sk - logS
        term = torch.where(p > 0, logp - lq, 0.0)
        self.T, self.p, self.at, self.V, self.K = T, p, at, V, idx.shape[1]
        self.loss = torch.where(self.has, T * T * (p * term).sum(1), 0.0)
        self.lse = torch.where(self.has, lse, 0.0)
        self.q = (s - m - logS).exp()
        self.s = s - m
        chain = V / 256 + 64
        self.tol_lse = U * (chain + 8 * lse.abs())
        self.tol_loss = T * T * U * (chain + 32 * torch.where(p > 0, p * (logp.abs() + sk.abs() + logS), 0.0).sum(1)
                                     + (64 + self.K) * (p * (1 + logp.abs()) * term.abs()).sum(1))
        self.logp = logp

    def grad(self, g, g_lse=None):
        """(gradient, its tolerance before the last rounding)."""
        g = torch.zeros_like(self.loss) if g is None else g.double()
        A = g * self.T + (0.0 if g_lse is None else g_lse.double() / self.T)
        mag = g.abs() * self.T + (0.0 if g_lse is None else g_lse.double().abs() / self.T)
        d = self.q * A[:, None]
        d = d.scatter_add(1, self.at, -self.p * (g * self.T)[:, None])
        tol = self.q * mag[:, None] * (self.V / 256 + 64 + 16 * (1 + torch.nan_to_num(self.s.abs(), posinf=0.0)))
        tol = tol.scatter_add(1, self.at, self.p * (1 + self.logp.abs()) * mag[:, None] * (self.K + 64))
        zero = ~self.has[:, None]
        return d.masked_fill(zero, 0.0), U * tol.masked_fill(zero, 0.0)


def close(got, want, tol, dtype):
    small = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    half = torch.finfo(dtype).eps / 2
    assert got.dtype == dtype and not torch.isnan(got).any()
    err = (got.double() - want).abs()
    over = err - (tol + half * want.abs() * (1 + 2 ** -8) + small)
    assert float(over.max()) <= 0, f"off by {float(err.max())}, {float(over.max())} over the tolerance"


def make(R, V, K, dtype, T=1.0, ld=None, seed=0, idx_dtype=torch.int64, val_dtype=torch.float32, empty=True, scale=2.5,
         shift=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or V
    z = (torch.randn(R * ld + shift, device="cuda", generator=g) * scale).to(dtype)[shift:].view(R, ld)[:, :V]
    teacher = z.float() + torch.randn(R, V, device="cuda", generator=g)
    if K <= V:
        val, idx = torch.topk(teacher, K, dim=1)
    else:
        idx = torch.randint(0, V, (R, K), device="cuda", generator=g)
        val = teacher.gather(1, idx)
    val, idx = val.to(val_dtype), idx.to(idx_dtype)
    if empty and R > 2:
        idx[1] = -1                                   # no teacher
        val[R - 1] = -math.inf                        # none either
        val[1] = math.nan                             # not looked at
        if K > 3:
            idx[2, K // 2:] = -100                    # a short list
            val[0, 1] = -math.inf                     # an entry without mass
    return z, idx, val


# rows, vocab, K, dtype, T, row stride, first element's offset, index and value dtypes
CASES = [
    (1, 128256, 8, "bf16", 1.0, None, 0, torch.int64, torch.float32),
    (1, 1, 1, "f32", 1.0, None, 0, torch.int64, torch.float32),
    (3, 5, 256, "f32", 0.5, None, 0, torch.int32, torch.float32),
    (7, 1003, 33, "bf16", 2.0, 1008, 0, torch.int32, torch.bfloat16),
    (5, 1003, 31, "f16", 4.0, None, 0, torch.int64, torch.float16),
    (64, 50257, 256, "f16", 1.0, None, 0, torch.int64, torch.float32),
    (33, 4099, 64, "f32", 0.7, 4100, 0, torch.int64, torch.float32),
    (300, 32003, 20, "bf16", 1.0, None, 3, torch.int64, torch.float32),
    (700, 8192, 65, "bf16", 1.0, None, 0, torch.int32, torch.float32),
    (2, 70001, 100, "f32", 1.0, 70010, 1, torch.int64, torch.float32),
    (9, 2047, 7, "f16", 1.0, None, 1, torch.int64, torch.float32),
    (40, 151936, 16, "bf16", 1.0, None, 0, torch.int64, torch.float32),
    # many short rows, a warp each
    (1200, 1003, 33, "bf16", 2.0, 1008, 0, torch.int32, torch.bfloat16),
    (1300, 777, 65, "f16", 1.0, None, 3, torch.int64, torch.float32),
    (1000, 1501, 256, "f32", 0.7, 1510, 1, torch.int64, torch.float32),
    (5000, 9, 4, "bf16", 1.0, None, 0, torch.int64, torch.float32),
    # long rows, a wide CTA each
    (310, 70001, 16, "f32", 1.0, None, 0, torch.int64, torch.float32),
]
IDS = ["-".join(str(v) for v in c).replace("torch.", "") for c in CASES]


def build(case):
    R, V, K, dt, T, ld, shift, it, vt = case
    return make(R, V, K, DTYPES[dt], T, ld, seed=V + K, idx_dtype=it, val_dtype=vt, shift=shift), DTYPES[dt], T


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_rows_forward(case):
    from zotitan_b200 import kernels as K
    (z, idx, val), _, T = build(case)
    loss, lse = K.distill_rows(z, idx, val, T)
    e = Exact(z, idx, val, T)
    close(loss, e.loss, e.tol_loss, torch.float32)
    close(lse, e.lse, e.tol_lse, torch.float32)
    assert not loss[~e.has].any() and not lse[~e.has].any()


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_rows_backward(case):
    from zotitan_b200 import kernels as K
    (z, idx, val), dtype, T = build(case)
    g = torch.Generator(device="cuda").manual_seed(1)
    gl, gs = (torch.randn(z.shape[0], device="cuda", generator=g) for _ in range(2))
    leaf = z.detach().requires_grad_()
    loss, lse = K.distill_rows(leaf, idx, val, T)
    e = Exact(z, idx, val, T)
    close(loss.detach(), e.loss, e.tol_loss, torch.float32)
    for a, b in ((gl, None), (gl, gs), (None, gs)):
        outs = [o for o, w in ((loss, a), (lse, b)) if w is not None]
        got, = torch.autograd.grad(outs, leaf, [w for w in (a, b) if w is not None], retain_graph=True)
        want, tol = e.grad(a, b)
        close(got, want, tol, dtype)
        assert not got[~e.has].any()
    got, = torch.autograd.grad(loss.sum(), leaf)      # one value expanded over the rows
    want, tol = e.grad(torch.ones_like(gl))
    close(got, want, tol, dtype)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_rows_grad(case, in_place):
    from zotitan_b200 import kernels as K
    (z, idx, val), dtype, T = build(case)
    weight = torch.rand(z.shape[0], device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) + 0.5
    e = Exact(z, idx, val, T)
    base = z._base
    beside = base.clone()
    loss, lse, grad = K.distill_rows_grad(z, idx, val, weight, T, out=z if in_place else None)
    close(loss, e.loss, e.tol_loss, torch.float32)
    close(lse, e.lse, e.tol_lse, torch.float32)
    want, tol = e.grad(weight)
    close(grad, want, tol, dtype)
    assert not grad[~e.has].any()
    assert (grad is z) == in_place
    outside = torch.ones_like(base, dtype=torch.bool)  # the storage between and around the rows stays
    outside.as_strided(z.shape, z.stride(), z.storage_offset()).fill_(not in_place)
    assert torch.equal(base[outside], beside[outside])


def test_rows_backward_against_differences():
    """d/ds of the sum of g loss along a direction, by central differences of the 64-bit formula
    (step 2^-9: truncation about 1e-6 of the sum's magnitude)."""
    from zotitan_b200 import kernels as K
    z, idx, val = make(12, 501, 20, torch.float32, seed=3)
    g = torch.randn(12, device="cuda")
    leaf = z.detach().requires_grad_()
    for out in (0, 1):
        got, = torch.autograd.grad(K.distill_rows(leaf, idx, val, 2.0)[out], leaf, g)
        d = torch.randn(z.shape, device="cuda", dtype=torch.float64)
        h = 2.0 ** -9
        up, down = (Exact(z.double() + s * d, idx, val, 2.0) for s in (h, -h))
        want = float(((up.loss if out == 0 else up.lse) * g).sum() - ((down.loss if out == 0 else down.lse) * g).sum()) / (2 * h)
        terms = got.double() * d
        assert abs(float(terms.sum()) - want) <= 1e-5 * float(terms.abs().sum())


COPIES = pytest.mark.parametrize("copies", [1, 200])   # a CTA a row, and a warp a row


@COPIES
def test_repeated_index(copies):
    """The same token several times in a list: its masses add, in the loss and the gradient."""
    from zotitan_b200 import kernels as K
    z, idx, val = make(6, 1000, 70, torch.float32, seed=4, empty=False)
    idx[:, 40:] = idx[:, :30]
    idx[3] = 17
    idx[4, 1::2] = -1
    z, idx, val = (t.repeat(copies, 1) for t in (z, idx, val))
    e = Exact(z, idx, val, 1.0)
    leaf = z.detach().requires_grad_()
    loss, _ = K.distill_rows(leaf, idx, val)
    close(loss.detach(), e.loss, e.tol_loss, torch.float32)
    g = torch.rand(6 * copies, device="cuda") + 0.5
    want, tol = e.grad(g)
    got, = torch.autograd.grad(loss, leaf, g)
    close(got, want, tol, torch.float32)
    close(K.distill_rows_grad(z, idx, val, g)[2], want, tol, torch.float32)


@COPIES
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_masked_logits(dt, copies):
    """Student logits masked by -inf or the type's lowest value, teacher values likewise."""
    from zotitan_b200 import kernels as K
    dtype = DTYPES[dt]
    low = torch.finfo(dtype).min
    z, idx, val = make(8, 3000, 10, dtype, seed=5, empty=False)
    z[0, 100:2000] = low
    z[1, 5:2900] = -math.inf
    idx[0], idx[1] = torch.arange(10, device="cuda"), torch.arange(2950, 2960, device="cuda")
    z[2] = low                                        # nothing but the lowest: uniform
    val[3, 5:] = torch.finfo(torch.float32).min       # masked by value, mass underflows to 0
    val[4] = torch.finfo(torch.float32).min           # all alike: uniform
    z, idx, val = (t.repeat(copies, 1) for t in (z, idx, val))
    e = Exact(z, idx, val, 1.0)
    e.tol_lse[2::8] = U * 8 * abs(low)
    leaf = z.detach().requires_grad_()
    loss, lse = K.distill_rows(leaf, idx, val)
    close(loss.detach(), e.loss, e.tol_loss, torch.float32)
    close(lse.detach(), e.lse, e.tol_lse, torch.float32)
    g = torch.full((8 * copies,), 100.0, device="cuda")
    want, tol = e.grad(g)
    got, = torch.autograd.grad(loss, leaf, g)
    close(got, want, tol, dtype)
    close(K.distill_rows_grad(z, idx, val, g)[2], want, tol, dtype)
    assert not got[1::8, 5:2900].any()


@pytest.mark.parametrize("vocab,copies", [(5001, 1), (1501, 200)])
def test_rows_that_are_not_numbers(vocab, copies):
    """NaN and infinities stay in their rows, and rows without a teacher take none of them."""
    from zotitan_b200 import kernels as K
    z, idx, val = make(10, vocab, 12, torch.float32, seed=6, empty=False)
    ones = torch.ones(10 * copies, device="cuda")

    def both_ways():   # each entry point adds a row up in its own order; the last ten rows
        zz, ii, vv = (t.repeat(copies, 1) for t in (z, idx, val))
        leaf = zz.detach().requires_grad_()
        loss, lse = K.distill_rows(leaf, ii, vv)
        a = (loss.detach(), lse.detach(), *torch.autograd.grad(loss, leaf, ones))
        return [[t[-10:] for t in r] for r in (a, K.distill_rows_grad(zz, ii, vv, ones))]

    clean = both_ways()
    z[0, 1400] = math.nan
    z[1, 7] = math.inf
    z[2] = -math.inf
    idx[3, 4] = vocab                                 # beyond the vocabulary
    val[4, 2] = math.nan
    val[5, 0] = math.inf
    z[6, idx[6, 1]] = -math.inf                       # mass on an impossible token
    z[7] = math.nan
    idx[7] = -1                                       # no teacher: whatever the logits are
    z[8, 3], idx[8, 1:], val[8, 1:] = math.inf, -5, math.nan
    val[8, 0] = -math.inf                             # no teacher either
    for (lo, ls, gr), was in zip(both_ways(), clean):
        assert torch.isnan(lo[:6]).all() and lo[6] == math.inf
        for r in (0, 1, 2, 3):
            assert torch.isnan(ls[r]) and torch.isnan(gr[r]).all()
        for r in (4, 5):
            assert torch.isnan(gr[r]).any()
        for r in (7, 8):
            assert lo[r] == 0 and ls[r] == 0 and not gr[r].any()
        assert torch.equal(lo[9], was[0][9]) and torch.equal(gr[9], was[2][9])
        assert torch.isfinite(gr[6]).all()


def test_expanded_and_strided_logits():
    """One row seen many times, and a transposed matrix: a copy is taken."""
    from zotitan_b200 import kernels as K
    z, idx, val = make(6, 777, 9, torch.bfloat16, seed=7)
    for view in (z[:1].expand(6, -1), z.t().contiguous().t(), z.repeat(1, 2)[:, ::2]):
        want = K.distill_rows(view.contiguous(), idx, val)
        leaf = view.detach().requires_grad_()
        got = K.distill_rows(leaf, idx, val)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        grad, = torch.autograd.grad(got[0], leaf, torch.ones(6, device="cuda"))
        e = Exact(view, idx, val, 1.0)
        close(grad, *e.grad(torch.ones(6, device="cuda")), torch.bfloat16)


def test_no_rows():
    from zotitan_b200 import kernels as K
    z = torch.empty(0, 100, device="cuda", requires_grad=True)
    idx, val = torch.empty(0, 4, dtype=torch.int64, device="cuda"), torch.empty(0, 4, device="cuda")
    loss, lse = K.distill_rows(z, idx, val)
    assert loss.shape == (0,) and lse.shape == (0,)
    assert torch.autograd.grad(loss.sum(), z)[0].shape == (0, 100)
    assert K.distill_rows_grad(z.detach(), idx, val, torch.empty(0, device="cuda"))[2].shape == (0, 100)


def test_far_rows():
    """A row whose first element lies beyond 2^31."""
    from zotitan_b200 import kernels as K
    ld = (1 << 30) + 8
    store = torch.empty(3 * ld, dtype=torch.bfloat16, device="cuda")
    z = store.as_strided((3, 40000), (ld, 1))
    small, idx, val = make(3, 40000, 16, torch.bfloat16, seed=8, empty=False)
    z.copy_(small)
    w = torch.ones(3, device="cuda")
    want = K.distill_rows_grad(small, idx, val, w)
    got = K.distill_rows_grad(z, idx, val, w, out=z)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_streams_and_graphs():
    """A side stream, and two captured graphs replayed after the inputs changed."""
    from zotitan_b200 import kernels as K
    z, idx, val = make(40, 5003, 24, torch.bfloat16, seed=9)
    x = torch.randn(40, 128, device="cuda").bfloat16()
    w = (torch.randn(5003, 128, device="cuda") * 0.1).bfloat16()
    g = torch.rand(40, device="cuda")
    leaf = z.detach().requires_grad_()

    def step():
        loss, lse = K.distill_rows(leaf, idx, val)
        return [t.detach() for t in (loss, lse, *torch.autograd.grad(loss, leaf, g), *K.distill_rows_grad(leaf.detach(), idx, val, g),
                                     *K.linear_distill(x, w, idx, val))]

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = step()
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    with torch.no_grad():
        leaf.copy_(torch.randn(z.shape, device="cuda") * 3)
        x.copy_(torch.randn(x.shape, device="cuda"))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# ---- the fused head ---------------------------------------------------------------------

def operands(R, V, k, top, seed, idx_dtype=torch.int64, empty=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(R, k, device="cuda", generator=g).bfloat16()
    w = (torch.randn(V, k, device="cuda", generator=g) * (2.0 / math.sqrt(k))).bfloat16()
    idx = torch.empty(R, top, dtype=idx_dtype, device="cuda")
    val = torch.empty(R, top, device="cuda")
    for r in range(0, R, 512):
        z = (x[r:r + 512] @ w.t()).float()
        z += torch.randn(z.shape, device="cuda", generator=g)
        if top <= V:
            val[r:r + 512], i = torch.topk(z, top, dim=1)
        else:
            i = torch.randint(0, V, (z.shape[0], top), device="cuda", generator=g)
            val[r:r + 512] = z.gather(1, i)
        idx[r:r + 512] = i
    if empty and R > 2:
        idx[1], val[1] = -1, math.nan
        val[R - 1] = -math.inf
        if top > 3:
            idx[0, top // 2:] = -7
    return x, w, idx, val


LINEAR = [(1, 1, 64, 1, 1.0), (37, 1003, 256, 5, 1.0), (300, 1000, 128, 64, 2.0), (257, 5000, 64, 256, 0.7),
          (700, 4096, 320, 33, 1.0), (5, 100, 64, 200, 1.0), (1, 128256, 2048, 64, 1.0), (1100, 50257, 512, 100, 1.0)]


@pytest.mark.parametrize("R,V,k,top,T", LINEAR)
def test_linear(R, V, k, top, T):
    from zotitan_b200 import kernels as K
    x, w, idx, val = operands(R, V, k, top, seed=R + V, idx_dtype=torch.int32 if top % 2 else torch.int64)
    loss, lse = K.linear_distill(x, w, idx, val, T)
    torch.cuda.synchronize()
    assert K.linear_distill_take_error() == 0
    wd = w.double().t()
    for r in range(0, R, 256):
        rows = slice(r, r + 256)
        e = Exact(x[rows].double() @ wd, idx[rows], val[rows], T)
        ez = (k / 16 + 16) * 2 * U * (x[rows].double().abs() @ wd.abs()).amax(1)
        close(loss[rows], e.loss, e.tol_loss + 2 * T * ez, torch.float32)
        close(lse[rows], e.lse, e.tol_lse + ez / T, torch.float32)
        assert not loss[rows][~e.has].any() and not lse[rows][~e.has].any()


def test_linear_list_corners():
    """Unsorted lists, the same token many times, tokens at tile borders and at both ends of the
    vocabulary, all rows of a warp asking for one column, an index beyond the vocabulary."""
    from zotitan_b200 import kernels as K
    R, V, k = 300, 1537, 64
    x, w, idx, val = operands(R, V, k, 16, seed=3, empty=False)
    idx[:] = torch.tensor([1536, 0, 255, 256, 511, 512, 1535, 1280, 0, 7, 1536, 300, 1024, 1023, 256, 5], device="cuda")
    idx[5] = 256
    val[:, 3] = -math.inf
    idx[9, 2] = V
    loss, lse = K.linear_distill(x, w, idx, val)
    keep = torch.arange(R, device="cuda") != 9
    e = Exact((x.double() @ w.double().t())[keep], idx[keep], val[keep], 1.0)
    ez = (k / 16 + 16) * 2 * U * (x.double().abs() @ w.double().abs().t()).amax(1)[keep]
    close(loss[keep], e.loss, e.tol_loss + 2 * ez, torch.float32)
    close(lse[keep], e.lse, e.tol_lse + ez, torch.float32)
    assert torch.isnan(loss[9]) and torch.isnan(lse[9])


def test_linear_matches_rows_on_its_own_logits():
    """x rows that pick single columns make the logits exact in bf16: the fused head and
    distill_rows then see the same numbers."""
    from zotitan_b200 import kernels as K
    x, w, idx, val = operands(64, 3001, 64, 12, seed=4)
    x = torch.eye(64, device="cuda").bfloat16()
    a = K.linear_distill(x, w, idx, val)
    z = w.t().contiguous()
    b = K.distill_rows(z, idx, val)
    e = Exact(z, idx, val, 1.0)
    for got in (a, b):
        close(got[0], e.loss, e.tol_loss, torch.float32)
        close(got[1], e.lse, e.tol_lse, torch.float32)


def test_linear_wait_expiry():
    """A loader that issues nothing: the bounded wait expires, reports and leaves the context usable."""
    from zotitan_b200 import kernels as K
    x, w, idx, val = operands(40, 1000, 64, 4, seed=5)
    want = K.linear_distill(x, w, idx, val)
    assert K.linear_distill_take_error() == 0
    K.linear_distill(x, w, idx, val, test_stall_loads=True, test_wait_cycles=2_000_000)
    assert K.linear_distill_take_error() != 0
    assert K.linear_distill_take_error() == 0
    got = K.linear_distill(x, w, idx, val)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_head_distill_paths():
    """Without gradients fused, or in chunks where the fused kernel does not take the operands;
    with a frozen head the hidden gradient, with a trained one both gradients. The logits
    of all but the fused path are rounded to bf16: half a step (2^-8) of |z|, which moves the
    loss by at most 2 T max |z| 2^-8. It moves q_v by q_v (dz_v - sum q dz), at most
    q_v 2 max |z| 2^-8 (of q, not of q - p), and the gradient of the logits by |g| T times that; their
    gradient is then rounded itself (2^-8 of |dz|). Both reach the products with w or x term
    by term; the results are rounded once, and once more by the upstream gradient (2^-7)."""
    from zotitan_b200 import kernels as K
    from zotitan_b200.losses import head_distill
    R, V, k, T = 150, 2000, 128, 1.0
    x, w, idx, val = operands(R, V, k, 16, seed=6)
    z = x.double() @ w.double().t()
    e = Exact(z, idx, val, T)
    zmax = z.abs().amax(1)
    fused = head_distill(x, idx, val, w)
    assert torch.equal(fused[0], K.linear_distill(x, w, idx, val)[0])
    bias = torch.zeros(V, device="cuda").bfloat16()
    chunks = head_distill(x, idx, val, w, bias, chunk_rows=64)
    close(chunks[0], e.loss, e.tol_loss + 2 * T * zmax * 2 ** -8, torch.float32)
    g = torch.rand(R, device="cuda") + 0.5
    dz, _ = e.grad(g)
    want = dz @ w.double()
    off = 2 ** -8 * (dz.abs() + 2 * zmax[:, None] * e.q * g[:, None] * T) * e.has[:, None] * (1 + 2 ** -6)
    tol = off @ w.double().abs()
    for head_grad in (False, True):
        xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_(head_grad)
        loss, lse = head_distill(xl, idx, val, wl, chunk_rows=64)
        close(loss.detach(), e.loss, e.tol_loss + 2 * T * zmax * 2 ** -8, torch.float32)
        grads = torch.autograd.grad(loss, (xl, wl) if head_grad else (xl,), g)
        close(grads[0], want, tol + 2 ** -7 * want.abs(), torch.bfloat16)
        assert not grads[0][~e.has].any()
        if head_grad:
            wantw = dz.t() @ x.double()
            tolw = off.t() @ x.double().abs()
            close(grads[1], wantw, tolw + 2 ** -7 * wantw.abs(), torch.bfloat16)


def model_with_head_norms(seed=0, layers=2, window=None):
    from transformers import Qwen3Config, Qwen3ForCausalLM
    cfg = Qwen3Config(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=layers, num_attention_heads=6,
                      num_key_value_heads=2, head_dim=64, max_position_embeddings=256, tie_word_embeddings=False,
                      attn_implementation="sdpa")
    torch.manual_seed(seed)
    m = Qwen3ForCausalLM(cfg)
    with torch.no_grad():
        for n, p in m.named_parameters():
            p.normal_(1.0, 0.1) if "norm" in n else p.normal_(0.0, 0.05)
    return m.to("cuda", torch.bfloat16).eval()


def teacher_batch(B, S, top, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, 1000, (B, S), device="cuda", generator=g)
    val, idx = torch.topk(torch.randn(B, S, 1000, device="cuda", generator=g) * 2, top, dim=-1)
    idx[:, -1] = -1
    return {"input_ids": ids, "labels": ids.clone(), "teacher_idx": idx, "teacher_logits": val}


def test_attention_with_head_norms():
    """The fused attention against the module's own forward: the modules round five times where
    the kernel rounds once, so q and k differ by a few bf16 steps (2^-8 each) and scores, of
    size |q||k| / sqrt(hd) <= about 8 sqrt(hd) / sqrt(hd), by 8 * 6 * 2^-8 at most, the
    probabilities by as much of themselves; o_proj sums 384 values of that relative error."""
    from zotitan_b200.llama_fused import fuse_llama, unfuse_llama
    m = model_with_head_norms()
    attn = m.model.layers[1].self_attn
    x = torch.randn(3, 40, 256, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    for pos in (torch.arange(40, device="cuda")[None], torch.arange(40, device="cuda")[None] + torch.tensor([[0], [9], [100]], device="cuda")):
        pe = m.model.rotary_emb(x, pos)
        with torch.inference_mode():
            want, _ = attn(x, pe, None)
            assert fuse_llama(m) == 2 * 2 + 1 + 2 + 2 + 2 * 2   # norms (q and k among them), attentions, MLPs
            got, _ = attn(x, pe, None)
        leaf = x.detach().requires_grad_()
        trained, _ = attn(leaf, pe, None)                    # with gradients: the out-of-place form
        assert unfuse_llama(m) == 13
        scale = float(want.float().square().mean().sqrt())
        assert float((got.float() - want.float()).square().mean().sqrt()) <= 0.02 * scale
        assert torch.equal(trained.detach(), got)
        gr = torch.randn_like(trained)
        d1, = torch.autograd.grad(trained, leaf, gr)
        leaf2 = x.detach().requires_grad_()
        d2, = torch.autograd.grad(attn(leaf2, pe, None)[0], leaf2, gr)
        s2 = float(d2.float().square().mean().sqrt())
        assert float((d1.float() - d2.float()).square().mean().sqrt()) <= 0.03 * s2


def test_criterion_zeroth_and_first_order():
    """The operators together, as they are used: a model with q/k norms scored against a
    teacher without gradients (ZOOptimizer's losses) and with them (adapters' gradients)."""
    from zotitan_b200.llama_fused import fuse_llama
    from zotitan_b200.objective import CrossEntropyCriterion, DistillationCriterion, RubricObjective
    from zotitan_b200.train_zo import ZOConfig, ZOOptimizer
    m = model_with_head_norms(seed=2)
    batch = teacher_batch(4, 32, 20, seed=3)
    crit = DistillationCriterion(temperature=2.0, z_loss_weight=1e-3)
    fuse_llama(m)
    with torch.inference_mode():
        value, metrics = crit(m, batch)
        logits = m(input_ids=batch["input_ids"]).logits
    e = Exact(logits.reshape(-1, 1000), batch["teacher_idx"].reshape(-1, 20), batch["teacher_logits"].reshape(-1, 20), 2.0)
    n = int(e.has.sum())
    assert n == 4 * 31
    # the model's own logits are rounded to bf16: 2^-8 |z| each
    slack = 2 * 2.0 * float(logits.float().abs().max()) * 2 ** -8
    assert abs(float(metrics["distill"]) - float(e.loss.sum() / n)) <= slack
    want_z = 1e-3 * float(e.lse.square().sum() / n)
    assert abs(float(metrics["z_loss"]) - want_z) <= 1e-3 * 2 * float(e.lse.abs().max()) * slack
    assert float(value) == float(metrics["distill"] + metrics["z_loss"])
    # first order on an adapter-like parameter, the head frozen
    for p in m.parameters():
        p.requires_grad_(False)
    w = m.model.layers[0].self_attn.q_norm.weight.requires_grad_(True)
    first, _ = DistillationCriterion(temperature=2.0)(m, batch)
    grad, = torch.autograd.grad(first, w)
    assert torch.isfinite(grad).all() and bool(grad.any())
    with pytest.raises(NotImplementedError):
        crit(m, batch)
    # and the zeroth-order step over both criteria
    obj = RubricObjective([(CrossEntropyCriterion(), 0.5), (DistillationCriterion(), 1.0)])
    cfg = ZOConfig()
    opt = ZOOptimizer([("w", w)], cfg, obj.score, total_steps=2)
    before = w.detach().clone()
    out = opt.step(m, [batch])
    assert math.isfinite(float(out["loss"])) and not torch.equal(before, w.detach())


def test_differentiable_once():
    from zotitan_b200 import kernels as K
    z, idx, val = make(4, 300, 5, torch.float32, seed=14)
    leaf = z.detach().requires_grad_()
    one = torch.ones(4, device="cuda")
    plain, = torch.autograd.grad(K.distill_rows(leaf, idx, val)[0], leaf, one)
    grad, = torch.autograd.grad(K.distill_rows(leaf, idx, val)[0], leaf, one, create_graph=True)
    assert torch.equal(grad, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), leaf)


def test_padded_batch():
    """Most rows without a teacher, their logits NaN: zeros there, the others as on their own."""
    from zotitan_b200 import kernels as K
    for dt, rows, vocab, shift in (("bf16", 400, 30001, 0), ("f32", 400, 9001, 1), ("f16", 400, 5003, 3), ("bf16", 1500, 1003, 1),
                                   ("f32", 320, 40001, 0)):
        z, idx, val = make(rows, vocab, 8, DTYPES[dt], seed=15, empty=False, shift=shift)
        w = torch.rand(rows, device="cuda")
        keep = torch.arange(rows, device="cuda") % 5 == 2
        alone = K.distill_rows_grad(z[keep].contiguous(), idx[keep], val[keep], w[keep])
        z[~keep], idx[~keep] = math.nan, -1
        leaf = z.detach().requires_grad_()
        loss, lse = K.distill_rows(leaf, idx, val)
        grad, = torch.autograd.grad(loss, leaf, w)
        one = K.distill_rows_grad(z, idx, val, w)
        for lo, ls, gr in ((loss, lse, grad), one):
            assert not lo[~keep].any() and not ls[~keep].any() and not gr[~keep].any()
        e = Exact(z[keep], idx[keep], val[keep], 1.0)
        want, tol = e.grad(w[keep])
        close(grad[keep], want, tol, DTYPES[dt])
        close(one[2][keep], want, tol, DTYPES[dt])
        close(one[0][keep], e.loss, e.tol_loss, torch.float32)
        close(alone[0], e.loss, e.tol_loss, torch.float32)


@COPIES
def test_large_biases(copies):
    """Logits far from zero: the common part cancels in loss and gradient (16-bit logits that far
    apart are exact inputs all the same)."""
    from zotitan_b200 import kernels as K
    for dt, shift in (("f32", 3000.0), ("f32", 726817.0), ("f32", 1e7), ("f32", -1e20), ("f16", -2000.0), ("bf16", 1e4), ("f32", 2e30)):
        dtype = DTYPES[dt]
        z, idx, val = make(6, 2000, 9, dtype, seed=16, empty=False)
        z, idx, val = ((t.repeat(copies, 1)) for t in ((z.float() + shift).to(dtype), idx, val))
        e = Exact(z, idx, val, 1.0)
        leaf = z.detach().requires_grad_()
        loss, lse = K.distill_rows(leaf, idx, val)
        # mc = round(m log2 e) is the same for every term; its own rounding shows in lse alone
        close(loss.detach(), e.loss, e.tol_loss, torch.float32)
        close(lse.detach(), e.lse, e.tol_lse, torch.float32)
        g = torch.full((6 * copies,), 64.0, device="cuda")
        want, tol = e.grad(g)
        got, = torch.autograd.grad(loss, leaf, g)
        close(got, want, tol, dtype)
        close(K.distill_rows_grad(z, idx, val, g)[2], want, tol, dtype)


def test_generation_with_a_cache():
    """The fused attention with a key-value cache: a prompt, then a token, against the whole
    sequence at once."""
    from zotitan_b200.llama_fused import fuse_llama
    m = model_with_head_norms(seed=4)
    ids = torch.randint(0, 1000, (2, 17), device="cuda")
    with torch.inference_mode():
        plain = m(input_ids=ids).logits[:, -1].float()
        fuse_llama(m)
        whole = m(input_ids=ids).logits[:, -1].float()
        first = m(input_ids=ids[:, :-1], use_cache=True)
        last = m(input_ids=ids[:, -1:], past_key_values=first.past_key_values, use_cache=True).logits[:, -1].float()
    scale = float(plain.square().mean().sqrt())
    for got in (whole, last):
        assert float((got - plain).square().mean().sqrt()) <= 0.05 * scale


def test_hooked_head_norms_are_left_alone():
    from zotitan_b200.llama_fused import fuse_llama
    m = model_with_head_norms(seed=5, layers=1)
    fuse_llama(m)
    seen = []
    m.model.layers[0].self_attn.q_norm.register_forward_hook(lambda *_: seen.append(1))
    with torch.inference_mode():
        m(input_ids=torch.randint(0, 1000, (1, 8), device="cuda"))
    assert seen


FIRST = """
import torch
from zotitan_b200 import kernels as K
g = torch.Generator(device="cuda").manual_seed(0)
z = torch.randn(40, 3000, device="cuda", generator=g).bfloat16()
val, idx = torch.topk(z.float(), 8, dim=1)
x, w = torch.randn(40, 64, device="cuda", generator=g).bfloat16(), torch.randn(3000, 64, device="cuda", generator=g).bfloat16()
q, k = torch.randn(2, 9, 4, 64, device="cuda", generator=g).bfloat16(), torch.randn(2, 9, 2, 64, device="cuda", generator=g).bfloat16()
wt, tab = torch.ones(64, device="cuda").bfloat16(), torch.rand(9, 64, device="cuda", generator=g).bfloat16()
weight = torch.ones(40, device="cuda")

def step():
    a, b = z.detach().requires_grad_(), q.detach().requires_grad_()
    loss, lse = K.distill_rows(a, idx, val)
    out = [loss, lse, *torch.autograd.grad(loss, a, weight), *K.distill_rows_grad(z, idx, val, weight), *K.linear_distill(x, w, idx, val)]
    rot = K.qk_norm_rope(b, k, wt, wt, tab, tab)
    return [t.detach() for t in (*out, *rot, *torch.autograd.grad(rot[0], b, torch.ones_like(rot[0])))]

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = step()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(p, r) for p, r in zip(out, step()))
print("captured first")
"""


def test_captured_before_any_other_call():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("V", [1000, 1003])
def test_gradient_room_of_one_position_a_sequence(V):
    """Rows a whole sequence apart: the gradient takes the room of its rows, not of the sequences."""
    from zotitan_b200 import kernels as K
    z, idx, val = make(4, V, 6, torch.bfloat16, seed=18, empty=False)
    whole = torch.zeros(4, 50, V, dtype=torch.bfloat16, device="cuda")
    whole[:, -1] = z
    last = whole[:, -1].detach()
    g = torch.full((4,), 64.0, device="cuda")
    e = Exact(z, idx, val, 1.0)
    want, tol = e.grad(g)
    leaf = last.clone().requires_grad_()
    loss, _ = K.distill_rows(leaf.as_strided(last.shape, (V, 1)), idx, val)
    strided = last.requires_grad_()
    loss2, _ = K.distill_rows(strided, idx, val)
    for got in (torch.autograd.grad(loss, leaf, g)[0], torch.autograd.grad(loss2, strided, g)[0],
                K.distill_rows_grad(last.detach(), idx, val, g)[2]):
        close(got, want, tol, torch.bfloat16)
        assert got.untyped_storage().nbytes() <= 4 * (V + 8) * 2


def test_refusals():
    from zotitan_b200 import kernels as K
    z, idx, val = make(8, 500, 6, torch.bfloat16, seed=12)
    w8 = torch.ones(8, device="cuda")
    for args in [(z.double(), idx, val), (z[0], idx[0], val[0]), (z, idx[:7], val[:7]), (z, idx.float(), val), (z, idx, val.double()),
                 (z, idx, val[:, :5]), (z, idx[:, :0], val[:, :0]), (z, idx.repeat(1, 50), val.repeat(1, 50)), (z[:, :0], idx, val),
                 (z, idx.cpu(), val), (z.cpu(), idx, val), (z, idx, val.detach().requires_grad_()), (z, idx, val, 0.0),
                 (z, idx, val, -1.0), (z, idx, val, math.nan), (z, idx, val, math.inf)]:
        with pytest.raises(ValueError):
            K.distill_rows(*args)
        with pytest.raises(ValueError):
            K.distill_rows_grad(args[0], args[1], args[2], w8, *args[3:])
    for kw in [dict(weight=w8[:7]), dict(weight=w8.double()), dict(weight=w8.cpu()), dict(out=z[:, :400]), dict(out=z.float()),
               dict(out=torch.empty(500, 8, dtype=torch.bfloat16, device="cuda").t()),
               dict(out=torch.empty(1, 500, dtype=torch.bfloat16, device="cuda").expand(8, -1))]:
        with pytest.raises(ValueError):
            K.distill_rows_grad(z, idx, val, **({"weight": w8} | kw))
    store = torch.zeros(8 * 500 + 4, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        K.distill_rows_grad(store[:4000].view(8, 500), idx, val, w8, out=store[4:].view(8, 500))
    out = torch.zeros(8, 500, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        K.distill_rows_grad(z.float(), idx, val, out.view(-1)[:8], out=out)
    x, w, idx, val = operands(8, 500, 64, 6, seed=13)
    for args in [(x.float(), w, idx, val), (x[:, :32], w[:, :32], idx, val), (x, w[:, :0], idx, val), (x, w, idx[:4], val[:4]),
                 (x, w, idx, val, 0.0), (x.detach().requires_grad_(), w, idx, val), (x, w, idx.cpu(), val.cpu())]:
        with pytest.raises(ValueError):
            K.linear_distill(*args)
