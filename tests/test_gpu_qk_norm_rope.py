"""Per-head q/k RMS norm with the rotary embedding (zt_qk_norm_rope) on the GPU.

Against the formula in 64 bits, with tolerances counted from the kernel's roundings
(u = 2^-24, one fp32 rounding; h = eps / 2 of the output type, its one rounding):

- forward: out = y cos -+ y' sin with y = x n w. n: hd squares in chains of at most 16 with 5
  adds across lanes, halved by the root (11 u), rsqrtf (2 ulp = 4 u); three products and
  the last add (4 u). So |error| <= 32 u (|y cos| + |y' sin|) + h |out|.
- dx = n (w dy - x m), m = n^2 mean(w dy x): w dy carries 4 u of (|g cos| + |g' sin|) |w|, the
  mean 2 * 16 + 5 + 6 u of the sum of magnitudes, n^2 30 u: 96 u of
  n (|w| d + |x| n^2 mean(|w| d |x|)), d = |g cos| + |g' sin|, plus h.
- dw = sum of N products with relative errors of at most 32 u, added in chains of at most N:
  (N + 64) u of the sum of d |x| n, plus h.

fp16 outputs may be subnormal: 2^-25 absolute, half their step.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-38


def rotate(x):
    a, b = x.chunk(2, -1)
    return torch.cat((-b, a), -1)


def unrotate(x):
    a, b = x.chunk(2, -1)
    return torch.cat((b, -a), -1)


def exact(x, w, cos, sin, g=None, eps=1e-6):
    """out, and with g its tolerance scale and (dx, dw) with theirs, in 64 bits; x [B, T, H, hd]."""
    x, w, cos, sin = x.detach().double(), w.detach().double(), cos.double(), sin.double()
    cos, sin = (t.reshape(-1, *t.shape[-2:]).unsqueeze(2) for t in (cos, sin))
    n = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = x * n * w
    out = y * cos + rotate(y) * sin
    scale = (y * cos).abs() + (rotate(y) * sin).abs()
    if g is None:
        return out, scale
    g = g.double()
    dy = g * cos + unrotate(g * sin)
    d = (g * cos).abs() + unrotate(g * sin).abs()
    wd = w * dy
    dx = n * (wd - x * n.square() * (wd * x).mean(-1, keepdim=True))
    sx = n * (w.abs() * d + x.abs() * n.square() * (w.abs() * d * x.abs()).mean(-1, keepdim=True))
    dw = (dy * x * n).sum((0, 1, 2))
    sw = (d * x.abs() * n).sum((0, 1, 2))
    return out, scale, dx, sx, dw, sw


def close(got, want, tol, dtype):
    err = (got.double() - want).abs()
    bad = err - (tol + half(dtype) * want.abs() * (1 + 2 ** -8) + tiny(dtype))
    assert got.dtype == dtype
    assert not torch.isnan(got).any()
    assert float(bad.max()) <= 0, f"off by {float(err.max())}, {float(bad.max())} over the tolerance"


def make(B, T, hq, hk, hd, dtype, layout="plain", tables="shared", side="same", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if layout == "packed":            # slices of a fused projection
        row = rand(B, T, (hq + 2 * hk) * hd).to(dtype)
        q = row[..., :hq * hd].unflatten(-1, (hq, hd))
        k = row[..., hq * hd:(hq + hk) * hd].unflatten(-1, (hk, hd))
    elif layout == "head_major":      # [B, H, T, hd] storage
        q, k = rand(B, hq, T, hd).to(dtype).transpose(1, 2), rand(B, hk, T, hd).to(dtype).transpose(1, 2)
    elif layout == "shifted":         # storage that starts one element off its alignment
        q = rand(B * T * hq * hd + 1).to(dtype)[1:].view(B, T, hq, hd)
        k = rand(B * T * hk * hd + 1).to(dtype)[1:].view(B, T, hk, hd)
    elif layout == "strided":         # heads whose elements are not adjacent
        q, k = rand(B, T, hq, hd, 2).to(dtype)[..., 0], rand(B, T, hk, hd, 2).to(dtype)[..., 0]
    elif layout == "expanded":        # one batch entry seen B times
        q, k = rand(1, T, hq, hd).to(dtype).expand(B, -1, -1, -1), rand(1, T, hk, hd).to(dtype).expand(B, -1, -1, -1)
    else:
        q, k = rand(B, T, hq, hd).to(dtype), rand(B, T, hk, hd).to(dtype)
    other = torch.float32 if side == "f32" else dtype
    start = torch.randint(0, 5000, (B if tables == "batch" else 1, 1), device="cuda", generator=g).double()
    pos = start + torch.arange(T, device="cuda")
    ang = (pos[..., None] * 10000.0 ** (-torch.arange(0, hd, 2, device="cuda").double() / hd)).repeat(1, 1, 2)
    cos, sin = ang.cos().to(other), ang.sin().to(other)
    wq, wk = (1 + 0.3 * rand(hd)).to(other), (1 + 0.3 * rand(hd)).to(other)
    gq, gk = rand(B, hq, T, hd).to(dtype).transpose(1, 2), rand(B, hk, T, hd).to(dtype)
    return q, k, wq, wk, cos, sin, gq, gk.transpose(1, 2)


CASES = [
    (1, 1, 32, 8, 128, "bf16", "plain", "shared", "same"),
    (1, 1, 1, 1, 2, "f32", "plain", "shared", "same"),
    (2, 37, 5, 1, 64, "f16", "packed", "batch", "same"),
    (3, 11, 4, 2, 80, "f32", "head_major", "batch", "same"),
    (1, 7, 3, 3, 6, "bf16", "plain", "shared", "same"),
    (2, 5, 7, 2, 50, "bf16", "plain", "shared", "f32"),
    (1, 9, 2, 2, 512, "f32", "packed", "shared", "same"),
    (1, 9, 2, 1, 512, "bf16", "packed", "shared", "same"),
    (1, 300, 32, 8, 128, "bf16", "packed", "shared", "same"),
    (2, 3, 1, 1, 256, "f16", "plain", "shared", "f32"),
    (2, 65, 6, 2, 96, "bf16", "shifted", "batch", "same"),
    (2, 4, 3, 1, 160, "f32", "shifted", "shared", "same"),
    (2, 17, 15, 3, 80, "bf16", "strided", "shared", "same"),
    (3, 13, 4, 4, 64, "f16", "expanded", "shared", "same"),
    (2, 21, 9, 3, 72, "bf16", "plain", "batch", "f32"),
    (1, 2500, 2, 1, 64, "bf16", "plain", "shared", "same"),
]
IDS = ["-".join(str(v) for v in c) for c in CASES]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward(case):
    from zotitan_b200 import kernels as K
    B, T, hq, hk, hd, dt, layout, tables, side = case
    dtype = DTYPES[dt]
    q, k, wq, wk, cos, sin, _, _ = make(B, T, hq, hk, hd, dtype, layout, tables, side, seed=hd + T)
    keep = q.clone(), k.clone()
    qo, ko = K.qk_norm_rope(q, k, wq, wk, cos, sin)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        want, scale = exact(x, w, cos, sin)
        assert got.shape == x.shape and got.is_contiguous()
        close(got, want, 32 * U * scale, dtype)
    assert torch.equal(q, keep[0]) and torch.equal(k, keep[1])


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_backward(case):
    from zotitan_b200 import kernels as K
    B, T, hq, hk, hd, dt, layout, tables, side = case
    dtype = DTYPES[dt]
    q, k, wq, wk, cos, sin, gq, gk = make(B, T, hq, hk, hd, dtype, layout, tables, side, seed=hd + T)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    qo, ko = K.qk_norm_rope(*leaves, cos, sin)
    grads = torch.autograd.grad((qo, ko), leaves, (gq, gk))
    for x, w, g, dx, dw, heads in ((q, wq, gq, grads[0], grads[2], hq), (k, wk, gk, grads[1], grads[3], hk)):
        _, _, want, sx, wantw, sw = exact(x, w, cos, sin, g)
        close(dx, want, 96 * U * sx, dtype)
        close(dw, wantw, (B * T * heads + 64) * U * sw, w.dtype)
    again = torch.autograd.grad(K.qk_norm_rope(*leaves, cos, sin), leaves, (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))   # sums in a fixed order


def test_backward_against_differences():
    """d/ds of <out(x + s d), g> by central differences of the 64-bit formula: step 2^-10 leaves
    a truncation of about 1e-6 of the sum's scale, far above the fp32 kernel's error."""
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, gq, gk = make(2, 9, 4, 2, 64, torch.float32, seed=4)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(K.qk_norm_rope(*leaves, cos, sin), leaves, (gq, gk))
    gen = torch.Generator(device="cuda").manual_seed(9)
    for i, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, device="cuda", generator=gen, dtype=torch.float64)
        x, w, g = (q, wq, gq) if i in (0, 2) else (k, wk, gk)

        def value(s):
            a, b = (x.double() + s * d, w.double()) if i < 2 else (x.double(), w.double() + s * d)
            return float((exact(a, b, cos, sin)[0] * g.double()).sum())

        h = 2.0 ** -10
        want = (value(h) - value(-h)) / (2 * h)
        got = float((grads[i].double() * d).sum())
        scale = float((grads[i].double() * d).abs().sum())
        assert abs(got - want) <= 1e-5 * scale


def test_only_some_gradients():
    """Frozen weights, or only one of q and k: the others' gradients stay the same."""
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, gq, gk = make(2, 9, 4, 2, 64, torch.bfloat16, seed=5)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    want = torch.autograd.grad(K.qk_norm_rope(*leaves, cos, sin), leaves, (gq, gk))
    for i in range(4):
        ins = [t.detach() for t in (q, k, wq, wk)]
        ins[i].requires_grad_()
        got, = torch.autograd.grad(K.qk_norm_rope(*ins, cos, sin), ins[i], (gq, gk))
        assert torch.equal(got, want[i])
    qo, _ = K.qk_norm_rope(*leaves, cos, sin)       # k's output takes no part
    dq, dk = torch.autograd.grad(qo, leaves[:2], gq)
    assert torch.equal(dq, want[0]) and not dk.any()


@pytest.mark.parametrize("layout", ["plain", "packed", "head_major", "shifted"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_in_place(layout, dt):
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, _, _ = make(3, 19, 6, 2, 64, DTYPES[dt], layout, "batch", seed=6)
    want = K.qk_norm_rope(q, k, wq, wk, cos, sin)
    rest = None
    if layout == "packed":
        rest = q._base[..., 8 * 64:].clone()
    version = q._version
    got = K.qk_norm_rope_(q, k, wq, wk, cos, sin)
    assert got[0] is q and got[1] is k and q._version > version
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    if rest is not None:
        assert torch.equal(q._base[..., 8 * 64:], rest)    # the values beside them


def test_unbatched_and_empty():
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, _, _ = make(1, 23, 4, 2, 64, torch.bfloat16, seed=7)
    want = K.qk_norm_rope(q, k, wq, wk, cos, sin)
    got = K.qk_norm_rope(q[0], k[0], wq, wk, cos[0], sin[0])
    assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[1][0]) and got[0].dim() == 3
    e = q[:, :0].detach().requires_grad_()
    w = wq.detach().requires_grad_()
    qo, ko = K.qk_norm_rope(e, k[:, :0], w, wk, cos[:, :0], sin[:, :0])
    assert qo.shape == (1, 0, 4, 64) and ko.shape == (1, 0, 2, 64)
    de, dw = torch.autograd.grad(qo, (e, w), qo.detach())
    assert de.shape == e.shape and not dw.any()


def test_zero_heads_and_heads_apart():
    """A head of zeros gives zeros and finite gradients; a head with an infinity or a NaN
    touches no other head."""
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, gq, gk = make(2, 9, 4, 2, 128, torch.bfloat16, seed=8)
    q[0, 3, 1] = 0
    want = K.qk_norm_rope(q, k, wq, wk, cos, sin)
    assert not want[0][0, 3, 1].any()
    leaf = q.detach().requires_grad_()
    dq, = torch.autograd.grad(K.qk_norm_rope(leaf, k, wq, wk, cos, sin)[0], leaf, gq)
    assert torch.isfinite(dq).all()
    bad = q.clone()
    bad[1, 4, 2, 7], bad[0, 0, 0, 100] = float("inf"), float("nan")
    got = K.qk_norm_rope(bad, k, wq, wk, cos, sin)
    keep = torch.ones(q.shape[:3], dtype=torch.bool, device="cuda")
    keep[1, 4, 2] = keep[0, 0, 0] = False
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1], want[1])
    assert torch.isnan(got[0][0, 0, 0]).all()


def test_another_stream_and_graph():
    """On a side stream, and captured: replays read the current inputs, forward and backward."""
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, gq, gk = make(2, 33, 8, 2, 128, torch.bfloat16, seed=10)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]

    def step():
        out = K.qk_norm_rope(*leaves, cos, sin)
        return *out, *torch.autograd.grad(out, leaves, (gq, gk))

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = [t.detach() for t in step()]
        graphs.append((graph, out))
    new = torch.randn(q.shape, device="cuda").bfloat16()
    with torch.no_grad():
        leaves[0].copy_(new)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = step()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, _, _ = make(2, 9, 4, 2, 64, torch.bfloat16, seed=11)
    for args in [(q, k[:, :8], wq, wk, cos, sin), (q, k.float(), wq, wk, cos, sin), (q.double(), k.double(), wq, wk, cos, sin),
                 (q[..., :63], k[..., :63], wq[:63], wk[:63], cos[..., :63], sin[..., :63]),
                 (q, k, wq[:32], wk, cos, sin), (q, k, wq.half(), wk.half(), cos, sin), (q, k, wq, wk.float(), cos, sin),
                 (q, k, wq, wk, cos[:, :8], sin[:, :8]), (q, k, wq, wk, cos, sin.float()), (q, k, wq, wk, cos.expand(3, -1, -1), sin.expand(3, -1, -1)),
                 (q[0, 0], k[0, 0], wq, wk, cos, sin), (q, k[:, :, :0], wq, wk, cos, sin), (q, k.cpu(), wq, wk, cos, sin),
                 (q, k, wq, wk, cos.float().requires_grad_(), sin.float())]:
        with pytest.raises(ValueError):
            K.qk_norm_rope(*args)
    with pytest.raises(ValueError, match="overlap"):
        K.qk_norm_rope_(q, q, wq, wk, cos, sin)
    with pytest.raises(ValueError, match="overlap"):
        K.qk_norm_rope_(q[:, :, :2], q[:, :, 1:3], wq, wk, cos, sin)
    # every stride holds a position's q and k, but a position of one batch row reaches another's k
    store = torch.zeros(4096, dtype=torch.bfloat16, device="cuda")
    lying = [store.as_strided((2, 2, 1, 64), (192, 128, 64, 1), at) for at in (0, 64)]
    with pytest.raises(ValueError, match="overlap"):
        K.qk_norm_rope_(*lying, wq, wk, cos[:, :2], sin[:, :2])
    K.qk_norm_rope_(q[:, :, :2], q[:, :, 2:], wq, wk, cos, sin)
    with pytest.raises(ValueError, match="twice"):
        K.qk_norm_rope_(q[:1].expand(2, -1, -1, -1), k, wq, wk, cos, sin)
    with pytest.raises(ValueError, match="differentiable"):
        K.qk_norm_rope_(q, k, wq.detach().requires_grad_(), wk, cos, sin)


def test_far_elements():
    """Positions whose elements lie beyond 2^31, read, written in place and differentiated."""
    from zotitan_b200 import kernels as K
    step = (1 << 30) + 64
    q, k, wq, wk, cos, sin, gq, gk = make(1, 3, 4, 2, 64, torch.bfloat16, seed=12)
    store = torch.empty(3 * step, dtype=torch.bfloat16, device="cuda")
    fq = store.as_strided((1, 3, 4, 64), (0, step, 64, 1))
    fk = store.as_strided((1, 3, 2, 64), (0, step, 64, 1), 4096)
    fq.copy_(q), fk.copy_(k)
    want = K.qk_norm_rope(q, k, wq, wk, cos, sin)
    got = K.qk_norm_rope(fq, fk, wq, wk, cos, sin)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a, b = q.detach().requires_grad_(), fq.detach().requires_grad_()
    grads = [torch.autograd.grad(K.qk_norm_rope(x, y, wq, wk, cos, sin)[0], x, gq)[0] for x, y in ((a, k), (b, fk))]
    assert torch.equal(*grads)
    K.qk_norm_rope_(fq, fk, wq, wk, cos, sin)
    assert torch.equal(fq, want[0]) and torch.equal(fk, want[1])


def test_differentiable_once():
    from zotitan_b200 import kernels as K
    q, k, wq, wk, cos, sin, gq, _ = make(1, 5, 2, 1, 64, torch.float32, seed=13)
    leaf = q.detach().requires_grad_()
    plain, = torch.autograd.grad(K.qk_norm_rope(leaf, k, wq, wk, cos, sin)[0], leaf, gq)
    dq, = torch.autograd.grad(K.qk_norm_rope(leaf, k, wq, wk, cos, sin)[0], leaf, gq, create_graph=True)
    assert torch.equal(dq, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), leaf)


def test_two_at_once():
    """The same weights and tables on two streams at the same time."""
    from zotitan_b200 import kernels as K
    cases = [make(4, 64, 8, 2, 128, torch.bfloat16, seed=s) for s in (14, 15)]
    want = []
    for q, k, wq, wk, cos, sin, gq, gk in cases:
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        want.append(torch.autograd.grad(K.qk_norm_rope(*leaves, cos, sin), leaves, (gq, gk)))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (q, k, wq, wk, cos, sin, gq, gk) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
                got[i].append(torch.autograd.grad(K.qk_norm_rope(*leaves, cos, sin), leaves, (gq, gk)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in (0, 1) for g in got[i] for a, b in zip(g, want[i]))
