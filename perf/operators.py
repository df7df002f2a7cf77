"""Cases, plain forms and exact values of the decoder operators for distillation.

Four entry points of ``zotitan_b200.kernels``:

- ``qk_norm_rope``: RMS norm of every query and key head with the rotary embedding in the
  same pass, forward and backward;
- ``distill_rows``: the loss of a row of logits against a teacher's top logits, forward and
  backward (autograd);
- ``distill_rows_grad``: that loss and its gradient in one call, for row weights known
  beforehand;
- ``linear_distill``: the lm_head product and that loss together, without the logits.

``own`` picks the framework's kernels; otherwise ``run`` computes the same in elementary
torch operations, in fp32 and rounded once at the end.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6


def _qk(name, direction, batch, seq, hq, hk, hd, dtype, packed, per_sequence):
    """A query/key case: `packed` heads are slices of one fused projection's rows, `per_sequence`
    gives every sequence its own positions (left padding, continued sequences)."""
    return {"name": name, "op": "qk_norm_rope", "direction": direction, "batch": batch, "seq": seq, "hq": hq, "hk": hk,
            "hd": hd, "dtype": dtype, "packed": packed, "per_sequence": per_sequence}


def _rows(name, op, direction, rows, vocab, top, dtype, temperature):
    return {"name": name, "op": op, "direction": direction, "rows": rows, "vocab": vocab, "top": top, "dtype": dtype,
            "temperature": temperature}


def _linear(name, rows, vocab, k, top, temperature):
    return {"name": name, "op": "linear_distill", "direction": "forward", "rows": rows, "vocab": vocab, "k": k,
            "top": top, "dtype": "bf16", "temperature": temperature}


def listed():
    return [
        # one new token of one sequence: the smallest call, latency only
        _qk("qk_one_token", "forward", 1, 1, 32, 8, 128, "bf16", False, False),
        # a long prompt batch of the 8B head layout, heads cut out of a fused projection
        _qk("qk_prompt", "forward", 16, 2048, 32, 8, 128, "bf16", True, False),
        # a training batch of the 8B head layout
        _qk("qk_train", "train", 16, 512, 32, 8, 128, "bf16", False, False),
        # fp32 training with an odd batch, five queries to a key head and every sequence's own positions
        _qk("qk_train_f32_odd", "train", 5, 333, 15, 3, 80, "f32", False, True),
        # the next token of one sequence against a short teacher list
        _rows("distill_one_row", "distill_rows", "forward", 1, 128256, 8, "bf16", 1.0),
        # a first-order training step on a batch of the 128256-token vocabulary
        _rows("distill_train", "distill_rows", "train", 4096, 128256, 64, "bf16", 1.0),
        # an odd vocabulary in fp16 with a softened teacher
        _rows("distill_train_f16_odd", "distill_rows", "train", 1001, 50257, 33, "f16", 2.0),
        # one chunk of logits turned into its own gradient
        _rows("distill_grad", "distill_rows_grad", "grad", 2048, 128256, 64, "bf16", 1.0),
        # small fp32 logits
        _rows("distill_grad_f32_odd", "distill_rows_grad", "grad", 509, 32003, 20, "f32", 1.5),
        # a toy head: latency
        _linear("head_small", 37, 1003, 256, 5, 1.0),
        # the Llama-1B scorer batch: 16 x 512 positions
        _linear("head_1b", 8192, 128256, 2048, 64, 1.0),
        # 4 x 512 positions of the 8B head, a long teacher list
        _linear("head_8b", 2048, 128256, 4096, 128, 2.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "qk_norm_rope", "distill_rows", "distill_rows", "distill_rows_grad", "linear_distill",
                     "linear_distill"])
    if op == "qk_norm_rope":
        hq, hk = rng.choice([(32, 8), (15, 3), (16, 8), (8, 1), (4, 4), (7, 7)])
        hd = rng.choice([64, 80, 96, 128, 160, 256])
        direction = rng.choice(["forward", "train"])
        dtype = rng.choice(["bf16", "f16", "f32"])
        most = 32768 * 40 * 128 // ((hq + hk) * hd) // (4 if direction == "train" else 1) // (_BYTES[dtype] // 2)
        rows = _log_int(rng, 1, most)
        batch = min(rows, _log_int(rng, 1, 32))
        return _qk("", direction, batch, max(1, rows // batch), hq, hk, hd, dtype, rng.random() < 0.5, rng.random() < 0.3)
    temperature = rng.choice([0.7, 1.0, 1.0, 2.0, 4.0])
    top = _log_int(rng, 1, 256)
    if op == "linear_distill":
        rows, vocab = _log_int(rng, 1, 8192), _log_int(rng, 1000, 128256)
        most = min(4096, 8192 * 128256 * 2048 // (rows * vocab))
        k = 64 * _log_int(rng, 1, max(1, most // 64))
        return _linear("", rows, vocab, k, top, temperature)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = _log_int(rng, 1000, 151936)
    most = (4096 if op == "distill_rows" else 2048) * 128256 // vocab // (_BYTES[dtype] // 2)
    rows = _log_int(rng, 1, min(8192, most))
    direction = rng.choice(["forward", "train"]) if op == "distill_rows" else "grad"
    return _rows("", op, direction, rows, vocab, top, dtype, temperature)


def work(case):
    b = _BYTES[case["dtype"]]
    if case["op"] == "qk_norm_rope":
        rows, hd = case["batch"] * case["seq"], case["hd"]
        heads = rows * (case["hq"] + case["hk"]) * hd
        tables = 2 * (rows if case["per_sequence"] else case["seq"]) * hd
        train = case["direction"] == "train"
        # in: heads, tables, weights (and the upstream gradient); out: heads (and the gradients)
        return {"bytes": b * (heads * (4 if train else 2) + tables + hd * (4 if train else 2)),
                "flops": heads * (24 if train else 8)}
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    listed_bytes = rows * top * 12 + rows * 8   # int64 index and fp32 logit in, loss and lse out
    if case["op"] == "linear_distill":
        return {"bytes": b * (rows + vocab) * case["k"] + listed_bytes, "flops": 2.0 * rows * vocab * case["k"]}
    two = case["direction"] != "forward"        # the gradient is as large as the logits
    return {"bytes": b * rows * vocab * (2 if two else 1) + listed_bytes + (rows * 4 if two else 0),
            "flops": rows * vocab * (8 if two else 4)}


# ---- inputs ------------------------------------------------------------------------------

def _prepare_qk(case, g):
    dt = _DTYPES[case["dtype"]]
    B, T, hq, hk, hd = (case[n] for n in ("batch", "seq", "hq", "hk", "hd"))

    def rand(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if case["packed"]:
        row = rand(B, T, (hq + 2 * hk) * hd).to(dt)
        q = row[..., :hq * hd].unflatten(-1, (hq, hd))
        k = row[..., hq * hd:(hq + hk) * hd].unflatten(-1, (hk, hd))
    else:
        q, k = rand(B, T, hq, hd).to(dt), rand(B, T, hk, hd).to(dt)
    first = torch.zeros(1, 1, dtype=torch.float64, device="cuda")
    if case["per_sequence"]:
        first = torch.randint(0, 4096, (B, 1), device="cuda", generator=g).double()
    elif T == 1:
        first = torch.randint(0, 32768, (1, 1), device="cuda", generator=g).double()
    pos = first + torch.arange(T, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    angle = (pos[..., None] * freq).repeat(1, 1, 2)              # the model's rotary module: [1 or B, T, hd]
    s = {"case": case, "q": q, "k": k, "wq": (1 + 0.2 * rand(hd)).to(dt), "wk": (1 + 0.2 * rand(hd)).to(dt),
         "cos": angle.cos().to(dt), "sin": angle.sin().to(dt)}
    if case["direction"] == "train":
        for n in ("q", "k", "wq", "wk"):
            s[n] = s[n].detach().requires_grad_()
        # attention returns its gradients head-major
        s["gq"] = rand(B, hq, T, hd).to(dt).transpose(1, 2)
        s["gk"] = rand(B, hk, T, hd).to(dt).transpose(1, 2)
    return s


def _teacher_list(s, g, rows, top):
    """Rows without a teacher (the last position of each sequence, padding) and lists that end early."""
    r = torch.arange(rows, device="cuda")
    none = (r % 512 == 511) | (torch.rand(rows, device="cuda", generator=g) < 0.03) & (rows > 1)
    length = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.1,
                         torch.randint(1, top + 1, (rows,), device="cuda", generator=g), top)
    gone = none[:, None] | (torch.arange(top, device="cuda") >= length[:, None])
    s["idx"].masked_fill_(gone, -1)
    s["val"].masked_fill_(gone, -math.inf)


def _prepare_rows(case, g):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    s = {"case": case, "z": torch.empty(rows, vocab, dtype=_DTYPES[case["dtype"]], device="cuda"),
         "idx": torch.empty(rows, top, dtype=torch.int64, device="cuda"),
         "val": torch.empty(rows, top, dtype=torch.float32, device="cuda")}
    step = max(1, (1 << 27) // vocab)
    for r in range(0, rows, step):
        z = torch.randn(min(step, rows - r), vocab, device="cuda", generator=g).mul_(2.5)
        s["z"][r:r + step] = z
        # a teacher that mostly agrees with the student
        z.add_(torch.randn(z.shape, device="cuda", generator=g))
        s["val"][r:r + step], s["idx"][r:r + step] = torch.topk(z, top, dim=1)
    _teacher_list(s, g, rows, top)
    if case["direction"] == "train":
        s["z"].requires_grad_()
    if case["direction"] != "forward":
        # the mean over the rows, times the loss scale that fp16 training keeps its gradients normal with
        scale = (4096.0 if case["dtype"] == "f16" else 1.0) / rows
        s["g"] = torch.rand(rows, device="cuda", generator=g).add_(0.5).mul_(scale)
    return s


def _prepare_linear(case, g):
    rows, vocab, k, top = case["rows"], case["vocab"], case["k"], case["top"]
    x = torch.randn(rows, k, device="cuda", generator=g).bfloat16()
    w = torch.empty(vocab, k, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 27) // k)
    for v in range(0, vocab, step):
        w[v:v + step] = torch.randn(min(step, vocab - v), k, device="cuda", generator=g).mul_(2.0 / math.sqrt(k))
    s = {"case": case, "x": x, "w": w, "idx": torch.empty(rows, top, dtype=torch.int64, device="cuda"),
         "val": torch.empty(rows, top, dtype=torch.float32, device="cuda")}
    step = max(1, (1 << 27) // vocab)
    for r in range(0, rows, step):
        z = (x[r:r + step] @ w.t()).float()
        z.add_(torch.randn(z.shape, device="cuda", generator=g))
        s["val"][r:r + step], s["idx"][r:r + step] = torch.topk(z, top, dim=1)
    _teacher_list(s, g, rows, top)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "qk_norm_rope":
        return _prepare_qk(case, g)
    return _prepare_linear(case, g) if case["op"] == "linear_distill" else _prepare_rows(case, g)


# ---- plain forms ---------------------------------------------------------------------------

def _head_plain(x, w, cos, sin):
    """(normed and rotated heads, x / rms, 1 / rms) in fp32; cos and sin are [1 or B, T, 1, hd]."""
    x = x.float()
    n = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    u = x * n
    y = w.float() * u
    a, b = y.chunk(2, dim=-1)
    return y * cos + torch.cat((-b, a), dim=-1) * sin, u, n


def _head_backward_plain(gr, w, cos, sin, u, n):
    gr = gr.float()
    a, b = (gr * sin).chunk(2, dim=-1)
    dy = gr * cos + torch.cat((b, -a), dim=-1)
    dw = (dy * u).double().sum((0, 1, 2)).float()
    du = dy * w.float()
    return n * (du - u * (du * u).mean(-1, keepdim=True)), dw


def _run_qk(s):
    dt = s["q"].dtype
    cos, sin = s["cos"].float().unsqueeze(2), s["sin"].float().unsqueeze(2)
    oq, uq, nq = _head_plain(s["q"], s["wq"], cos, sin)
    ok, uk, nk = _head_plain(s["k"], s["wk"], cos, sin)
    out = {"q": oq.to(dt), "k": ok.to(dt)}
    if s["case"]["direction"] == "train":
        dq, dwq = _head_backward_plain(s["gq"], s["wq"], cos, sin, uq, nq)
        dk, dwk = _head_backward_plain(s["gk"], s["wk"], cos, sin, uk, nk)
        out |= {"dq": dq.to(dt), "dk": dk.to(dt), "dwq": dwq.to(dt), "dwk": dwk.to(dt)}
    return out


def _teacher_plain(idx, val, temperature):
    """(rows with a teacher, p, log p) of the valid entries; 0 where there is none."""
    valid = (idx >= 0) & (val > -math.inf)
    t = torch.where(valid, val.float() / temperature, -math.inf)
    has = valid.any(1, keepdim=True)
    t = t - torch.where(has, t.amax(1, keepdim=True), 0.0)
    total = torch.where(has, t.exp().sum(1, keepdim=True), 1.0)
    p = t.exp() / total
    return has, p, torch.where(p > 0, t - total.log(), 0.0)


def _distill_plain(z, idx, val, temperature):
    """(loss, lse, z / T, rows with a teacher, p) with z in fp32."""
    has, p, logp = _teacher_plain(idx, val, temperature)
    zt = z / temperature
    m = zt.amax(1, keepdim=True)
    lse = m + (zt - m).exp().sum(1, keepdim=True).log()
    at = idx.clamp_min(0)
    loss = torch.where(p > 0, p * (logp - (zt.gather(1, at) - lse)), 0.0).sum(1) * temperature ** 2
    return loss, torch.where(has, lse, 0.0)[:, 0], zt, has, p


def _run_rows(s):
    T = s["case"]["temperature"]
    z = s["z"].float()
    loss, lse, zt, has, p = _distill_plain(z, s["idx"], s["val"], T)
    out = {"loss": loss, "lse": lse}
    if s["case"]["direction"] != "forward":
        q = zt.sub_(lse[:, None]).exp_()
        q.scatter_add_(1, s["idx"].clamp_min(0), -p)
        out["grad"] = q.mul_(torch.where(has, s["g"][:, None] * T, 0.0)).to(s["z"].dtype)
    return out


def _run_linear(s):
    z = s["x"].float() @ s["w"].float().t()
    loss, lse, *_ = _distill_plain(z, s["idx"], s["val"], s["case"]["temperature"])
    return {"loss": loss, "lse": lse}


def run(s):
    case = s["case"]
    op, train = case["op"], case["direction"] == "train"
    if not own:
        with torch.no_grad():
            return _run_qk(s) if op == "qk_norm_rope" else _run_linear(s) if op == "linear_distill" else _run_rows(s)
    from zotitan_b200 import kernels as K
    if op == "qk_norm_rope":
        q, k = K.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], _EPS)
        if not train:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if op == "linear_distill":
        loss, lse = K.linear_distill(s["x"], s["w"], s["idx"], s["val"], case["temperature"])
        return {"loss": loss, "lse": lse}
    if op == "distill_rows_grad":
        loss, lse, grad = K.distill_rows_grad(s["z"], s["idx"], s["val"], s["g"], case["temperature"])
        return {"loss": loss, "lse": lse, "grad": grad}
    loss, lse = K.distill_rows(s["z"], s["idx"], s["val"], case["temperature"])
    if not train:
        return {"loss": loss, "lse": lse}
    grad, = torch.autograd.grad(loss, s["z"], s["g"])
    return {"loss": loss.detach(), "lse": lse.detach(), "grad": grad}


# ---- exact values --------------------------------------------------------------------------

def _exact_heads(x, w, cos, sin):
    x = x.detach().double().requires_grad_()
    w = w.detach().double().requires_grad_()
    h = x.shape[-1] // 2
    y = x / (x.square().mean(-1, keepdim=True) + _EPS).sqrt() * w
    out = torch.empty_like(y)
    out[..., :h] = y[..., :h] * cos[..., :h] - y[..., h:] * sin[..., :h]
    out[..., h:] = y[..., h:] * cos[..., h:] + y[..., :h] * sin[..., h:]
    return x, w, out


def _exact_qk(s):
    cos, sin = s["cos"].double().unsqueeze(2), s["sin"].double().unsqueeze(2)
    q, wq, oq = _exact_heads(s["q"], s["wq"], cos, sin)
    k, wk, ok = _exact_heads(s["k"], s["wk"], cos, sin)
    out = {"q": oq.detach(), "k": ok.detach()}
    if s["case"]["direction"] == "train":
        out["dq"], out["dwq"] = torch.autograd.grad(oq, (q, wq), s["gq"].double())
        out["dk"], out["dwk"] = torch.autograd.grad(ok, (k, wk), s["gk"].double())
    return out


def _exact_loss(z, idx, val, temperature):
    """The loss as a cross entropy less the teacher's entropy, row by row of the definition."""
    use = (idx >= 0) & torch.isfinite(val)
    t = val.double().masked_fill(~use, -math.inf) / temperature
    some = use.any(1)
    p = torch.softmax(t.masked_fill(~some[:, None], 0.0), dim=1) * use
    entropy = -torch.special.xlogy(p, p).sum(1)
    logq = torch.log_softmax(z / temperature, dim=1)
    cross = -(p * logq.gather(1, idx.clamp_min(0))).sum(1)
    lse = torch.logsumexp(z.detach() / temperature, dim=1) * some
    return temperature ** 2 * (cross - entropy), lse


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "qk_norm_rope":
        return _exact_qk(s)
    rows, T = case["rows"], case["temperature"]
    got = {"loss": [], "lse": []} | ({"grad": []} if case["direction"] != "forward" else {})
    step = max(1, (1 << 26) // case["vocab"])
    w = s["w"].double().t() if case["op"] == "linear_distill" else None
    for r in range(0, rows, step):
        z = s["x"][r:r + step].double() @ w if w is not None else s["z"][r:r + step].detach().double()
        z.requires_grad_("grad" in got)
        loss, lse = _exact_loss(z, s["idx"][r:r + step], s["val"][r:r + step], T)
        if "grad" in got:
            got["grad"].append(torch.autograd.grad(loss, z, s["g"][r:r + step].double())[0])
        got["loss"].append(loss.detach())
        got["lse"].append(lse)
    return {n: torch.cat(v) for n, v in got.items()}
