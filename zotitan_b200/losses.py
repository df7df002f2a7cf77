"""Cross-entropy scorers over the model's LM head (zotitan/losses.py).

``get_xentropy(fused)`` picks the scorer as the reference does (zotitan/losses.py:7-15):
``fused=True`` -> ``fused_xentropy``: the decoder's hidden states and ``zt_linear_xent``, the
lm_head GEMM on the tensor cores with the per-row loss, logsumexp and first argmax kept in
its epilogue so no logit reaches HBM, in place of the Liger fused linear cross-entropy
(zotitan/losses.py:17-52); heads it cannot take (a bias, other dtypes, an inner dimension
that is not a multiple of 64) go through the lm_head GEMM in row chunks and
``zt_xent_rows`` (one CUDA read of each logits row). ``fused=False`` -> ``torch_xentropy``,
the reference's torch path (zotitan/losses.py:55-79), run eagerly. Both return
(ce, z_loss | None, extra | None) with ce and z_loss kept apart, as the reference's
contract does.

``distill_xentropy`` scores against a teacher instead of labels: each position's loss is the
divergence from the teacher's top logits there (``head_distill``). Without gradients, as the
zeroth-order losses run, the head's GEMM and the loss are one kernel (``zt_linear_distill``);
with gradients and a frozen head the logits exist one chunk of rows at a time and become their
own gradient in place (``zt_distill_rows_grad``).
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import kernels as K

IGNORE_INDEX = -100
CHUNK_ROWS = 8192


def torch_xentropy(model, batch, z_loss_weight: float, compute_accuracy: bool):
    """Full forward, CE from materialised logits, optional z-loss and accuracy
    (zotitan/losses.py:55-79). Returns (loss, z_loss | None, extra | None)."""
    out = model(**batch)
    loss = out.loss
    extra = None
    if compute_accuracy:
        logits = out.logits[:, :-1, :]
        labels = batch["labels"][:, 1:]
        mask = labels != IGNORE_INDEX
        correct = (logits.argmax(-1) == labels) & mask
        extra = {"acc": correct.sum() / mask.sum().clamp_min(1)}
    if z_loss_weight == 0.0:
        return loss, None, extra
    logits = out.logits[:, :-1, :].float()
    labels = batch["labels"][:, 1:]
    mask = labels != IGNORE_INDEX
    lse = torch.logsumexp(logits, dim=-1)
    z_loss = z_loss_weight * (lse.square() * mask).sum() / mask.sum().clamp_min(1)
    return loss, z_loss, extra


def head_xentropy(hidden: torch.Tensor, targets: torch.Tensor, weight: torch.Tensor, bias=None,
                  want_lse: bool = True, want_correct: bool = True, chunk_rows: int = CHUNK_ROWS):
    """Per-row (loss, lse, correct) of next-token CE for hidden rows [R, d] against
    targets [R] (negative = ignored), logits = bf16(hidden @ weight^T (+ bias)): the fused
    kernel (zt_linear_xent) when it takes the operands, else one chunk of rows at a time
    through the GEMM and zt_xent_rows."""
    if bias is None and K.linear_xent_supported(hidden, weight):
        return K.linear_xent(hidden, weight, targets, want_lse, want_correct)
    R = hidden.shape[0]
    dev = hidden.device
    loss = torch.empty(R, dtype=torch.float32, device=dev)
    lse = torch.empty(R, dtype=torch.float32, device=dev) if want_lse else None
    correct = torch.empty(R, dtype=torch.int32, device=dev) if want_correct else None
    for r0 in range(0, R, chunk_rows):
        r1 = min(R, r0 + chunk_rows)
        logits = F.linear(hidden[r0:r1], weight, bias)
        lo, ls, co = K.xent_rows(logits, targets[r0:r1], want_lse, want_correct)
        loss[r0:r1] = lo
        if want_lse:
            lse[r0:r1] = ls
        if want_correct:
            correct[r0:r1] = co
        del logits
    return loss, lse, correct


def fused_xentropy(model, batch, z_loss_weight: float, compute_accuracy: bool):
    """The fused scorer: decoder forward, causal shift (hidden[:, :-1] predicts
    labels[:, 1:], -100 ignored), head_xentropy. Every position is scored against the next
    label, the last one of each sequence against -100 (ignored), so the hidden states are
    read in place. Same return contract and reductions as the reference's paths:
    ce = mean CE over the unmasked positions, z_loss = z_loss_weight * mean(lse^2),
    acc = mean(argmax == label)."""
    m = getattr(model, "_orig_mod", model)
    hidden = m.get_decoder()(input_ids=batch["input_ids"], attention_mask=batch.get("attention_mask"),
                             use_cache=False).last_hidden_state
    head = m.get_output_embeddings()
    B, S, d = hidden.shape
    shift_h = hidden.reshape(-1, d)
    labels = batch["labels"]
    shift_t = torch.full((B, S), IGNORE_INDEX, dtype=torch.int64, device=labels.device)
    shift_t[:, :-1] = labels[:, 1:]
    shift_t = shift_t.reshape(-1)
    if shift_h.dtype != torch.bfloat16:
        raise NotImplementedError("the fused scorer reads bf16 logits; use fused=False for other dtypes")
    has_z = z_loss_weight != 0.0
    loss, lse, correct = head_xentropy(shift_h, shift_t, head.weight, getattr(head, "bias", None),
                                       want_lse=has_z, want_correct=compute_accuracy)
    mask = shift_t != IGNORE_INDEX
    n = mask.sum().clamp_min(1)
    ce = loss.sum() / n
    extra = {"acc": correct.sum() / n} if compute_accuracy else None
    if not has_z:
        return ce, None, extra
    z_loss = z_loss_weight * (lse.square() * mask).sum() / n
    return ce, z_loss, extra


class _FrozenHeadDistill(torch.autograd.Function):
    """head_distill through a head that is not trained: a chunk's logits turn into
    dloss_r/dlogits_r in place and then into dloss_r/dhidden_r, which the backward scales by
    each row's upstream gradient. lse is not differentiable here.

    Rounded twice, as autograd rounds it that knows the upstream gradient: the logits' gradient
    to their type, and the result to the hidden type; dloss_r/dhidden_r waits in fp32. In fp16 a
    probability below 2^-25 would vanish before a loss scale could help, so there the logits'
    gradient is taken times a power of two, the largest that keeps T (q - p), at most T, below
    fp16's 65504."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, top_idx, top_logits, temperature, chunk_rows):
        R, dev = hidden.shape[0], hidden.device
        loss = torch.empty(R, dtype=torch.float32, device=dev)
        lse = torch.empty(R, dtype=torch.float32, device=dev)
        dx = torch.empty(hidden.shape, dtype=torch.float32, device=dev)
        scale = 2.0 ** (15 - math.frexp(temperature)[1]) if hidden.dtype == torch.float16 else 1.0
        scales = torch.full((min(R, chunk_rows),), scale, dtype=torch.float32, device=dev)
        for r0 in range(0, R, chunk_rows):
            r1 = min(R, r0 + chunk_rows)
            logits = F.linear(hidden[r0:r1], weight, bias)
            loss[r0:r1], lse[r0:r1], grad = K.distill_rows_grad(logits, top_idx[r0:r1], top_logits[r0:r1], scales[:r1 - r0],
                                                                temperature, out=logits)
            if grad.dtype == torch.float32:
                torch.mm(grad, weight, out=dx[r0:r1])
            else:
                torch.mm(grad, weight, out_dtype=torch.float32, out=dx[r0:r1])
            del logits, grad
        ctx.save_for_backward(dx)
        ctx.rest = scale, hidden.dtype
        ctx.mark_non_differentiable(lse)
        return loss, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        dx, = ctx.saved_tensors
        scale, dtype = ctx.rest
        g = g if scale == 1.0 else g / scale
        return torch.mul(dx, g[:, None], out=torch.empty_like(dx, dtype=dtype)), None, None, None, None, None, None


def _drops_logits(hidden, weight, bias) -> bool:
    """Whether head_distill, with gradients, keeps no logits: a head that is not trained, outside autocast."""
    return (torch.is_grad_enabled() and hidden.requires_grad and not torch.is_autocast_enabled("cuda")
            and not weight.requires_grad and (bias is None or not bias.requires_grad))


def head_distill(hidden: torch.Tensor, top_idx: torch.Tensor, top_logits: torch.Tensor, weight: torch.Tensor, bias=None,
                 temperature: float = 1.0, chunk_rows: int = CHUNK_ROWS):
    """Per-row (loss, lse) of hidden rows [R, d] through the head against the teacher's lists
    [R, top] (kernels.distill_rows): without gradients the fused kernel (zt_linear_distill)
    when it takes the operands, which does not round the logits, else a chunk of rows at a
    time through the GEMM and zt_distill_rows. Differentiable in hidden, and in the head
    where that requires grad (then, and under autocast, the whole logits are kept, as the
    backward needs them); lse is differentiable only in that last form."""
    train_head = weight.requires_grad or (bias is not None and bias.requires_grad)
    if torch.is_grad_enabled() and (train_head or torch.is_autocast_enabled("cuda")):
        return K.distill_rows(F.linear(hidden, weight, bias), top_idx, top_logits, temperature)
    if _drops_logits(hidden, weight, bias):
        return _FrozenHeadDistill.apply(hidden, weight, bias, top_idx, top_logits, temperature, chunk_rows)
    if bias is None and K.linear_xent_supported(hidden, weight):
        return K.linear_distill(hidden, weight, top_idx, top_logits, temperature)
    R, dev = hidden.shape[0], hidden.device
    loss = torch.empty(R, dtype=torch.float32, device=dev)
    lse = torch.empty(R, dtype=torch.float32, device=dev)
    for r0 in range(0, R, chunk_rows):
        r1 = min(R, r0 + chunk_rows)
        logits = F.linear(hidden[r0:r1], weight, bias)
        loss[r0:r1], lse[r0:r1] = K.distill_rows(logits, top_idx[r0:r1], top_logits[r0:r1], temperature)
        del logits
    return loss, lse


def distill_xentropy(model, batch, temperature: float = 1.0, z_loss_weight: float = 0.0):
    """The distillation scorer: decoder forward, then head_distill of every position against
    batch["teacher_idx"], batch["teacher_logits"] [B, S, top] (the teacher's logits for the
    token after position s; index -1 or logit -inf: no entry). Positions without an entry
    (padding, the last one of a sequence) do not count. Returns (loss, z_loss | None, None)
    as the cross-entropy scorers do: loss = mean over the counted positions,
    z_loss = z_loss_weight * mean(lse^2) with lse = logsumexp(logits / temperature)."""
    m = getattr(model, "_orig_mod", model)
    hidden = m.get_decoder()(input_ids=batch["input_ids"], attention_mask=batch.get("attention_mask"),
                             use_cache=False).last_hidden_state
    head = m.get_output_embeddings()
    idx, val = batch["teacher_idx"], batch["teacher_logits"]
    if idx.dim() != 3 or idx.shape[:2] != hidden.shape[:2] or val.shape != idx.shape:
        raise ValueError("teacher_idx and teacher_logits must be [batch, positions, top]")
    hidden = hidden.reshape(-1, hidden.shape[-1])
    idx, val = idx.reshape(-1, idx.shape[-1]), val.reshape(-1, val.shape[-1])
    bias = getattr(head, "bias", None)
    if z_loss_weight != 0.0 and _drops_logits(hidden, head.weight, bias):
        raise NotImplementedError("the z-loss has no gradient through a frozen head: use z_loss_weight=0")
    loss, lse = head_distill(hidden, idx, val, head.weight, bias, temperature)
    n = ((idx >= 0) & (val != -float("inf"))).any(-1).sum().clamp_min(1)
    value = loss.sum() / n
    return value, None if z_loss_weight == 0.0 else z_loss_weight * lse.square().sum() / n, None


def get_xentropy(fused: bool, compile_mode: str | None = None):
    """The scorer for (fused, compile_mode) (zotitan/losses.py:7-15). compile_mode is
    accepted for signature compatibility; nothing on this path is compiled."""
    del compile_mode
    return fused_xentropy if fused else torch_xentropy
