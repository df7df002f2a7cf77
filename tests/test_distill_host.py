"""Host-side checks of the distillation and q/k norm entry points: what they refuse is refused
before any CUDA work (CPU only)."""
import ctypes
import math

import pytest
import torch

from zotitan_b200 import _lib as L
from zotitan_b200 import kernels as K
from zotitan_b200.build import build


@pytest.fixture(scope="module")
def lib():
    build()
    return L.load()


def test_struct_layouts(lib):
    assert ctypes.sizeof(L.ZtDistillArgs) == 128 and L.ZtDistillArgs.rows.offset == 72
    assert L.ZtDistillArgs.temperature.offset == 120
    assert ctypes.sizeof(L.ZtLinearDistillArgs) == 120 and L.ZtLinearDistillArgs.top.offset == 88
    assert L.ZtLinearDistillArgs.test_wait_cycles.offset == 112
    assert ctypes.sizeof(L.ZtQkArgs) == 304 and L.ZtQkArgs.q_strides.offset == 112
    assert L.ZtQkArgs.batch.offset == 256 and L.ZtQkArgs.eps.offset == 300


def rows_args(**kw):
    a = L.ZtDistillArgs()
    a.logits = a.grad = 256
    a.top_idx = a.top_logits = a.weight = a.loss = a.lse = a.stats = 512
    a.rows, a.vocab, a.ld, a.ld_grad, a.dtype = 4, 100, 100, 100, L.ZT_BF16
    a.top, a.idx_bits, a.top_dtype, a.temperature = 8, 64, L.ZT_F32, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_ROWS = [("rows", -1, L.ZT_ERR_INVALID), ("vocab", 0, L.ZT_ERR_INVALID), ("ld", 99, L.ZT_ERR_INVALID), ("vocab", 2**31, L.ZT_ERR_INVALID),
            ("rows", 2**30, L.ZT_ERR_LIMIT), ("dtype", 7, L.ZT_ERR_INVALID), ("top", 0, L.ZT_ERR_LIMIT), ("top", 257, L.ZT_ERR_LIMIT),
            ("idx_bits", 16, L.ZT_ERR_INVALID), ("top_dtype", 9, L.ZT_ERR_INVALID), ("temperature", 0.0, L.ZT_ERR_INVALID),
            ("temperature", math.nan, L.ZT_ERR_INVALID), ("temperature", 2e3, L.ZT_ERR_INVALID), ("logits", None, L.ZT_ERR_INVALID),
            ("logits", 257, L.ZT_ERR_INVALID), ("top_idx", None, L.ZT_ERR_INVALID), ("top_logits", None, L.ZT_ERR_INVALID)]


@pytest.mark.parametrize("field,value,code", BAD_ROWS)
def test_rows_refuse(lib, field, value, code):
    for fn in (lib.zt_distill_rows, lib.zt_distill_rows_backward, lib.zt_distill_rows_grad):
        assert fn(ctypes.byref(rows_args(**{field: value})), None) == code
        assert lib.zt_last_error()


def test_rows_refuse_their_own(lib):
    assert lib.zt_distill_rows(None, None) == L.ZT_ERR_INVALID
    assert lib.zt_distill_rows(ctypes.byref(rows_args(loss=None)), None) == L.ZT_ERR_INVALID
    assert lib.zt_distill_rows_backward(ctypes.byref(rows_args(stats=None)), None) == L.ZT_ERR_INVALID
    assert lib.zt_distill_rows_grad(ctypes.byref(rows_args(weight=None)), None) == L.ZT_ERR_INVALID
    for fn in (lib.zt_distill_rows_backward, lib.zt_distill_rows_grad):
        assert fn(ctypes.byref(rows_args(grad=None)), None) == L.ZT_ERR_INVALID
        assert fn(ctypes.byref(rows_args(ld_grad=99)), None) == L.ZT_ERR_INVALID
        assert fn(ctypes.byref(rows_args(ld_grad=104)), None) == L.ZT_ERR_INVALID      # in place, another stride
        assert b"in place" in lib.zt_last_error()
    empty = rows_args(rows=0, logits=None, grad=None, top_idx=None, top_logits=None)
    for fn in (lib.zt_distill_rows, lib.zt_distill_rows_backward, lib.zt_distill_rows_grad):
        assert fn(ctypes.byref(empty), None) == L.ZT_OK


@pytest.mark.parametrize("shape", [(0, 10, 64, 1), (10, 0, 64, 1), (10, 10, 0, 1), (10, 10, 65, 1), (10, 10, 64, 0), (10, 10, 64, 257),
                                   (2**29, 10, 64, 1), (10, 2**29, 64, 1), (2**28, 2**28, 64, 1)])
def test_linear_refuse_shapes(lib, shape):
    assert lib.zt_linear_distill_workspace_bytes(*shape) == 0
    assert lib.zt_last_error()


def test_linear_refuse(lib):
    good = dict(x=256, w=512, top_idx=1024, top_logits=1024, loss=1024, lse=1024, workspace=2048, workspace_bytes=1 << 30,
                rows=4, vocab=100, k=64, top=8, idx_bits=64, top_dtype=L.ZT_F32, temperature=1.0)
    for kw in (dict(x=None), dict(w=None), dict(top_idx=None), dict(top_logits=None), dict(loss=None), dict(lse=None),
               dict(workspace=None), dict(x=8), dict(w=8), dict(workspace=8), dict(k=72), dict(top=300), dict(idx_bits=8),
               dict(top_dtype=5), dict(temperature=-1.0)):
        a = L.ZtLinearDistillArgs()
        for k, v in (good | kw).items():
            setattr(a, k, v)
        assert lib.zt_linear_distill(ctypes.byref(a), None) in (L.ZT_ERR_INVALID, L.ZT_ERR_LIMIT), kw
    assert lib.zt_linear_distill(None, None) == L.ZT_ERR_INVALID
    assert lib.zt_linear_distill_take_error(None) == L.ZT_ERR_INVALID


def qk_args(**kw):
    a = L.ZtQkArgs()
    for n in ("q", "k", "q_out", "k_out", "q_grad", "k_grad", "q_weight", "k_weight", "cos", "sin", "dq_weight", "dk_weight", "workspace"):
        setattr(a, n, 256)
    a.workspace_bytes = 16
    a.batch, a.seq, a.q_heads, a.k_heads, a.head_dim = 2, 3, 4, 2, 64
    a.dtype = a.weight_dtype = a.table_dtype = L.ZT_BF16
    a.eps = 1e-6
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_qk_refuse(lib):
    for kw in (dict(batch=-1), dict(seq=-1), dict(q_heads=0), dict(k_heads=0), dict(head_dim=0), dict(head_dim=63), dict(head_dim=514),
               dict(dtype=8), dict(weight_dtype=L.ZT_F16), dict(table_dtype=L.ZT_F16), dict(table_batch=2), dict(eps=-1.0),
               dict(eps=math.nan), dict(eps=math.inf), dict(batch=2**20, seq=2**20), dict(q_heads=2**17), dict(q=None), dict(k_out=None),
               dict(q_weight=None), dict(cos=None)):
        for fn in (lib.zt_qk_norm_rope, lib.zt_qk_norm_rope_backward):
            assert fn(ctypes.byref(qk_args(**kw)), None) in (L.ZT_ERR_INVALID, L.ZT_ERR_LIMIT), kw
    for kw in (dict(q_grad=None), dict(dk_weight=None), dict(workspace=None), dict(workspace_bytes=0)):
        assert lib.zt_qk_norm_rope_backward(ctypes.byref(qk_args(**kw)), None) == L.ZT_ERR_INVALID, kw
    assert lib.zt_qk_norm_rope(None, None) == L.ZT_ERR_INVALID
    assert lib.zt_qk_norm_rope(ctypes.byref(qk_args(seq=0)), None) == L.ZT_OK
    assert lib.zt_qk_norm_rope_workspace_bytes(63) == 0 and lib.zt_qk_norm_rope_workspace_bytes(514) == 0


def test_wrappers_refuse_cpu_tensors():
    z, idx, val = torch.zeros(4, 10), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    for call in (lambda: K.distill_rows(z, idx, val), lambda: K.distill_rows_grad(z, idx, val, torch.ones(4)),
                 lambda: K.linear_distill(z.bfloat16(), z.bfloat16(), idx, val),
                 lambda: K.qk_norm_rope(*[torch.zeros(1, 2, 2, 8)] * 2, torch.ones(8), torch.ones(8), torch.zeros(2, 8), torch.zeros(2, 8))):
        with pytest.raises(ValueError):
            call()


def test_memory_overlap_rules():
    """What decides whether two views may be written in one launch."""
    t = torch.zeros(4, 6, 8)
    assert not K._shares_memory_inside(t) and not K._shares_memory_inside(t.transpose(0, 1))
    assert not K._shares_memory_inside(t[:, ::2]) and K._shares_memory_inside(t[:1].expand(4, -1, -1))
    assert K._shares_memory_inside(torch.zeros(20).as_strided((4, 8), (4, 1)))
    assert not K._shares_memory_inside(torch.zeros(20).as_strided((1, 8), (0, 1)))
    assert K._overlap(t[:2], t[1:3]) and not K._overlap(t[:2], t[2:]) and not K._overlap(t[:0], t)


def test_criterion_and_scorer_shape_checks():
    from zotitan_b200.objective import DistillationCriterion
    assert DistillationCriterion.name == "distill" and DistillationCriterion.differentiable
    from zotitan_b200.losses import distill_xentropy
    from toy_models import TOY, build_llama
    m = build_llama(TOY)
    ids = torch.zeros(2, 5, dtype=torch.int64)
    with pytest.raises(ValueError):
        distill_xentropy(m, {"input_ids": ids, "teacher_idx": ids, "teacher_logits": ids.float()})
