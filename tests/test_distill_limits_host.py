"""Limits and layouts of the distillation and q/k norm entry points on the host (CPU only)."""
import ctypes

import pytest

from test_distill_host import lib, qk_args  # noqa: F401  (lib is a fixture)
from zotitan_b200 import _lib as L


@pytest.mark.parametrize("batch,seq,fits", [(1, 2**25, True), (2**25, 1, True), (2**13, 2**12, True), (5, 6710886, True), (5, 6710887, False),
                                            (1, 2**25 + 1, False), (2**25 + 1, 1, False), (2**62, 2**62, False)])
def test_positions_up_to_the_documented_limit(lib, batch, seq, fits):  # noqa: F811
    """batch * seq <= 2^25: what is within passes on to the next check, a missing pointer."""
    for fn in (lib.zt_qk_norm_rope, lib.zt_qk_norm_rope_backward):
        assert fn(ctypes.byref(qk_args(batch=batch, seq=seq, q=None)), None) == (L.ZT_ERR_INVALID if fits else L.ZT_ERR_LIMIT)
        assert (b"null pointer" if fits else b"2^25") in lib.zt_last_error()


@pytest.mark.parametrize("version", [11, 3])
def test_library_of_another_build(tmp_path, monkeypatch, version):
    """A library without some of the entry points, or of another version, says so when it is loaded."""
    import subprocess
    src, so = tmp_path / "old.c", tmp_path / "old.so"
    src.write_text(f"int zt_abi_version(void) {{ return {version}; }}\nconst char* zt_last_error(void) {{ return \"\"; }}\n")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-o", str(so), str(src)])
    monkeypatch.setattr(L, "_lib", None)
    monkeypatch.setattr(L, "LIB_PATH", str(so))
    with pytest.raises(L.ZtError, match="zt_distill_rows" if version == L.ABI_VERSION else "ABI version 3"):
        L.load()
    assert L._lib is None


class Recorder:
    """In the library's place: keeps the argument bytes of the last call."""

    def __getattr__(self, name):
        def call(args, stream):
            self.name, self.args, self.stream = name, args, stream
            return L.ZT_OK
        return call


@pytest.fixture
def recorder(monkeypatch):
    import contextlib

    from zotitan_b200 import kernels as K
    rec = Recorder()
    monkeypatch.setattr(L, "load", lambda: rec)
    monkeypatch.setattr(K, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(K, "_raw_stream", lambda device: 77)
    return rec


def fields(struct, raw):
    assert len(raw) == ctypes.sizeof(struct)
    a = struct.from_buffer_copy(raw)
    return {n: list(getattr(a, n)) if isinstance(getattr(a, n), ctypes.Array) else getattr(a, n) for n, _ in struct._fields_}


def test_qk_arguments_as_the_header_lays_them_out(recorder):
    """The bytes that the wrappers pack, read back through the mirror of the C struct."""
    import torch

    from zotitan_b200 import kernels as K
    q, k = torch.zeros(2, 5, 9, 64).bfloat16()[:, :, :4], torch.zeros(2, 5, 3, 64).bfloat16()
    qo, ko, gq, gk = (torch.empty(2, 5, h, 64 + e)[..., :64].bfloat16() for h, e in ((4, 0), (3, 0), (4, 0), (3, 0)))
    gq = torch.zeros(2, 7, 4, 64).bfloat16()[:, :5]
    w, w2, cos, sin = torch.zeros(64), torch.zeros(64), torch.zeros(10, 64), torch.zeros(10, 64)
    ptr = torch.Tensor.data_ptr
    for back in (False, True):
        extra = (gq, gk, 1111, 2222, 3333, 4444) if back else ()
        K._qk_call("zt_qk_norm_rope", q, k, qo, ko, w, w2, cos, sin, 1e-5, True, *extra)
        got = fields(L.ZtQkArgs, recorder.args)
        assert recorder.stream == 77
        want = dict(q=ptr(q), k=ptr(k), q_out=ptr(qo), k_out=ptr(ko), q_grad=ptr(gq) if back else None, k_grad=ptr(gk) if back else None,
                    q_weight=ptr(w), k_weight=ptr(w2), cos=ptr(cos), sin=ptr(sin), dq_weight=1111 if back else None,
                    dk_weight=2222 if back else None, workspace=3333 if back else None, workspace_bytes=4444 if back else 0,
                    q_strides=[2880, 576, 64], k_strides=[960, 192, 64], q_out_strides=[1280, 256, 64], k_out_strides=[960, 192, 64],
                    q_grad_strides=[1792, 256, 64] if back else [0] * 3, k_grad_strides=[960, 192, 64] if back else [0] * 3,
                    batch=2, seq=5, q_heads=4, k_heads=3, head_dim=64, dtype=L.ZT_BF16, weight_dtype=L.ZT_F32, table_dtype=L.ZT_F32,
                    table_batch=1, eps=ctypes.c_float(1e-5).value)
        assert got == want


def test_distill_arguments_as_the_header_lays_them_out(recorder):
    import torch

    from zotitan_b200 import kernels as K
    z, grad = torch.zeros(6, 20).half()[:, :17], torch.zeros(6, 24).half()[:, :17]
    idx, val, w, wl = torch.zeros(6, 3, dtype=torch.int32), torch.zeros(6, 3).bfloat16(), torch.zeros(6), torch.zeros(6)
    K._distill_call("zt_distill_rows_grad", z, idx, val, 0.5, grad=grad, weight=w, weight_lse=wl, loss=11, lse=22, stats=33)
    ptr = torch.Tensor.data_ptr
    assert fields(L.ZtDistillArgs, recorder.args) == dict(
        logits=ptr(z), grad=ptr(grad), top_idx=ptr(idx), top_logits=ptr(val), weight=ptr(w), weight_lse=ptr(wl), loss=11, lse=22, stats=33,
        rows=6, vocab=17, ld=20, ld_grad=24, dtype=L.ZT_F16, top=3, idx_bits=32, top_dtype=L.ZT_BF16, temperature=0.5, reserved=0)


def test_linear_distill_arguments_as_the_header_lays_them_out(recorder, monkeypatch):
    import torch

    from zotitan_b200 import kernels as K
    monkeypatch.setattr(K, "linear_xent_supported", lambda x, w: True)
    Recorder.zt_linear_distill_workspace_bytes = lambda self, *shape: 4096
    try:
        x, w = torch.zeros(6, 64).bfloat16(), torch.zeros(17, 64).bfloat16()
        idx, val = torch.zeros(6, 3, dtype=torch.int64), torch.zeros(6, 3)
        loss, lse = K.linear_distill(x, w, idx, val, 0.5, True, 12345)
    finally:
        del Recorder.zt_linear_distill_workspace_bytes
    got = fields(L.ZtLinearDistillArgs, recorder.args)
    ptr = torch.Tensor.data_ptr
    assert got.pop("workspace") not in (None, 0)
    assert got == dict(x=ptr(x), w=ptr(w), top_idx=ptr(idx), top_logits=ptr(val), loss=ptr(loss), lse=ptr(lse), workspace_bytes=4096, rows=6,
                       vocab=17, k=64, top=3, idx_bits=64, top_dtype=L.ZT_F32, temperature=0.5, test_stall_loads=1, reserved=0,
                       test_wait_cycles=12345)


@pytest.mark.parametrize("dt", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("vocab,ld,shift", [(1000, 1000, 0), (1000, 1001, 1), (1003, 1003, 3), (1003, 50 * 1003, 7), (17, 24, 5), (1, 9, 2)])
def test_gradient_room_is_aligned_as_the_logits_are(dt, vocab, ld, shift):
    """Every row of the gradient starts at the 16-byte phase of its row of logits, within a row more of room."""
    import torch

    from zotitan_b200 import kernels as K
    dtype = getattr(torch, dt)
    x = torch.zeros(4 * ld + shift, dtype=dtype)[shift:].view(4, ld)[:, :vocab]
    g = K._grad_of(x)
    assert g.shape == x.shape and g.dtype == dtype and g.stride(1) == 1 and g.stride(0) >= vocab
    for r in range(4):
        assert g[r].data_ptr() % 16 == x[r].data_ptr() % 16
    assert g.untyped_storage().nbytes() <= 4 * (vocab + 8) * x.element_size() + 16
