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
