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
