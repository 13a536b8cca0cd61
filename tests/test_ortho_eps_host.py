"""Newton-Schulz: an eps that could leave the norm's quotient above 1 is refused (no GPU: every call ends before a launch)."""
import ctypes as C

import pytest


@pytest.mark.parametrize("eps", [-1e-7, -1.0, float("nan"), -float("inf")])
def test_negative_eps_is_refused(eps):
    from recsys_amd._lib import MuonArgs, OrthoArgs, lib
    for cls, fn in ((OrthoArgs, lib.rx_orthogonalize), (MuonArgs, lib.rx_muon_step)):
        a = cls()
        a.count, a.steps, a.rows[0], a.cols[0] = 1, 5, 300, 400
        a.a, a.b, a.c, a.eps = 3.4445, -4.7750, 2.0315, eps
        a.g[0] = 1 << 20
        if cls is OrthoArgs:
            a.out[0] = 1 << 30
        else:
            a.w[0], a.mom[0] = 1 << 30, 1 << 32
        assert fn(C.byref(a), None, 0, 0, None) != 0
        assert b"eps" in lib.rx_last_error(), lib.rx_last_error()
