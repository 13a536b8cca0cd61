"""Host-side refusals and struct layouts of the catalogue and orthogonalisation entry points (no GPU: every call below ends
before a launch)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from conftest import ROOT


def _cat(**kw):
    from recsys_amd._lib import CatalogArgs
    base = dict(x=4096, table=4096, ld_x=8, ld_t=8, bias=0, targets=4096, R=4, V=10, D=8, bf16=0)
    base.update(kw)
    return CatalogArgs(**base)


@pytest.mark.parametrize("kw,text", [(dict(D=0), b"bad shape"), (dict(D=257, ld_x=257, ld_t=257), b"bad shape"), (dict(V=0), b"bad shape"),
                                     (dict(R=-1), b"bad shape"), (dict(R=(1 << 24) + 1), b"bad shape"), (dict(V=(1 << 30) + 1), b"bad shape"),
                                     (dict(ld_x=(1 << 22) + 1), b"apart"), (dict(ld_t=1 << 40), b"apart"),
                                     (dict(ld_x=7), b"row strides"), (dict(ld_t=7), b"row strides"), (dict(bf16=3), b"element type"),
                                     (dict(x=0), b"null"), (dict(table=0), b"null"), (dict(targets=0), b"null"), (dict(table=4098), b"aligned")])
def test_catalog_refusals(kw, text):
    from recsys_amd._lib import lib
    a, p = _cat(**kw), C.c_void_p(4096)
    assert lib.rx_catalog_fwd(C.byref(a), p, p, p, p, p, 1 << 40, None, 0, None) != 0
    assert text in lib.rx_last_error()
    assert lib.rx_catalog_bwd(C.byref(a), p, p, p, p, p, p, None, p, 1 << 40, 0, None) != 0
    assert text in lib.rx_last_error()


def test_catalog_workspaces_and_gradient_buffers():
    from recsys_amd._lib import lib
    a, p = _cat(), C.c_void_p(4096)
    for call, text in ((lambda: lib.rx_catalog_fwd(C.byref(a), p, p, p, p, p, 8, None, 0, None), b"workspace"),
                       (lambda: lib.rx_catalog_fwd(C.byref(a), None, p, p, p, p, 1 << 30, None, 0, None), b"null output"),
                       (lambda: lib.rx_catalog_bwd(C.byref(a), None, p, p, p, p, p, None, p, 1 << 30, 0, None), b"stats"),
                       (lambda: lib.rx_catalog_bwd(C.byref(a), p, None, p, p, p, p, None, p, 1 << 30, 0, None), b"means"),
                       (lambda: lib.rx_catalog_bwd(C.byref(a), p, p, p, p, p, p, p, p, 1 << 30, 0, None), b"bias"),
                       (lambda: lib.rx_catalog_bwd(C.byref(a), p, p, p, p, p, p, None, p, 8, 0, None), b"workspace"),
                       (lambda: lib.rx_catalog_bwd(C.byref(a), p, p, p, p, p, C.c_void_p(4100), None, p, 1 << 30, 0, None), b"aligned")):
        assert call() != 0
        assert text in lib.rx_last_error()
    f, b = lib.rx_catalog_fwd_workspace_bytes, lib.rx_catalog_bwd_workspace_bytes
    assert f(0, 10, 8, 0, 1) == 0 and b(0, 10, 8, 0, 1) == 0 and f(4, 10, 300, 0, 1) == 0
    assert f(100, 10000, 64, 0, 1) > f(100, 10000, 64, 0, 0) > 0 and b(100, 10000, 64, 0, 0) > 0


def test_ortho_and_muon_refusals():
    from recsys_amd._lib import MuonArgs, OrthoArgs, lib
    def both(setup, text):
        for cls, fn, q in ((OrthoArgs, lib.rx_orthogonalize, lib.rx_orthogonalize_workspace_bytes),
                           (MuonArgs, lib.rx_muon_step, lib.rx_muon_step_workspace_bytes)):
            a = cls()
            a.count, a.steps, a.rows[0], a.cols[0] = 1, 5, 300, 400
            a.g[0] = 1 << 20
            if cls is OrthoArgs:
                a.out[0] = 1 << 30
            else:
                a.w[0], a.mom[0] = 1 << 30, 1 << 32
            assert q(C.byref(a)) > 0
            setup(a)
            assert fn(C.byref(a), None, 0, 0, None) != 0
            assert text in lib.rx_last_error(), lib.rx_last_error()
    both(lambda a: None, b"workspace")
    both(lambda a: setattr(a, "count", 25), b"at most 24")
    both(lambda a: setattr(a, "steps", 0), b"steps")
    both(lambda a: a.rows.__setitem__(0, 0), b"matrix 0")
    both(lambda a: a.cols.__setitem__(0, 16385), b"matrix 0")
    both(lambda a: a.g.__setitem__(0, 0), b"null")
    both(lambda a: a.g.__setitem__(0, (1 << 30) + 64), b"overlap")


def test_overlaps_in_lists_longer_than_a_chunk():
    import torch
    from recsys_amd.ops import _apart
    a = [torch.zeros(4, 5) for _ in range(30)]
    b = [torch.zeros(4, 5) for _ in range(30)]
    _apart("x", a, b)
    _apart("x", a[:1] * 30, b)                    # what is only read may be the same
    _apart("x", a[:5], a[:5])                     # short lists are the library's to check
    flat = torch.zeros(2000)
    for writes in (b[:29] + b[:1], b[:29] + a[:1], [flat[0:20].view(4, 5)] + b[:28] + [flat[19:39].view(4, 5)]):
        with pytest.raises(ValueError, match="overlap"):
            _apart("x", a, writes)
    _apart("x", a, [flat[0:20].view(4, 5)] + b[:28] + [flat[20:40].view(4, 5)])


def test_struct_layouts(tmp_path):
    from recsys_amd import _lib
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "recsys_hip.h"\nint main(void){printf("%zu %zu %zu %zu %zu %zu %zu", '
                   'sizeof(rx_catalog_args), offsetof(rx_catalog_args, D), sizeof(rx_ortho_args), offsetof(rx_ortho_args, a), '
                   'sizeof(rx_muon_args), offsetof(rx_muon_args, count), offsetof(rx_muon_args, scale));return 0;}\n')
    exe = tmp_path / "s"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    c, o, m = _lib.CatalogArgs, _lib.OrthoArgs, _lib.MuonArgs
    assert got == [C.sizeof(c), c.D.offset, C.sizeof(o), o.a.offset, C.sizeof(m), m.count.offset, m.scale.offset]


def test_wrappers_refuse_host_tensors():
    from recsys_amd import autograd as rxa, ops
    with pytest.raises(ValueError, match="GPU"):
        rxa.catalog_logprob(torch.zeros(2, 3), torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        ops.orthogonalize([torch.zeros(2, 3)])
    with pytest.raises(ValueError, match="GPU"):
        ops.muon_step([torch.zeros(2, 3)], [torch.zeros(2, 3)], [torch.zeros(2, 3)], [0.1])
