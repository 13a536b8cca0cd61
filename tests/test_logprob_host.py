"""Host-side refusals of the log-probability entry points (no GPU: every call below ends before a launch)."""
import ctypes as C

import pytest
import torch


def _args(**kw):
    from recsys_amd._lib import LogProbArgs
    base = dict(logits=4096, ld=8, R=2, V=8, lengths=0, targets=4096, T=1, k=0, bf16=0, logprob=4096, lse=4096, entropy=4096,
                top_logprob=4096, top_index=4096, stats=4096)
    base.update(kw)
    return LogProbArgs(**base)


@pytest.mark.parametrize("kw,text", [
    (dict(V=0), b"bad shape"), (dict(ld=7), b"bad shape"), (dict(R=-1), b"bad shape"), (dict(V=1 << 31, ld=1 << 31), b"bad shape"),
    (dict(T=1025), b"targets per row"), (dict(T=-1), b"targets per row"), (dict(bf16=2), b"element type"), (dict(k=65), b"alternatives"),
    (dict(logits=0), b"null"), (dict(targets=0), b"null"), (dict(lse=0), b"null"), (dict(k=3, top_index=0), b"null"),
    (dict(logits=4097), b"aligned"), (dict(stats=4100), b"aligned"), (dict(R=1, V=100000, ld=100000), b"workspace")])
def test_forward_refusals(kw, text):
    from recsys_amd._lib import lib
    a = _args(**kw)
    assert lib.rx_logprob_fwd(C.byref(a), None, 0, None, 0, None) != 0
    assert text in lib.rx_last_error()


def test_backward_refusals():
    from recsys_amd._lib import lib
    for kw, ld, out, text in ((dict(), 7, 4096, b"row stride"), (dict(), 8, 0, b"gradient buffer"), (dict(stats=0), 8, 4096, b"gradient buffer"),
                              (dict(V=0), 8, 4096, b"bad shape")):
        a = _args(**kw)
        assert lib.rx_logprob_bwd(C.byref(a), None, None, None, C.c_void_p(out), ld, 0, None) != 0
        assert text in lib.rx_last_error()


def test_workspace_query_and_struct_layout(tmp_path):
    import os
    import subprocess
    from conftest import ROOT
    from recsys_amd import _lib
    q = _lib.lib.rx_logprob_workspace_bytes
    assert q(0, 10 ** 6, 5) == 0 and q(1000, 1024, 5) == 0 and q(1, 100000, 65) == 0
    assert q(1, 1000000, 0) > 0 and q(1, 1000000, 50) > q(1, 1000000, 10)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "recsys_hip.h"\nint main(void){printf("%zu %zu %zu", '
                   'sizeof(rx_logprob_args), offsetof(rx_logprob_args, logprob), offsetof(rx_logprob_args, stats));return 0;}\n')
    exe = tmp_path / "s"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = [int(v) for v in subprocess.check_output([str(exe)]).split()]
    A = _lib.LogProbArgs
    assert got == [C.sizeof(A), A.logprob.offset, A.stats.offset]


def test_wrappers_refuse_host_tensors():
    from recsys_amd import autograd as rxa
    with pytest.raises(ValueError, match="GPU"):
        rxa.log_probs(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
