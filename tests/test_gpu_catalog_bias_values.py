"""Catalogue softmax: biases that are not numbers are not taken for masks."""
import pytest
import torch

from test_gpu_catalog import INF, _make, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), INF])
def test_a_bias_that_is_no_number(bad, dtype):
    for R, V, D in ((40, 300, 20), (5, 4000, 64), (130, 70, 100)):
        x, t, y, b = _make(R, V, D, dtype, True, R)
        y[y == V // 3] = 0
        y[0] = -1
        b[V // 3] = bad
        g, gl = torch.ones(R, device="cuda"), torch.ones(R, device="cuda")
        gl[:] = 0.5
        got = _run(x, t, y, b, g, gl)
        assert got[1].isnan().all()                       # as a score of +inf or NaN does in rx_logprob
        assert got[0][1:].isnan().all() and got[0][0] == 0
        assert got[2].isnan().all() and got[3].isnan().all() and got[4].isnan().all()
