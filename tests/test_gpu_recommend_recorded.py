"""utils.recommend in a recording: positions to leave out are looked at on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_positions_out_of_range_in_a_recording_are_left_alone():
    """Beyond the score row (or below -1) a position means nothing in a replay, where nobody can raise; eagerly it is an error."""
    from recsys_amd import ops
    from recsys_amd.models.matrix_factorization import VanillaMF
    from recsys_amd.utils import recommend
    ops.set_index_check("deferred")
    try:
        m = VanillaMF(n_users=30, n_items=80, embedding_dim=16).cuda().eval()
        users = torch.arange(12, device="cuda")
        exclude = torch.full((12, 3), -1, dtype=torch.int64, device="cuda")
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call = lambda e: recommend(m, {"user_code": users, "item_code": None}, k=5, exclude=e)
            call(exclude)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                rec = call(exclude)
        torch.cuda.current_stream().wait_stream(stream)
        for value in (80, 81, -2, 7, 1 << 40, -(1 << 40)):
            exclude.fill_(-1)
            exclude[:, 1] = value
            exclude[:, 2] = torch.arange(12, device="cuda")
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            good = exclude.clone()
            if not 0 <= value < 80:
                good[:, 1] = -1
            for a, b in zip(rec, call(good)):
                assert torch.equal(a, b)
            if not -1 <= value < 80:
                with pytest.raises(IndexError):
                    call(exclude)
        ops.raise_if_index_error()
    finally:
        ops.set_index_check("sync")
