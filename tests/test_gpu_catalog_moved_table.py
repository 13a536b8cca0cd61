"""A table with a fused sparse rule and no clip takes its step inside the backward pass: a second backward pass over the catalogue as
it was before is refused, not computed from rows that have moved since."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model():
    from recsys_amd.models.matrix_factorization import BiasMF
    torch.manual_seed(1)
    return BiasMF(50, 70, 16).cuda().set_objective("catalog")


def _batch(seed):
    g = torch.Generator().manual_seed(seed)
    return {"user_code": torch.randint(0, 50, (30,), generator=g).cuda(), "item_code": torch.randint(0, 70, (30, 2), generator=g).cuda()}


def test_two_losses_in_one_backward_pass():
    from recsys_amd.optim import FusedOptimizer
    m = _model()
    opt = FusedOptimizer(m, kind="sgd", lr=0.1)
    opt.zero_grad()
    with pytest.raises(RuntimeError, match="moved"):
        (m.loss(_batch(1)) + m.loss(_batch(2))).backward()
    # one after the other is what gradient accumulation without a clip comes to
    opt.zero_grad()
    for seed in (1, 2):
        m.loss(_batch(seed)).backward()
    opt.step()
    late = m.loss(_batch(3))
    m.loss(_batch(4)).backward()
    with pytest.raises(RuntimeError, match="moved"):
        late.backward()


def test_with_a_clip_both_gradients_count():
    from recsys_amd.optim import FusedOptimizer
    m, ref = _model(), _model()
    opt = FusedOptimizer(m, kind="sgd", lr=0.1, clip_norm=1e9)
    opt.zero_grad()
    (m.loss(_batch(1)) + m.loss(_batch(2))).backward()
    opt.step()
    (ref.loss(_batch(1)) + ref.loss(_batch(2))).backward()
    for (n, p), q in zip(m.named_parameters(), ref.parameters()):
        if q.grad is not None:
            # two fp32 gradients, added to the weight one by one or together
            assert (p - (q - 0.1 * q.grad)).abs().max() <= 4 * 2.0 ** -24 * q.abs().max() + 1e-6 * q.grad.abs().max(), n
    late = m.loss(_batch(3))
    opt.zero_grad()
    m.loss(_batch(4)).backward()
    opt.step()
    with pytest.raises(RuntimeError, match="moved"):
        late.backward()
