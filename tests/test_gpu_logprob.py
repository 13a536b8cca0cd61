"""List-wise log-probabilities, entropy, alternatives and their gradient (rx_logprob_*) against the definition in fp64.

Tolerances.  u = 2^-24.  A lane adds at most ``seq`` terms one after the other before the tree sums (``_seq``), so the sum
s carries a relative error of at most (seq + 16) u from additions, 4 u from the exponential, and 2 |d| u per term from its
argument d = (l - m) log2 e, which the weights e^d bring to at most 2 (log V + 1) u on average.  log s moves by that much;
the score's own term, the logarithm and the final product add 4 u each relative to the result.  ``_tol`` is their sum.
bf16 gradients add half a bf16 step, 2^-8 of the value."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


def _seq(V):
    return max(16, math.ceil(V / 256) + 16)


def _tol(V, value):
    return U * (_seq(V) + 32 + 4 * math.log(V + 1)) + 8 * U * value.abs()


def _ref(logits, targets, lengths, k):
    z = logits.detach().double().cpu()
    R, V = z.shape
    if lengths is not None:
        z = z.masked_fill(torch.arange(V)[None] >= lengths.cpu().clamp(0, V)[:, None], -INF)
    m = z.max(1, keepdim=True).values
    m = torch.where(m == -INF, torch.zeros_like(m), m)
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    empty = (s == 0)[:, 0]
    logp = torch.where(e > 0, (z - m) - s.log(), torch.full_like(z, -INF))
    logp = torch.where(z == -INF, logp, (z - m) - s.log())          # below exp's range: still a log-probability
    lse = (m + s.log())[:, 0]
    p = logp.exp()
    H = -(p * torch.where(p > 0, logp, torch.zeros_like(logp))).sum(1)
    H[empty] = 0
    t = targets.cpu().reshape(R, -1)
    lp = torch.where(t < 0, torch.zeros(t.shape, dtype=torch.float64), logp.gather(1, t.clamp(min=0)))
    kk = min(k, V)
    val, idx = torch.sort(z, dim=1, descending=True, stable=True)
    dead = val[:, :kk] == -INF
    top = logp.gather(1, idx[:, :kk]).masked_fill(dead, -INF)
    idx = idx[:, :kk].masked_fill(dead, -1)
    pad = (0, k - kk)
    return (lp.reshape(targets.shape), H, lse, torch.nn.functional.pad(top, pad, value=-INF), torch.nn.functional.pad(idx, pad, value=-1)), logp, p


def _check(name, got, ref, V, scale=None):
    got, ref = got.detach().double().cpu(), ref
    assert got.shape == ref.shape, name
    fin = torch.isfinite(ref)
    assert torch.equal(got.isnan(), ref.isnan()), name
    inf = ~fin & ~ref.isnan()
    assert torch.equal(got[inf], ref[inf]), name
    err = (got - ref).abs()[fin]
    tol = _tol(V, ref[fin] if scale is None else scale[fin])
    assert (err <= tol).all(), (name, float((err / tol).max()), float(err.max()))


def _compare(out, ref, V):
    names = ("logprob", "entropy", "lse", "top_logprob")
    for name, got, want in zip(names, out, ref):
        _check(name, got, want, V)
    assert torch.equal(out.top_index.cpu(), ref[4])


def _make(R, V, dtype, T, seed, ragged=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn(R, V, generator=g, device="cuda") * 3).to(dtype)
    targets = torch.randint(0, V, (R, T), generator=g, device="cuda")
    targets[::3, 0] = -1
    lengths = torch.randint(0, V + 1, (R,), generator=g, device="cuda") if ragged else None
    return logits, targets, lengths


SIZES = [(1, 1), (3, 2), (70, 5), (9, 8), (9, 9), (33, 32), (5, 33), (7, 64), (7, 65), (130, 100), (3, 257), (3, 1000), (6, 1024),
         (6, 1025), (5, 1031), (4, 4099), (3, 8192), (2, 20011), (1, 70001), (1, 1000003), (1100, 1500)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", SIZES)
def test_forward_over_sizes(R, V, dtype):
    from recsys_amd import autograd as rxa
    for k, T, ragged in ((0, 1, False), (10, 3, True), (64, 1, False), (1, 2, True)):
        logits, targets, lengths = _make(R, V, dtype, T, R * 7 + V + k, ragged)
        out = rxa.log_probs(logits, targets, lengths=lengths, k=k)
        _compare(out, _ref(logits, targets, lengths, k)[0], V)
        again = rxa.log_probs(logits, targets, lengths=lengths, k=k)
        assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("V", [5, 40, 200, 1024, 1500, 9001, 30000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_and_extreme_rows(V, dtype):
    """-inf masks, masks of the type's lowest value, rows with nothing left, offsets where exp(l) leaves fp32, ties."""
    from recsys_amd import autograd as rxa
    lowest = torch.finfo(dtype).min
    g = torch.Generator(device="cuda").manual_seed(V)
    base = torch.randn(14, V, generator=g, device="cuda") * 2
    hide = torch.rand(14, V, generator=g, device="cuda") < 0.7
    base[0] = -INF
    base[1] = lowest
    base[2] = torch.where(hide[2], torch.full_like(base[2], -INF), torch.full_like(base[2], lowest))
    base[3][hide[3]] = -INF
    base[4][hide[4]] = lowest
    base[5] = 0.0
    base[6] = torch.arange(V, device="cuda") / 64.0                 # every score beats all before it
    base[7] = -torch.arange(V, device="cuda") / 64.0
    base[8] += 3000.0
    base[9] -= 3000.0
    base[10] = -INF
    base[10, V - 1] = lowest
    base[11] = 3.0e38
    base[12] = torch.where(hide[12], torch.full_like(base[12], -0.0), torch.zeros_like(base[12]))
    base[13] = -INF
    base[13, V // 2] = 1.5
    logits = base.to(dtype)
    targets = torch.stack([torch.zeros(14, dtype=torch.int64), torch.full((14,), V - 1), torch.full((14,), V // 2)], 1).cuda()
    out = rxa.log_probs(logits, targets, k=min(64, V))
    ref, _, _ = _ref(logits, targets, None, min(64, V))
    # entropy and log-probabilities are taken from the reference score, not from the rounded lse; lse itself has half a step
    _compare(out, ref, V)
    assert out.lse[0] == -INF and out.entropy[0] == 0 and (out.top_index[0] == -1).all()


def test_hidden_columns_may_hold_anything():
    from recsys_amd import autograd as rxa
    for V in (6, 90, 1000, 5000, 40000):
        logits, targets, lengths = _make(9, V, torch.float32, 2, V, True)
        lengths[0] = 0
        lengths[1] = V
        ref, _, _ = _ref(logits, targets, lengths, 7)
        for junk in (float("nan"), INF, -INF, 3e38):
            x = torch.where(torch.arange(V, device="cuda")[None] < lengths[:, None], logits, torch.full_like(logits, junk))
            x.requires_grad_(True)
            out = rxa.log_probs(x, targets, lengths=lengths, k=7)
            _compare(out, ref, V)
            dl, = torch.autograd.grad((out.logprob.clamp(min=-1e3).sum(), out.entropy.sum()), x)
            assert torch.isfinite(dl).all()
            assert not dl[torch.arange(V, device="cuda")[None] >= lengths[:, None]].any()


def test_nan_and_plus_inf_spoil_their_row_only():
    from recsys_amd import autograd as rxa
    for V in (7, 300, 3000, 30000):
        for bad in (float("nan"), INF):
            logits, targets, _ = _make(6, V, torch.float32, 1, V)
            good = rxa.log_probs(logits, targets, k=4)
            x = logits.clone()
            x[2, V // 3] = bad
            out = rxa.log_probs(x, targets, k=4)
            keep = torch.arange(6, device="cuda") != 2
            for a, b in zip(out, good):
                assert torch.equal(a[keep], b[keep])
            assert out.lse[2].isnan() and out.entropy[2].isnan() and out.logprob[2].isnan().all()
            assert ((out.top_index[2] >= -1) & (out.top_index[2] < V)).all()


def _ref_grad(logits, targets, lengths, g, gh, gl):
    """dl from its formula in fp64, and the sum of the absolute values of its terms."""
    R, V = logits.shape
    (lp, H, lse, _, _), logp, p = _ref(logits, targets, lengths, 1)
    t = targets.cpu().reshape(R, -1)
    z = logits.detach().double().cpu()
    live = (t >= 0) & (z.gather(1, t.clamp(min=0)) > -INF)
    if lengths is not None:
        live &= t < lengths.cpu()[:, None]
    g = torch.where(live, g.double().cpu().reshape(R, -1), torch.zeros(t.shape, dtype=torch.float64))
    gh, gl = gh.double().cpu(), gl.double().cpu()
    lpz = torch.where(p > 0, logp, torch.zeros_like(logp))
    hot = torch.zeros_like(p).scatter_add_(1, t.clamp(min=0), g)
    d = hot + p * (gl - g.sum(1))[:, None] - gh[:, None] * p * (lpz + H[:, None])
    size = torch.zeros_like(p).scatter_add_(1, t.clamp(min=0), g.abs()) \
        + p * (gl.abs() + g.abs().sum(1) + gh.abs() * H.abs())[:, None] + gh.abs()[:, None] * p * lpz.abs()
    noise = U * (_seq(V) + 64 + 8 * math.log(V + 1)) * size + 4 * U * size * lpz.abs()
    return d, noise


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [s for s in SIZES if s[1] <= 70001])
def test_gradient_over_sizes(R, V, dtype):
    from recsys_amd import autograd as rxa
    for T, ragged in ((1, False), (5, True)):
        logits, targets, lengths = _make(R, V, dtype, T, R + 3 * V, ragged)
        targets[:, -1] = targets[:, 0]                       # the same column twice
        if V > 3:
            logits[0, ::2] = -INF
        x = logits.clone().requires_grad_(True)
        out = rxa.log_probs(x, targets, lengths=lengths, k=1)
        g = torch.randn(R, T, device="cuda")
        gh, gl = torch.randn(R, device="cuda"), torch.randn(R, device="cuda")
        dl, = torch.autograd.grad((out.logprob, out.entropy, out.lse), x, (g, gh, gl))
        ref, noise = _ref_grad(logits, targets, lengths, g, gh, gl)
        tol = noise + (2.0 ** -8 * (ref.abs() + noise) if dtype == torch.bfloat16 else 0) + 1e-38
        err = (dl.double().cpu() - ref).abs()
        assert (err <= tol).all(), float((err / tol).max())
        again, = torch.autograd.grad(rxa.log_probs(x, targets, lengths=lengths)[:3], x, (g, gh, gl))
        assert torch.equal(dl, again)


def test_gradient_against_differences():
    from recsys_amd import autograd as rxa
    R, V, T = 4, 23, 3
    logits, targets, lengths = _make(R, V, torch.float32, T, 5, True)
    lengths[0] = V
    x = logits.clone().requires_grad_(True)
    w, wh, wl = torch.randn(R, T, device="cuda"), torch.randn(R, device="cuda"), torch.randn(R, device="cuda")

    def f(z):
        (lp, H, lse, _, _), _, _ = _ref(z, targets, lengths, 1)
        ok = torch.isfinite(lp)
        row = torch.isfinite(lse)
        return float((lp[ok] * w.double().cpu()[ok]).sum() + (H * wh.double().cpu()).sum() + (lse[row] * wl.double().cpu()[row]).sum())

    o = rxa.log_probs(x, targets, lengths=lengths)
    dl, = torch.autograd.grad((o.logprob, o.entropy, o.lse), x, (w, wh, wl))
    z, h = logits.double(), 1e-5
    for r in range(R):
        for c in range(0, V, 3):
            a, b = z.clone(), z.clone()
            a[r, c] += h
            b[r, c] -= h
            # central difference: h^2 f'''/6 <= 1e-9 of the terms, and 1e-16 / h from rounding f
            want = (f(a) - f(b)) / (2 * h)
            assert abs(float(dl[r, c]) - want) <= 1e-6 * (1 + abs(want)), (r, c)


def test_strided_and_unaligned_rows():
    """Slices of a wider buffer: rows further apart than V, at every alignment; gradients land in the slice only."""
    from recsys_amd import autograd as rxa
    for dtype in (torch.float32, torch.bfloat16):
        for V in (7, 200, 1400, 9000):
            for off in (0, 1, 3, 5):
                buf = torch.full((6, V + 9), float("nan"), device="cuda", dtype=dtype)
                logits, targets, _ = _make(6, V, dtype, 2, V + off)
                buf[:, off:off + V] = logits
                buf.requires_grad_(True)
                out = rxa.log_probs(buf[:, off:off + V], targets, k=5)
                _compare(out, _ref(logits, targets, None, 5)[0], V)
                g = torch.randn(6, 2, device="cuda")
                db, = torch.autograd.grad(out.logprob, buf, g)
                # where a row starts decides which lane adds which score, so rows at two alignments agree to rounding only
                zero = torch.zeros(6, device="cuda")
                ref, noise = _ref_grad(logits, targets, None, g, zero, zero)
                tol = noise + (2.0 ** -8 * (ref.abs() + noise) if dtype == torch.bfloat16 else 0) + 1e-38
                assert ((db[:, off:off + V].double().cpu() - ref).abs() <= tol).all()
                assert not db[:, :off].any() and not db[:, off + V:].any()
    # columns that are not adjacent and rows that overlap are laid out first
    logits, targets, _ = _make(5, 12, torch.float32, 1, 1)
    a = rxa.log_probs(logits.t().contiguous().t(), targets, k=3)
    assert all(torch.equal(p, q) for p, q in zip(a, rxa.log_probs(logits, targets, k=3)))
    one = logits[:1].clone().requires_grad_(True)
    out = rxa.log_probs(one.expand(5, 12), targets.clamp(min=0))
    d, = torch.autograd.grad(out.logprob.sum(), one)
    full = logits[:1].repeat(5, 1).requires_grad_(True)
    e, = torch.autograd.grad(rxa.log_probs(full, targets.clamp(min=0)).logprob.sum(), full)
    assert (d - e.sum(0, keepdim=True)).abs().max() < 16 * U * 5


def test_recorded_and_replayed_on_another_stream():
    from recsys_amd import autograd as rxa, ops
    ops.set_index_check("deferred")
    try:
        for V in (5, 300, 2000, 100003):
            logits, targets, lengths = _make(4, V, torch.float32, 2, V, True)
            x = logits.clone()
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())

            def step():
                leaf = x.detach().requires_grad_(True)
                o = rxa.log_probs(leaf, targets, lengths=lengths, k=9)
                dl, = torch.autograd.grad((o.logprob, o.entropy), leaf, (torch.ones_like(o.logprob), torch.ones_like(o.entropy)))
                return tuple(o) + (dl,)

            with torch.cuda.stream(stream):
                step()
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    rec = step()
            torch.cuda.current_stream().wait_stream(stream)
            for seed in range(3):
                new, nt, nl = _make(4, V, torch.float32, 2, 100 + seed, True)
                x.copy_(new); targets.copy_(nt); lengths.copy_(nl)
                torch.cuda.synchronize()
                graph.replay()
                eager = step()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(rec, eager))
        ops.raise_if_index_error()
    finally:
        ops.set_index_check("sync")


def test_bad_targets_and_refusals():
    from recsys_amd import autograd as rxa, ops
    logits, targets, _ = _make(4, 20, torch.float32, 2, 3)
    for bad in (20, -2, 1 << 40):
        t = targets.clone()
        t[1, 1] = bad
        with pytest.raises(IndexError):
            rxa.log_probs(logits, t)
    ops.raise_if_index_error()
    with pytest.raises(TypeError):
        rxa.log_probs(logits.double(), targets)
    with pytest.raises(TypeError):
        rxa.log_probs(logits, targets.int())
    with pytest.raises(ValueError):
        rxa.log_probs(logits, targets[:3])
    with pytest.raises(ValueError):
        rxa.log_probs(logits, targets, k=65)
    with pytest.raises(ValueError):
        rxa.log_probs(logits, targets, lengths=torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        rxa.log_probs(logits, targets.cpu())
    with pytest.raises(ValueError):
        rxa.log_probs(logits[:, :0], targets)
    x = logits.clone().requires_grad_(True)
    out = rxa.log_probs(x, targets)
    d, = torch.autograd.grad(out.logprob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
    # empty batch
    out = rxa.log_probs(torch.empty(0, 7, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda"), k=3)
    assert out.logprob.shape == (0, 2) and out.top_index.shape == (0, 3)
