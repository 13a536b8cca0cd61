"""The list-wise log-probability, catalogue softmax and orthogonalised-update operators as measurable cases.

Three operators and the calls a user makes of them:

* ``logprob``: log-probabilities of given items from scores ``[R, V]`` that are already in hand, with each row's
  entropy and its ``k`` best alternatives (evaluation, serving), or with the gradient to the scores (list-wise loss).
* ``catalog``: log-probabilities of one given item per row under the softmax over a whole item table, scores
  ``x @ table.T + bias`` never stored; with the gradients to ``x``, the table and the bias (full-catalogue loss).
* ``ortho``: Newton-Schulz orthogonalisation of a list of weight updates (the dense half of a train step).

``own = False`` computes them with elementary torch operations in 32 bits; ``own = True`` calls the framework.
"""
import math

import torch

own = False

NS_STEPS, NS_COEFFS, NS_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases
def _logprob(mode, R, V, dtype, T=1, k=0, ragged=False, name=None):
    c = dict(op="logprob", mode=mode, R=R, V=V, dtype=dtype, T=T, k=k, ragged=ragged)
    return dict(c, name=name) if name else c


def _catalog(mode, R, V, D, dtype, bias, name=None):
    c = dict(op="catalog", mode=mode, R=R, V=V, D=D, dtype=dtype, bias=bias)
    return dict(c, name=name) if name else c


def _ortho(shapes, name=None):
    c = dict(op="ortho", shapes=",".join(f"{m}x{n}" for m, n in shapes))
    return dict(c, name=name) if name else c


def listed():
    return [
        # the train loader's lists: one positive and four sampled negatives per row; launch latency is all there is
        _logprob("train", 1024, 5, "fp32", name="list_step_n5"),
        # the evaluation loop's lists: every ML-1M user's held-out item among 99 negatives, ten best kept
        _logprob("score", 6040, 100, "fp32", k=10, name="eval_n100_top10"),
        # serving: one user's scores over a catalogue of a million items, fifty best with their log-probabilities
        _logprob("score", 1, 1000003, "fp32", T=4, k=50, name="serve_one_user_top50"),
        # list-wise loss with an entropy term over catalogue-wide scores whose rows end at different columns
        _logprob("train", 2048, 50021, "bf16", ragged=True, name="ragged_catalog_loss"),
        # a handful of users scored against the ML-1M catalogue (narrow embeddings): the smallest call
        _catalog("score", 7, 3706, 16, "fp32", True, name="score_few_users"),
        # the ML-1M-shaped MF train step (B = 1024, D = 64, item biases) under the softmax over its whole catalogue
        _catalog("train", 1024, 3706, 64, "fp32", True, name="train_ml1m_d64"),
        # a wide bf16 item tower, batch of 8192 against 10^5 items
        _catalog("train", 8192, 100003, 128, "bf16", False, name="train_100k_d128"),
        # a million-row fp32 item table, the largest call
        _catalog("train", 2048, 1000003, 64, "fp32", False, name="train_1m_d64"),
        # NeuMF's towers at embedding width 64: four small matrices, launch latency
        _ortho([(64, 128), (32, 64), (32, 64), (1, 64)], name="neumf_towers"),
        # odd and lopsided layers (one-column inputs, dense-feature layers, odd widths)
        _ortho([(845, 13), (63, 257), (300, 7), (1, 1), (129, 130)], name="odd_layers"),
        # DCN-v2 on Criteo-shaped rows: three cross layers and the 1024-512-256 tower
        _ortho([(432, 432), (432, 432), (432, 432), (1024, 432), (512, 1024), (256, 512)], name="dcnv2_layers"),
        # the widest tower of the benchmark's DeepFM (3344-3344-1672-836)
        _ortho([(3344, 3344), (1672, 3344), (836, 1672)], name="deepfm_wide_tower"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("logprob", "catalog", "ortho"))
    if op == "logprob":
        V = _log_int(rng, 1, 1000003)
        R = _log_int(rng, 1, max(1, min(8192, 100_000_000 // V)))
        mode = rng.choice(("score", "train"))
        T = rng.choice((1, 1, 2, 7))
        return _logprob(mode, R, V, rng.choice(("fp32", "bf16")), T=T, k=rng.choice((0, 1, 10, 50)) if mode == "score" else 0,
                        ragged=rng.random() < 0.5)
    if op == "catalog":
        D = _log_int(rng, 8, 256)
        R = _log_int(rng, 1, 8192)
        V = _log_int(rng, 2, max(2, min(1000003, 100_000_000_000 // (R * D), 1_500_000_000 // R)))
        return _catalog(rng.choice(("score", "train", "train")), R, V, D, rng.choice(("fp32", "bf16")), rng.random() < 0.5)
    shapes = []
    for _ in range(rng.randint(1, 6)):
        shapes.append((_log_int(rng, 1, 1500), _log_int(rng, 1, 1500)))
    return _ortho(shapes)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _skewed(n, size, g):
    """Item codes with the popularity skew of implicit feedback (cubed uniform numbers)."""
    u = torch.rand(size, generator=g, device="cuda", dtype=torch.float64)
    return (u * u * u * n).long().clamp_(max=n - 1)


def prepare(case, seed):
    g = _gen(seed)
    dev = "cuda"
    if own:
        from recsys_amd import ops
        ops.set_index_check("deferred")       # as train_loop runs: index errors are read once per epoch
    if case["op"] == "logprob":
        R, V, T, dt = case["R"], case["V"], case["T"], DTYPES[case["dtype"]]
        logits = (torch.randn(R, V, generator=g, device=dev) * 2.5).to(dt)
        lengths = None
        if case["ragged"]:
            lengths = torch.randint(0, V + 1, (R,), generator=g, device=dev)
            targets = (torch.rand(R, T, generator=g, device=dev, dtype=torch.float64) * lengths.clamp(min=1)[:, None]).long()
        else:
            targets = _skewed(V, (R, T), g)
        st = dict(case=case, logits=logits, targets=targets, lengths=lengths)
        if case["mode"] == "train":
            logits.requires_grad_(True)
            st["g_logprob"] = -torch.rand(R, T, generator=g, device=dev) / R      # weighted mean of -log p ...
            st["g_entropy"] = torch.full((R,), -0.01 / R, device=dev)             # ... minus a little entropy
        return st
    if case["op"] == "catalog":
        R, V, D, dt = case["R"], case["V"], case["D"], DTYPES[case["dtype"]]
        x = torch.randn(R, D, generator=g, device=dev).to(dt)
        table = (torch.randn(V, D, generator=g, device=dev) * (2.0 / math.sqrt(D))).to(dt)
        bias = torch.randn(V, generator=g, device=dev) if case["bias"] else None
        st = dict(case=case, x=x, table=table, bias=bias, targets=_skewed(V, (R,), g))
        if case["mode"] == "train":
            for t in (x, table, bias):
                if t is not None:
                    t.requires_grad_(True)
            st["g_logprob"] = -torch.rand(R, generator=g, device=dev) / R
        return st
    mats = []
    for m, n in _shapes(case):
        # a gradient of a layer: a few strong directions over noise
        r = max(1, min(m, n) // 8)
        a = torch.randn(m, r, generator=g, device=dev) * torch.logspace(0, -1.5, r, device=dev)
        b = torch.randn(r, n, generator=g, device=dev)
        mats.append((a @ b + 0.3 * torch.randn(m, n, generator=g, device=dev)) * 1e-3)
    return dict(case=case, mats=mats)


# ------------------------------------------------------------------ plain forms
def _plain_topk(l, k):
    """Indices of the k largest entries per row, the lower column first among equal ones; -1 where nothing is left."""
    R, V = l.shape
    bits = (l + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)           # monotone in the value
    key = order * (1 << 32) + (V - 1 - torch.arange(V, device=l.device))
    idx = torch.full((R, k), -1, dtype=torch.int64, device=l.device)
    val = torch.full((R, k), -math.inf, device=l.device)
    n = min(k, V)
    if n:
        top = torch.topk(key, n, dim=1).indices
        v = torch.gather(l, 1, top)
        live = v > -math.inf
        idx[:, :n] = torch.where(live, top, idx[:, :n])
        val[:, :n] = torch.where(live, v, val[:, :n])
    return idx, val


def _plain_logprob(st):
    c = st["case"]
    l = st["logits"].detach().float()
    R, V = l.shape
    if st["lengths"] is not None:
        l = torch.where(torch.arange(V, device=l.device)[None, :] < st["lengths"][:, None], l, torch.full_like(l, -math.inf))
    m = l.max(1).values
    alive = m > -math.inf
    shift = torch.where(alive, m, torch.zeros_like(m))
    d = l - shift[:, None]
    e = torch.exp(d)
    s = e.sum(1)
    lse = shift + torch.log(s)
    ed = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1)
    entropy = torch.where(alive, torch.log(s) - ed / s, torch.zeros_like(s))
    lt = torch.gather(l, 1, st["targets"])
    logprob = torch.where(lt > -math.inf, lt - lse[:, None], torch.full_like(lt, -math.inf))
    if c["mode"] == "score":
        if not c["k"]:
            return logprob, entropy, lse
        idx, val = _plain_topk(l, c["k"])
        top = torch.where(idx >= 0, val - lse[:, None], val)
        return logprob, entropy, lse, top, idx
    g, gh = st["g_logprob"], st["g_entropy"]
    p = torch.where(alive[:, None], e / s[:, None], torch.zeros_like(e))
    lp = torch.where(p > 0, d - torch.log(s)[:, None], torch.zeros_like(d))
    dl = -p * (g.sum(1, keepdim=True) + gh[:, None] * (lp + entropy[:, None]))
    onehot = torch.where(alive[:, None] & (lt > -math.inf), g, torch.zeros_like(g))
    dl.scatter_add_(1, st["targets"], onehot)
    return logprob, entropy, lse, dl.to(st["logits"].dtype)


def _plain_catalog(st):
    c = st["case"]
    x, t = st["x"].detach().float(), st["table"].detach().float()
    s = x @ t.t()
    if st["bias"] is not None:
        s = s + st["bias"].detach()
    m = s.max(1, keepdim=True).values
    rows = torch.arange(s.shape[0], device=s.device)
    st_t = s[rows, st["targets"]]
    e = torch.exp(s - m)
    z = e.sum(1, keepdim=True)
    lse = (m + torch.log(z))[:, 0]
    logprob = st_t - lse
    if c["mode"] == "score":
        return logprob, lse
    g = st["g_logprob"]
    dl = e * (-g[:, None] / z)
    dl[rows, st["targets"]] += g
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for v in range(0, t.shape[0], 32768):          # a sum over the whole catalogue: its pieces are added in 64 bits
        dx += dl[:, v:v + 32768] @ t[v:v + 32768]
    out = [logprob, lse, dx.to(st["x"].dtype), (dl.t() @ x).to(st["table"].dtype)]
    if st["bias"] is not None:
        out.append(dl.sum(0))
    return tuple(out)


def _plain_ortho(G):
    a, b, c = NS_COEFFS
    X = G.t() if G.shape[0] > G.shape[1] else G
    X = X / (torch.sqrt((X * X).sum()) + NS_EPS)
    for _ in range(NS_STEPS):
        A = X @ X.t()
        X = a * X + (b * A + c * (A @ A)) @ X
    return (X.t() if G.shape[0] > G.shape[1] else X).contiguous()


# ------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if own:
        from recsys_amd import autograd as rxa, ops
        if c["op"] == "logprob":
            r = rxa.log_probs(state["logits"], state["targets"], lengths=state["lengths"], k=c["k"])
            if c["mode"] == "train":
                dl, = torch.autograd.grad((r.logprob, r.entropy), state["logits"], (state["g_logprob"], state["g_entropy"]))
                return r.logprob.detach(), r.entropy.detach(), r.lse.detach(), dl
            if not c["k"]:
                return r.logprob, r.entropy, r.lse
            return r.logprob, r.entropy, r.lse, r.top_logprob, r.top_index
        if c["op"] == "catalog":
            leaves = [t for t in (state["x"], state["table"], state["bias"]) if t is not None]
            lp, lse = rxa.catalog_logprob(state["x"], state["table"], state["targets"], bias=state["bias"])
            if c["mode"] == "score":
                return lp, lse
            return (lp.detach(), lse.detach()) + torch.autograd.grad(lp, leaves, state["g_logprob"])
        return ops.orthogonalize(state["mats"], steps=NS_STEPS, coeffs=NS_COEFFS, eps=NS_EPS)
    if c["op"] == "logprob":
        return _plain_logprob(state)
    if c["op"] == "catalog":
        return _plain_catalog(state)
    return [_plain_ortho(G) for G in state["mats"]]


def work(case):
    if case["op"] == "logprob":
        R, V, T, k = case["R"], case["V"], case["T"], case["k"]
        size = 4 if case["dtype"] == "fp32" else 2
        live = R * V / 2 if case["ragged"] else R * V           # rows end anywhere: half the columns on average
        small = R * (T * 12 + 8 + k * 12) + (8 * R if case["ragged"] else 0)
        if case["mode"] == "score":
            return {"bytes": int(live * size + small), "flops": int(6 * live)}
        return {"bytes": int(live * size + R * V * size + small + R * (T * 4 + 4)), "flops": int(12 * live)}
    if case["op"] == "catalog":
        R, V, D = case["R"], case["V"], case["D"]
        size = 4 if case["dtype"] == "fp32" else 2
        b = (R + V) * D * size + R * 16 + (4 * V if case["bias"] else 0)
        if case["mode"] == "score":
            return {"bytes": b, "flops": 2 * R * V * D}
        return {"bytes": b + (R + V) * D * size + R * 4 + (4 * V if case["bias"] else 0), "flops": 6 * R * V * D}
    bytes_, flops = 0, 0
    for m, n in _shapes(case):
        m, n = min(m, n), max(m, n)
        bytes_ += 8 * m * n
        flops += NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n)     # two symmetric products and a full one
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    inf = float("inf")
    if case["op"] == "logprob":
        R, V = case["R"], case["V"]
        outs = []
        for r0 in range(0, R, max(1, 40_000_000 // V)):
            r1 = min(R, r0 + max(1, 40_000_000 // V))
            z = st["logits"].detach()[r0:r1].double()
            tg = st["targets"][r0:r1]
            n = torch.full((r1 - r0, 1), V, device=z.device) if st["lengths"] is None else st["lengths"][r0:r1, None]
            hidden = torch.arange(V, device=z.device).expand_as(z) >= n
            z = z.masked_fill(hidden, -inf)
            empty = n[:, 0] == 0
            lse = torch.logsumexp(z, 1)
            logp = (z - lse[:, None]).masked_fill(hidden, -inf)
            p = logp.exp()
            H = -(p * logp.masked_fill(p == 0, 0.0)).sum(1)
            H[empty] = 0.0
            lp = logp.gather(1, tg)
            if case["mode"] == "score":
                o = [lp, H, lse]
                if case["k"]:
                    k = min(case["k"], V)
                    val, idx = torch.sort(z, dim=1, descending=True, stable=True)
                    val, idx = val[:, :k], idx[:, :k]
                    dead = val == -inf
                    pad = (0, case["k"] - k)
                    o.append(torch.nn.functional.pad((val - lse[:, None]).masked_fill(dead, -inf), pad, value=-inf))
                    o.append(torch.nn.functional.pad(idx.masked_fill(dead, -1), pad, value=-1))
            else:
                g, gh = st["g_logprob"][r0:r1].double(), st["g_entropy"][r0:r1].double()
                onehots = torch.zeros_like(z).scatter_add_(1, tg, g)
                grad = onehots - p * g.sum(1, keepdim=True) - gh[:, None] * p * (logp.masked_fill(p == 0, 0.0) + H[:, None])
                o = [lp, H, lse, grad.masked_fill(hidden, 0.0)]
            outs.append(o)
        return tuple(torch.cat(parts) for parts in zip(*outs))
    if case["op"] == "catalog":
        R, V, D = case["R"], case["V"], case["D"]
        x, t = st["x"].detach().double(), st["table"].detach().double()
        b = torch.zeros(V, dtype=torch.float64, device=x.device) if st["bias"] is None else st["bias"].detach().double()
        step = max(1, 200_000_000 // R)
        parts = [torch.logsumexp(x @ t[v:v + step].t() + b[v:v + step], 1) for v in range(0, V, step)]
        lse = torch.logsumexp(torch.stack(parts, 1), 1)
        lp = (x * t[st["targets"]]).sum(1) + b[st["targets"]] - lse
        if case["mode"] == "score":
            return lp, lse
        g = st["g_logprob"].double()
        dx, dt, db = torch.zeros_like(x), torch.empty_like(t), torch.empty_like(b)
        for v in range(0, V, step):
            w = torch.exp(x @ t[v:v + step].t() + b[v:v + step] - lse[:, None]) * -g[:, None]
            here = (st["targets"] >= v) & (st["targets"] < v + step)
            rows = here.nonzero()[:, 0]
            w[rows, st["targets"][rows] - v] += g[rows]
            dx += w @ t[v:v + step]
            dt[v:v + step] = w.t() @ x
            db[v:v + step] = w.sum(0)
        return (lp, lse, dx, dt) + (() if st["bias"] is None else (db,))
    outs = []
    ca, cb, cc = NS_COEFFS
    for G in st["mats"]:
        # through the singular values: each step maps s to a s + b s^3 + c s^5 and leaves the vectors alone
        if min(G.shape) > 1200:
            return None
        U, s, Vh = torch.linalg.svd(G.double().cpu(), full_matrices=False)
        s = s / (torch.sqrt((s * s).sum()) + NS_EPS)
        for _ in range(NS_STEPS):
            s = ca * s + cb * s ** 3 + cc * s ** 5
        outs.append(((U * s) @ Vh).to(G.device))
    return outs
