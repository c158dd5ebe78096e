"""What is measured of the token operators beside the readout: the embedding lookup and its gradient by token, distillation
of the head from a teacher's top logits, and sampling of a token from the head or from given logits.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program has in hand before
the call, ``run`` makes one pass: in plain torch operations, or through the library where ``own`` is true.  ``exact`` states the
same results in 64 bits, ``work`` the bytes and operations a pass cannot do without.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a decode step of a server: one token of each of 64 requests looked up in the tied table
        dict(name="embed decode", op="embed", train=False, N=64, V=152064, D=2560, dtype="bf16", pad=0.0),
        # a training batch of 8 x 2048 tokens, the table as wide as the trunk
        dict(name="embed train", op="embed", train=True, N=16384, V=152064, D=2560, dtype="bf16", pad=0.0),
        # an fp32 codebook of odd sizes, a batch padded to two fifths
        dict(name="embed train fp32 padded", op="embed", train=True, N=5001, V=10007, D=200, dtype="fp32", pad=0.4),
        # a small head trained exactly in fp32
        dict(name="distill fp32", op="distill", train=True, N=256, K=64, V=1000, Kt=8, dtype="fp32", bias=True, T=2.0),
        # a ragged fp16 batch
        dict(name="distill fp16 ragged", op="distill", train=True, N=517, K=512, V=10007, Kt=20, dtype="fp16", bias=True, T=1.0),
        # evaluation: the loss of each token
        dict(name="distill eval", op="distill", train=False, N=2048, K=1024, V=19008, Kt=64, dtype="bf16", bias=False, T=1.0),
        # a training step of a large head
        dict(name="distill train", op="distill", train=True, N=8192, K=2560, V=152064, Kt=64, dtype="bf16", bias=True, T=1.5),
        # one request's next token
        dict(name="sample head 1", op="head", N=1, K=2560, V=152064, dtype="bf16", bias=True, T=0.8, k=50, p=0.95, m=0.0, rows=False),
        # a server's batch, settings of each request
        dict(name="sample head 64", op="head", N=64, K=4096, V=128256, dtype="bf16", bias=False, T=0.9, k=40, p=1.0, m=0.05, rows=True),
        # given logits, a nucleus
        dict(name="sample logits 16 fp32", op="logits", N=16, V=152064, dtype="fp32", T=0.7, k=0, p=0.9, m=0.0, rows=False),
        # rollouts: many rows, the whole distribution
        dict(name="sample logits 256", op="logits", N=256, V=128256, dtype="bf16", T=1.0, k=0, p=1.0, m=0.0, rows=False),
        # a small vocabulary, each row its own settings
        dict(name="sample logits 300 rows", op="logits", N=300, V=10007, dtype="bf16", T=1.0, k=100, p=0.9, m=0.02, rows=True),
    ]


def draw(rng):
    def spread(lo, hi, odd=True):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, n | 1 if odd and rng.random() < 0.5 else n))

    op = rng.choice(["embed", "embed", "distill", "distill", "head", "logits"])
    if op == "embed":
        return dict(op=op, train=rng.random() < 0.7, N=spread(1, 16384), V=spread(1000, 152064), D=spread(16, 2560),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), pad=rng.choice([0.0, 0.0, 0.3]))
    if op == "distill":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        big = dtype != "fp32"
        return dict(op=op, train=rng.random() < 0.7, N=spread(1, 8192 if big else 1024), K=8 * spread(8, 320 if big else 64, odd=False),
                    V=spread(1000, 152064 if big else 10007), Kt=spread(1, 128), dtype=dtype, bias=rng.random() < 0.5,
                    T=rng.choice([1.0, 1.5, 2.0]))
    T = rng.choice([0.0, 0.6, 0.8, 1.0])
    # from the head every case has a filter: without one the token hangs on the last bits of the product
    filt = rng.choice(["k", "m", "km", "kp"] if op == "head" else ["k", "p", "m", "kp", "none"])
    f = dict(T=T, k=spread(1, 200) if "k" in filt else 0, p=round(rng.uniform(0.5, 0.95), 2) if "p" in filt else 1.0,
             m=round(rng.uniform(0.01, 0.2), 3) if "m" in filt else 0.0, rows=rng.random() < 0.5)
    if op == "head":
        return dict(op=op, N=spread(1, 128), K=8 * spread(8, 512, odd=False), V=spread(1000, 128256), dtype=rng.choice(["bf16", "fp16"]),
                    bias=rng.random() < 0.5, **f)
    return dict(op=op, N=spread(1, 256), V=spread(1000, 152064), dtype=rng.choice(["bf16", "fp32"]), **f)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    N, V = case["N"], case["V"]
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "embed":
        D = case["D"]
        # word frequencies: the r-th token about 1 / r as often as the first, low ids the frequent ones
        tokens = (torch.exp(rand(N) * math.log(V)).long() - 1).clamp_(0, V - 1)
        if case["pad"]:
            tokens = torch.where(rand(N) < case["pad"], torch.full_like(tokens, 1), tokens)
        s.update(tokens=tokens, E=(0.02 * randn(V, D)).to(dt).requires_grad_(case["train"]), scale=D ** 0.5, padding=1 if case["pad"] else None,
                 g=randn(N, D).to(dt) if case["train"] else None)
        return s
    if case["op"] == "distill":
        K, Kt = case["K"], case["Kt"]
        train = case["train"]
        slot = torch.arange(Kt, device="cuda")
        ids = ((slot + rand(N, Kt)) * (V / Kt)).long().clamp_(0, V - 1)  # a token of each of Kt ranges: no token twice
        ids = ids.gather(1, rand(N, Kt).argsort(dim=1))
        s.update(h=randn(N, K).to(dt).requires_grad_(train), W=(3 * K ** -0.5 * randn(V, K)).to(dt).requires_grad_(train),
                 b=(0.5 * randn(V)).to(dt).requires_grad_(train) if case["bias"] else None, ids=ids,
                 t=(3.0 * randn(N, Kt)).sort(dim=1, descending=True).values, w=(rand(N) < 0.9).float().index_fill_(0, slot[:1], 1.0) if train else None,
                 up=torch.full((), 4096.0 if case["dtype"] == "fp16" else 1.0, device="cuda"))  # the loss scale of fp16 training
        return s
    rows = case["rows"]
    s.update(u=rand(N),
             T=(case["T"] * (0.75 + 0.5 * rand(N))) if rows else case["T"],
             k=(torch.clamp((case["k"] * (0.5 + rand(N))).int(), min=1) if case["k"] else None) if rows else (case["k"] or None),
             p=((case["p"] * (0.9 + 0.1 * rand(N))) if case["p"] < 1 else None) if rows else (case["p"] if case["p"] < 1 else None),
             m=((case["m"] * (0.5 + rand(N))) if case["m"] else None) if rows else (case["m"] or None))
    if case["op"] == "head":
        K = case["K"]
        # the scores of a trained head: a few tokens hold most of the probability
        s.update(h=randn(N, K).to(dt), W=(5 * K ** -0.5 * randn(V, K)).to(dt), b=(0.5 * randn(V)).to(dt) if case["bias"] else None)
    else:
        s.update(logits=(4 * randn(N, V)).to(dt))
    return s


# ------------------------------------------------------------------ plain forms

def _embed_plain(s):
    tokens, E, D = s["tokens"], s["E"].detach(), s["D"]
    out = (E[tokens].float() * s["scale"]).to(E.dtype)
    if not s["train"]:
        return out
    grad = s["g"].float() * s["scale"]
    if s["padding"] is not None:
        grad = grad * (tokens != s["padding"])[:, None]
    return out, torch.zeros(s["V"], D, device=E.device).index_add_(0, tokens, grad).to(E.dtype)


def _distill_plain(s):
    h, W, b, T, ids = s["h"].detach(), s["W"].detach(), s["b"], s["T"], s["ids"]
    hf, Wf = h.float(), W.float()
    z = hf @ Wf.T
    if b is not None:
        z += b.detach().float()
    z /= T
    top = z.max(dim=1, keepdim=True).values
    lse = top + (z - top).exp().sum(dim=1, keepdim=True).log()
    t = s["t"].float() / T
    logq = t - t.max(dim=1, keepdim=True).values
    logq = logq - logq.exp().sum(dim=1, keepdim=True).log()
    q = logq.exp()
    each = T * T * (q * (logq - z.gather(1, ids) + lse)).sum(dim=1)
    if not s["train"]:
        return each
    w = s["w"]
    den = w.sum()
    loss = (each * w).sum() / den
    z = (z - lse).exp_()
    z.scatter_add_(1, ids, -q)
    z *= (s["up"] * T * w / den)[:, None]
    out = [loss, (z @ Wf).to(h.dtype), (z.T @ hf).to(W.dtype)]
    return out + ([z.sum(dim=0).to(b.dtype)] if b is not None else [])


def _sample_plain(x, s):
    # 64 bits: the token hangs on the cumulative sums next to u
    x, N, V = x.double(), s["N"], s["V"]
    col = lambda v: v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((N, 1), float(v), dtype=torch.float64, device=x.device)  # noqa: E731
    T = col(s["T"])
    greedy = T <= 0
    best = x.max(dim=1, keepdim=True).values
    z = (x - best) / torch.where(greedy, torch.ones_like(T), T)
    z, order = z.sort(dim=1, descending=True, stable=True)
    w = z.exp()
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["k"] is not None:
        keep &= torch.arange(V, device=x.device) < col(s["k"])
    if s["p"] is not None:
        kept = w * keep
        keep &= kept.cumsum(dim=1) - kept < col(s["p"]) * kept.sum(dim=1, keepdim=True)
    if s["m"] is not None:
        keep &= w >= col(s["m"])
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    cdf = w.cumsum(dim=1)
    past = (cdf > s["u"].double()[:, None] * cdf[:, -1:]) & (w > 0)
    index = torch.arange(V, device=x.device)
    token = torch.where(past, index, V).min(dim=1).values
    first = torch.where(x == best, index, V).min(dim=1).values
    return torch.where(greedy[:, 0], first, token)


def _plain(s):
    if s["op"] == "embed":
        return _embed_plain(s)
    if s["op"] == "distill":
        return _distill_plain(s)
    if s["op"] == "logits":
        return _sample_plain(s["logits"], s)
    x = s["h"].float() @ s["W"].float().T
    return _sample_plain(x if s["b"] is None else x + s["b"].float(), s)


def _own(s):
    import swvr_b200 as swvr
    if s["op"] == "embed":
        out = swvr.embedding_lookup(s["tokens"], s["E"], scale=s["scale"], padding_idx=s["padding"])
        return (out, torch.autograd.grad(out, s["E"], s["g"])[0]) if s["train"] else out
    if s["op"] == "distill":
        args = (s["h"], s["W"], s["ids"], s["t"], s["b"])
        if not s["train"]:
            return swvr.softmax_distill(*args, temperature=s["T"], reduction="none")
        loss = swvr.softmax_distill(*args, temperature=s["T"], weight=s["w"])
        return [loss.detach(), *torch.autograd.grad(loss, [x for x in (s["h"], s["W"], s["b"]) if x is not None], s["up"])]
    kw = dict(temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
    if s["op"] == "logits":
        return swvr.sample_logits(s["logits"], s["u"], **kw)
    return swvr.softmax_sample(s["h"], s["W"], s["u"], s["b"], **kw)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    if case["op"] not in ("embed", "distill"):
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "embed":
        E = s["E"].detach().double()
        out = s["scale"] * E.index_select(0, s["tokens"])
        if not case["train"]:
            return out
        real = torch.arange(case["N"], device="cuda")
        if s["padding"] is not None:
            real = real[s["tokens"] != s["padding"]]
        dE = torch.zeros_like(E)
        dE.index_put_((s["tokens"][real],), s["g"].double()[real], accumulate=True)
        return out, s["scale"] * dE
    T, rows = case["T"], torch.arange(case["N"], device="cuda")[:, None]
    h, W = s["h"].detach().double(), s["W"].detach().double()
    logp = torch.mm(h, W.t())
    if s["b"] is not None:
        logp.add_(s["b"].detach().double())
    logp = torch.log_softmax(logp.div_(T), dim=1)
    logq = torch.log_softmax(s["t"].double() / T, dim=1)
    q = logq.exp()
    kl = T ** 2 * torch.sum(q * (logq - logp[rows, s["ids"]]), dim=1)
    if not case["train"]:
        return kl
    w = s["w"].double() / s["w"].double().sum()
    d = logp.exp_()
    d[rows, s["ids"]] -= q
    d.mul_((float(s["up"]) * T * w)[:, None])
    return [torch.dot(kl, w), torch.mm(d, W), torch.mm(d.t(), h)] + ([d.sum(0)] if s["b"] is not None else [])


def work(case):
    e, N, V = SIZE[case["dtype"]], case["N"], case["V"]
    if case["op"] == "embed":
        D = case["D"]
        b = 8 * N + 2 * e * N * D
        return {"bytes": b + (8 * N + e * N * D + e * V * D if case["train"] else 0), "flops": N * D * (2 if case["train"] else 1)}
    if case["op"] == "logits":
        return {"bytes": e * N * V + 12 * N, "flops": 4 * N * V}
    K = case["K"]
    if case["op"] == "head":
        return {"bytes": e * (V * K + N * K + (V if case["bias"] else 0)) + 12 * N, "flops": 2 * N * V * K}
    b = e * (N * K + V * K + (V if case["bias"] else 0)) + 12 * N * case["Kt"] + 4 * N
    return {"bytes": 2 * b if case["train"] else b, "flops": (6 if case["train"] else 2) * N * V * K}
