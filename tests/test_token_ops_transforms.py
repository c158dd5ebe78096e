"""The token operators under torch.func transforms, on the CPU: the kernels' wrappers are replaced by plain formulas, so
that what is tested is the way from the entry points through the custom ops.  And the same on the GPU with the kernels."""
import pytest
import torch

import swvr_b200 as swvr
from swvr_b200 import distill, embedding, sampling


def plain_embed(tokens, E, scale):
    return scale * E[tokens]


def plain_embed_bwd(g, tokens, V, scale, padding):
    keep = (tokens != padding)[:, None] * scale * g
    return torch.zeros(V, g.shape[1], dtype=g.dtype).index_add_(0, tokens, keep)


def plain_distill(h, W, bias, ids, logits, t_lse, weight, T, s, chunk, cdt, reduction):
    z = torch.log_softmax((s * h @ W.T + (0 if bias is None else bias)) / T, 1)
    logq = torch.log_softmax(logits / T, 1)
    each = T * T * (logq.exp() * (logq - z.gather(1, ids))).sum(1)
    saved = torch.zeros(distill._saved_numel(*ids.shape), dtype=h.dtype)
    return each if reduction == 0 else each.mean(), torch.zeros(ids.shape, dtype=torch.int32), saved


def plain_distill_bwd(grad, h, W, bias, ids, logits, t_lse, weight, sid, saved, T, s, chunk, cdt, reduction, *want):
    z = (s * h @ W.T + bias) / T
    q = torch.log_softmax(logits / T, 1).exp()
    dS = T * grad[:, None] * (torch.softmax(z, 1) * q.sum(1, keepdim=True)).scatter_add(1, ids, -q)
    return [g if w else None for g, w in zip((s * dS @ W, s * dS.T @ h, dS.sum(0)), want)] + [None]


def plain_sample(logits, u, *rest):
    assert logits.data_ptr() and u.data_ptr()  # which a batched tensor does not have
    cdf = logits.softmax(1).cumsum(1)
    token = (cdf <= u[:, None]).sum(1)
    return token, torch.zeros(len(u) if rest[-1] else 0)


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def device(request, monkeypatch):
    if request.param == "cpu":
        monkeypatch.setattr(embedding, "_embed_fwd", plain_embed)
        monkeypatch.setattr(embedding, "_embed_bwd", plain_embed_bwd)
        monkeypatch.setattr(distill, "_distill_fwd", plain_distill)
        monkeypatch.setattr(distill, "_distill_bwd", plain_distill_bwd)
        monkeypatch.setattr(sampling, "_sample_logits", plain_sample)
        monkeypatch.setattr(sampling, "_sample_head", lambda h, W, bias, u, *rest: plain_sample(h @ W.T + bias, u, *rest[2:]))
    return request.param


def inputs(device, *shapes):
    gen = torch.Generator().manual_seed(0)
    return [torch.randn(*s, generator=gen, dtype=torch.float32).to(device) for s in shapes]


def test_lookup_under_vmap(device):
    E, = inputs(device, (11, 8))
    tok = torch.randint(0, 11, (3, 5), generator=torch.Generator().manual_seed(1)).to(device)
    f = lambda t: swvr.embedding_lookup(t, E, scale=2.0, padding_idx=0)  # noqa: E731
    assert torch.equal(torch.func.vmap(f)(tok), f(tok))
    E.requires_grad_(True)
    a, b = (torch.autograd.grad((g(tok) ** 2).sum(), E)[0] for g in (torch.func.vmap(f), f))
    # a row's gradients, at most 15 equal ones, added in another order
    assert bool(((a - b).abs() <= 2 * 15 * 2.0 ** -24 * b.abs()).all())


def test_distillation_under_vmap(device):
    h, W, b, t = inputs(device, (3, 4, 8), (20, 8), (20,), (3, 4, 5))
    ids = torch.randint(0, 20, (3, 4, 5), generator=torch.Generator().manual_seed(1)).to(device)
    f = lambda h, i, t: swvr.softmax_distill(h, W, i, t, b, temperature=2.0, reduction="none")  # noqa: E731
    got, want = torch.func.vmap(f)(h, ids, t), f(h, ids, t)
    assert got.shape == want.shape == (3, 4)
    # either side's scores are off by at most e = 2^-20 (|h| |W|^T + |b|) / T, its losses by T^2 twice that, dh by T (4 e) |W|
    e = 2.0 ** -20 * float((h.abs() @ W.abs().T + b.abs()).max()) / 2
    assert float((got - want).abs().max()) <= 2 * 4 * 2 * e
    h.requires_grad_(True)
    a, c = (torch.autograd.grad(g(h, ids, t).sum(), h)[0] for g in (torch.func.vmap(f), f))
    assert float((a - c).abs().max()) <= 2 * 2 * 4 * e * float(W.abs().sum(0).max())


@pytest.mark.parametrize("logprobs", [False, True])
def test_sampling_under_vmap(device, logprobs):
    x, h, W, b = inputs(device, (3, 4, 20), (3, 4, 8), (20, 8), (20,))
    u, T = torch.rand(3, 4, generator=torch.Generator().manual_seed(1)).to(device), torch.full((3, 4), 0.7, device=device)
    f = lambda x, u, T: swvr.sample_logits(x, u, temperature=T, return_logprobs=logprobs)  # noqa: E731
    g = lambda h, u, T: swvr.softmax_sample(h, W, u, b, temperature=T, return_logprobs=logprobs)  # noqa: E731
    for fn, arg in ((f, x), (g, h)):
        got, want = torch.func.vmap(fn)(arg, u, T), fn(arg, u, T)
        assert torch.equal(got[0], want[0]) and torch.allclose(got[1], want[1], atol=1e-5) if logprobs else torch.equal(got, want)


@pytest.mark.parametrize("batched", [False, True])
def test_forward_mode_is_refused_not_zero(device, batched):
    """A tangent that the operator would drop raises; one that does not reach it does no harm."""
    E, W, b, t, w = inputs(device, (11, 8), (11, 8), (11,), (5, 3), (5,))
    tok = torch.randint(0, 11, (5,), generator=torch.Generator().manual_seed(1)).to(device)
    ids = torch.randint(0, 11, (5, 3), generator=torch.Generator().manual_seed(2)).to(device)
    h = E[:5].clone()
    lookup = lambda E: swvr.embedding_lookup(tok, E)  # noqa: E731
    loss = lambda h=h, W=W, b=b, w=w: swvr.softmax_distill(h, W, ids, t, b, weight=w)  # noqa: E731
    for f, x in ((lookup, E), (loss, h), (lambda x: loss(W=x), W), (lambda x: loss(b=x), b), (lambda x: loss(w=x), w)):
        g = torch.func.vmap(f) if batched else f
        x = torch.stack([x, x]) if batched else x
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(g, (x,), (x,))
        if not batched:
            with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(torch.autograd.forward_ad.make_dual(x, x))
    beside = lambda x: x + lookup(E).sum() + loss().sum()  # noqa: E731
    beside = torch.func.vmap(beside) if batched else beside
    x = torch.ones(2, 3, device=device)
    assert torch.equal(torch.func.jvp(beside, (x,), (x,))[1], x)
