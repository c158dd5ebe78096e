"""The token operators as they are used together: a tied table looked up, distilled and averaged in one
training step, and a decode loop that samples a token, looks it up and goes on; eager and captured."""
import pytest
import torch

import swvr_b200 as swvr

pytestmark = pytest.mark.gpu
f64 = torch.float64


def parts(dtype, N=96, K=64, V=1500, D=16, Kt=8):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=f64)  # noqa: E731
    put = lambda x: x.to(dtype).cuda().requires_grad_(True)  # noqa: E731
    W, E, b, g = put(3 * K ** -0.5 * r(V, K)), put(r(V, D)), put(0.5 * r(V)), put(1 + 0.1 * r(K))
    tok = torch.randint(0, V, (N,), generator=gen).cuda()
    ids = torch.stack([torch.randperm(V, generator=gen)[:Kt] for _ in range(N)]).cuda()
    return W, E, b, g, tok, ids, (2 * r(N, Kt)).float().cuda(), r(N, D).float().cuda()


def step(W, E, b, g, tok, ids, t, target, dtype=None):
    """Lookup in the tied W, a norm, then distillation over W and the readout's loss over (W, E)."""
    K = W.shape[1]
    x = swvr.embedding_lookup(tok, W, scale=K ** 0.5)
    h = torch.nn.functional.rms_norm(x, (K,), g, 1e-5)
    loss = swvr.softmax_distill(h, W, ids, t, b, temperature=1.5)
    return loss + 0.1 * swvr.softmax_readout_mse(h, W, E, target, b)


def reference(W, E, b, g, tok, ids, t, target):
    W, E, b, g, t, target = (x.detach().double().requires_grad_(x.requires_grad) for x in (W, E, b, g, t, target))
    K, T = W.shape[1], 1.5
    x = W[tok] * K ** 0.5
    h = x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + 1e-5) * g
    S = h @ W.T + b
    logq = torch.log_softmax(t / T, 1)
    each = T * T * (logq.exp() * (logq - torch.log_softmax(S / T, 1).gather(1, ids))).sum(1)
    loss = each.mean() + 0.1 * ((torch.softmax(S, 1) @ E - target) ** 2).mean()
    return loss, torch.autograd.grad(loss, (W, E, b, g))


@pytest.mark.parametrize("dtype,tol", [(f64, 1e-10), (torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
def test_tied_training_step(dtype, tol):
    """W takes gradients from three places: the lookup, the distillation and the readout.  Tolerances: the
    readout's own (fp32 1e-4, bf16 2e-2 norm-wise), which the step contains."""
    args = parts(dtype)
    loss = step(*args)
    got = torch.autograd.grad(loss, args[:4])
    want_loss, want = reference(*args)
    assert abs(float(loss.detach()) - float(want_loss.detach())) <= tol * abs(float(want_loss.detach()))
    for name, a, r in zip("WEbg", got, want):
        assert a.dtype == dtype
        assert float((a.double() - r).norm()) <= tol * float(r.norm()), name


def test_captured_training_step_beside_an_eager_one():
    args = parts(torch.bfloat16)
    W, E, b, g, tok, ids, t, target = args
    leaves = args[:4]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(step(*args), leaves)
        # an eager graph over the same leaves, kept while the capture runs (made on the side stream: one made on the
        # default stream ties the leaves' accumulation to it, and torch then refuses any capture of their backward)
        alive = step(*args)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss_g = step(*args)
        grads_g = torch.autograd.grad(loss_g, leaves)
    with torch.cuda.stream(s):
        assert len(torch.autograd.grad(alive, leaves)) == 4  # the eager graph is whole
    torch.cuda.synchronize()
    for seed in (3, 4):
        tok.copy_(torch.randint(0, W.shape[0], tok.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [loss_g.detach().clone(), *(x.clone() for x in grads_g)]
        loss = step(*args)
        for a, c in zip(got, [loss.detach(), *torch.autograd.grad(loss, leaves)]):
            assert torch.equal(a, c)
    del graph


def decode(W, b, tok, u, top_k, steps):
    """Each step looks the last token up and samples the next one from the tied head."""
    out = []
    for i in range(steps):
        x = swvr.embedding_lookup(tok, W, scale=0.25 * W.shape[1] ** 0.5)
        tok = swvr.softmax_sample(torch.tanh(x), W, u[i], b, temperature=0.8, top_k=top_k, top_p=0.95)
        out.append(tok)
    return torch.stack(out)


def test_decode_loop_eager_and_captured():
    W, E, b, *_ = parts(torch.bfloat16)
    W, b = W.detach(), b.detach()
    gen = torch.Generator(device="cuda").manual_seed(5)
    tok = torch.randint(0, W.shape[0], (12,), generator=gen, device="cuda")
    u = torch.rand(6, 12, generator=gen, device="cuda")
    k = torch.randint(1, 60, (12,), generator=gen, device="cuda")
    want = decode(W, b, tok, u, k, 6)
    assert want.dtype == torch.int64 and bool(((want >= 0) & (want < W.shape[0])).all())
    # the first step again from its own scores: the same tokens as sampling given logits
    x = torch.tanh(swvr.embedding_lookup(tok, W, scale=0.25 * W.shape[1] ** 0.5))
    S = x.double() @ W.double().T + b.double()
    near = swvr.sample_logits(S.float(), u[0], temperature=0.8, top_k=k, top_p=0.95)
    assert int((near != want[0]).sum()) <= 1  # fp32 scores of another summation order
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        decode(W, b, tok, u, k, 2)
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        got = decode(W, b, tok, u, k, 6)
    with torch.cuda.graph(two):  # a second graph with workspaces of its own
        got2 = decode(W, b, tok, u, k, 6)
    for graph, out in ((one, got), (two, got2), (one, got)):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    u.copy_(torch.rand(6, 12, generator=gen, device="cuda"))
    one.replay()
    two.replay()
    torch.cuda.synchronize()
    again = decode(W, b, tok, u, k, 6)
    assert torch.equal(got, again) and torch.equal(got2, again)
    del one, two


def test_two_streams_at_once():
    """The same operators on two streams, interleaved: each call has its own workspace and stream."""
    args = parts(torch.bfloat16)
    W, E, b, g, tok, ids, t, target = args
    u = torch.rand(96, device="cuda")
    want = (step(*args).detach(), swvr.softmax_sample(torch.tanh(W.detach()[tok]), W.detach(), u, b.detach(), top_k=9))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            loss = step(*args)
            grads = torch.autograd.grad(loss, args[:4])
            got.append((loss.detach(), swvr.softmax_sample(torch.tanh(W.detach()[tok]), W.detach(), u, b.detach(), top_k=9), grads))
    torch.cuda.synchronize()
    for loss, token, grads in got:
        assert torch.equal(loss, want[0]) and torch.equal(token, want[1])
        assert all(torch.equal(a, c) for a, c in zip(grads, got[0][2]))


def test_a_dispatch_mode_sees_the_operators():
    """Tracers and counters that work by a dispatch mode get the custom ops, and the same results."""
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    args = parts(torch.bfloat16)
    u = torch.rand(96, device="cuda")
    run = lambda: (*torch.autograd.grad(step(*args), args[:4]),  # noqa: E731
                   swvr.softmax_sample(torch.tanh(args[0].detach()[args[4]]), args[0].detach(), u, top_k=9))
    want = run()
    with Record():
        got = run()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    for op in ("embed", "embed_bwd", "distill", "distill_bwd", "sample"):
        assert f"swvr_b200.{op}.default" in seen
