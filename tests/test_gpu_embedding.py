"""GPU tests of the embedding lookup and its gradient by token against 64-bit indexing.

Tolerances.  The lookup rounds scale * x to the accumulation type (half a step, u) and once to
the table's type (half a step, r): (u + r) |x|, plus half the smallest subnormal.  The
gradient of a row that c tokens share adds c products' worth of rounding, u each, to terms
whose absolute sum is A: (c + 2) u A, then r |sum| once."""
import pytest
import torch

import swvr_b200 as swvr
from swvr_b200 import _native as nat

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float64, torch.bfloat16, torch.float16]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def acc_half_step(dt):
    return half_step(torch.float64 if dt == torch.float64 else torch.float32)


def tiny(dt):
    return torch.finfo(dt).smallest_normal * half_step(dt)


def check_lookup(out, tokens, E, scale):
    want = E.detach().double()[tokens.long()] * scale
    lim = (half_step(E.dtype) + acc_half_step(E.dtype)) * want.abs() + tiny(E.dtype)
    assert out.dtype == E.dtype and out.shape == (*tokens.shape, E.shape[1])
    assert bool(((out.double() - want).abs() <= lim).all())


def check_grad(dE, tokens, g, V, scale, padding=None):
    t, g2 = tokens.reshape(-1).long(), g.double().reshape(-1, g.shape[-1])
    live = (t >= 0) & (t < V)
    if padding is not None:
        live &= t != padding
    t, g2 = t[live], g2[live]
    zero = torch.zeros(V, g.shape[-1], dtype=torch.float64, device=g.device)
    want = zero.clone().index_add_(0, t, g2) * scale
    size = zero.clone().index_add_(0, t, g2.abs()) * abs(scale)
    count = torch.zeros(V, dtype=torch.float64, device=g.device).index_add_(0, t, torch.ones_like(t, dtype=torch.float64))
    lim = (count[:, None] + 2) * acc_half_step(g.dtype) * size + half_step(g.dtype) * want.abs() + tiny(g.dtype)
    assert dE.shape == (V, g.shape[-1]) and dE.dtype == g.dtype
    bad = (dE.double() - want).abs() > lim * (1 + 1e-9)
    assert not bool(bad.any()), int(bad.sum())
    assert bool((dE[count == 0] == 0).all())


def make(kind, N, V, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.rand(N, generator=gen, device="cuda")
    if kind == "uniform":
        return (u * V).long().clamp_(max=V - 1)
    if kind == "zipf":
        return (torch.exp(u * torch.log(torch.tensor(float(V)))).long() - 1).clamp_(0, V - 1)
    if kind == "one":
        return torch.full((N,), V - 1, device="cuda")
    if kind == "sorted":
        return (torch.arange(N, device="cuda") * V) // max(N, 1)
    raise ValueError(kind)


def table(V, D, dtype, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(V, D, generator=gen, device="cuda", dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (7, 41, 5), (64, 1000, 16), (333, 3001, 200), (1, 9000, 2560)])
@pytest.mark.parametrize("tdt", [torch.int64, torch.int32])
def test_lookup(dtype, N, V, D, tdt):
    E, tok = table(V, D, dtype), make("uniform", N, V).to(tdt)
    for scale in (1.0, D ** 0.5):
        check_lookup(swvr.embedding_lookup(tok, E, scale=scale), tok, E, scale)


@pytest.mark.parametrize("shape", [(), (0,), (2, 3), (4, 0, 2), (2, 3, 5)])
def test_lookup_shapes(shape):
    E = table(50, 24, torch.bfloat16).requires_grad_(True)
    tok = torch.randint(0, 50, shape, device="cuda")
    out = swvr.embedding_lookup(tok, E, scale=0.5)
    check_lookup(out.detach(), tok, E, 0.5)
    g = torch.randn(out.shape, device="cuda").to(out.dtype)
    check_grad(torch.autograd.grad(out, E, g)[0], tok, g, 50, 0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_tables_tokens_and_gradients(dtype):
    """Padded rows, an odd offset (no 16-byte alignment), a transposed table, tokens with a stride,
    an expanded gradient."""
    big = table(60, 40, dtype)
    tok = torch.randint(0, 60, (9, 6), device="cuda")[:, ::2]
    for E in (big[:, :32], big[:, 1:30], big.t().contiguous().t(), big[:, 3:4], big[::2].repeat(2, 1)[:60]):
        E = E.detach().requires_grad_(True)
        out = swvr.embedding_lookup(tok, E)
        check_lookup(out.detach(), tok, E, 1.0)
        wide = torch.randn(9, 3, E.shape[1] + 5, device="cuda").to(dtype)
        for g in (wide[..., 2:2 + E.shape[1]], wide[:1, :1, :1].expand(9, 3, E.shape[1])):
            check_grad(torch.autograd.grad(out, E, g, retain_graph=True)[0], tok, g, 60, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one", "sorted"])
@pytest.mark.parametrize("N,V,D", [(1, 41, 5), (16, 300, 16), (17, 1, 8), (2049, 3001, 40), (5001, 70000, 33)])
def test_gradient(dtype, kind, N, V, D):
    tok = make(kind, N, V, seed=N)
    gen = torch.Generator(device="cuda").manual_seed(3)
    g = torch.randn(N, D, generator=gen, device="cuda", dtype=torch.float64).to(dtype)
    E = torch.zeros(V, D, dtype=dtype, device="cuda", requires_grad=True)
    for scale, padding in ((1.0, None), (1.75, V - 1), (1.0, -V)):
        out = swvr.embedding_lookup(tok, E, scale=scale, padding_idx=padding)
        dE = torch.autograd.grad(out, E, g)[0]
        check_grad(dE, tok, g, V, scale, None if padding is None else padding % V)


def test_gradient_is_the_same_on_every_run():
    tok = make("zipf", 20000, 5000)
    g = torch.randn(20000, 96, device="cuda").bfloat16()
    E = torch.zeros(5000, 96, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    runs = [torch.autograd.grad(swvr.embedding_lookup(tok, E), E, g)[0] for _ in range(4)]
    assert all(torch.equal(r, runs[0]) for r in runs)


def test_many_tokens_span_many_chunks():
    """70,001 tokens, two fifths of them one token: its sum runs over hundreds of chunks."""
    N, V, D = 70001, 260, 24
    tok = make("uniform", N, V)
    tok[torch.rand(N, device="cuda") < 0.4] = 7
    g = torch.randn(N, D, device="cuda")
    E = torch.zeros(V, D, device="cuda", requires_grad=True)
    check_grad(torch.autograd.grad(swvr.embedding_lookup(tok, E), E, g)[0], tok, g, V, 1.0)


def test_gradient_by_differences():
    """The functional is linear in E: its difference quotient in fp64 is the gradient up to rounding."""
    tok = torch.tensor([3, 0, 3, 6, 3], device="cuda")
    E = table(7, 4, torch.float64).requires_grad_(True)
    w = torch.randn(5, 4, device="cuda", dtype=torch.float64)
    f = lambda t: float((swvr.embedding_lookup(tok, t, scale=1.5) * w).sum())  # noqa: E731
    dE = torch.autograd.grad((swvr.embedding_lookup(tok, E, scale=1.5) * w).sum(), E)[0]
    for v in range(7):
        for d in range(4):
            e = torch.zeros_like(E)
            e[v, d] = 0.5
            num = f(E.detach() + e) - f(E.detach() - e)
            assert abs(num - float(dE[v, d])) < 1e-12 * 40


@pytest.mark.parametrize("grad", [False, True])
def test_tokens_out_of_range_are_reported(grad):
    E = table(20, 16, torch.float32).requires_grad_(grad)
    tok = torch.tensor([4, 20, -1, 7, 2 ** 40], device="cuda")
    bad = torch.tensor([False, True, True, False, True], device="cuda")
    out = swvr.embedding_lookup(tok, E)
    assert bool(out[bad].isnan().all())
    check_lookup(out[~bad].detach(), tok[~bad], E, 1.0)
    with pytest.raises(RuntimeError, match=r"outside \[0, V\)"):
        nat.check_device_error()
    if grad:
        g = torch.ones(5, 16, device="cuda")
        check_grad(torch.autograd.grad(out, E, g)[0], tok, g, 20, 1.0)
        with pytest.raises(RuntimeError, match=r"outside \[0, V\)"):
            nat.check_device_error()
    nat.check_device_error()


def test_empty_table_and_empty_batch():
    E = torch.zeros(0, 8, device="cuda", requires_grad=True)
    out = swvr.embedding_lookup(torch.zeros(0, dtype=torch.int64, device="cuda"), E)
    assert out.shape == (0, 8)
    assert torch.autograd.grad(out.sum(), E)[0].shape == (0, 8)
    E = torch.ones(5, 8, device="cuda", requires_grad=True)
    out = swvr.embedding_lookup(torch.zeros(0, dtype=torch.int64, device="cuda"), E)
    assert bool((torch.autograd.grad(out.sum(), E)[0] == 0).all())
    assert swvr.embedding_lookup(torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(5, 0, device="cuda")).shape == (3, 0)


def test_offsets_past_32_bits():
    """A table of 2.4e9 elements: rows whose element offset does not fit 31 bits, both ways."""
    V, D = 300000, 8192
    E = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    tok = torch.tensor([V - 1, 0, V - 1, 270001], device="cuda")
    E[V - 1] = 3
    E[270001] = 5
    E.requires_grad_(True)
    out = swvr.embedding_lookup(tok, E)
    assert [float(x) for x in out.detach()[:, 0]] == [3, 0, 3, 5] and bool((out[0] == 3).all())
    dE = torch.autograd.grad(out, E, torch.ones_like(out))[0]
    assert bool((dE[V - 1] == 2).all()) and bool((dE[270001] == 1).all()) and bool((dE[0] == 1).all())
    assert float(dE.float().sum()) == 4 * D


def test_side_stream_and_captured_step():
    """A lookup and its gradient on a side stream, and captured and replayed on new tokens while an
    eager graph of the same table lives."""
    E = table(3000, 64, torch.bfloat16).requires_grad_(True)
    tok = make("zipf", 700, 3000)
    g = torch.randn(700, 64, device="cuda").bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            out = swvr.embedding_lookup(tok, E, scale=2.0)
            (dE,) = torch.autograd.grad(out, E, g)
    torch.cuda.current_stream().wait_stream(s)
    check_lookup(out.detach(), tok, E, 2.0)
    check_grad(dE, tok, g, 3000, 2.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out_g = swvr.embedding_lookup(tok, E, scale=2.0)
        (dE_g,) = torch.autograd.grad(out_g, E, g)
    for seed in (4, 5):
        tok.copy_(make("zipf", 700, 3000, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        check_lookup(out_g.detach(), tok, E, 2.0)
        check_grad(dE_g, tok, g, 3000, 2.0)
    del graph


def test_compiled_whole():
    E = table(500, 32, torch.float32).requires_grad_(True)
    tok = make("uniform", 40, 500)

    def f(t, e):
        return (swvr.embedding_lookup(t, e, scale=3.0) ** 2).sum()

    want = torch.autograd.grad(f(tok, E), E)[0]
    got = torch.autograd.grad(torch.compile(f, fullgraph=True, backend="aot_eager")(tok, E), E)[0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,N,V,D", [(torch.bfloat16, 3000, 40000, 2560), (torch.float32, 1, 9001, 4104), (torch.float16, 16384, 2000003, 40),
                                         (torch.float64, 700, 100000, 250)])
def test_gradient_of_a_large_table(dtype, N, V, D):
    """Every row that no token names is zero, in a buffer that held something else, and the others are the
    sums.  Tokens crowd at both ends and in runs, among them the padding row."""
    gen = torch.Generator().manual_seed(V)
    tok = torch.randint(0, V, (N,), generator=gen)
    tok[::3] = torch.randint(0, min(V, 40), (len(tok[::3]),), generator=gen)
    tok[1::5] = V - 1 - torch.randint(0, min(V, 40), (len(tok[1::5]),), generator=gen)
    tok[::7] = 5
    tok = tok.cuda()
    E = torch.zeros(V, D, dtype=dtype, device="cuda", requires_grad=True)
    g = torch.randn(N, D, device="cuda").to(dtype)
    for pad in (None, 5):
        junk = torch.full((V, D), 7.0, dtype=dtype, device="cuda")
        del junk  # the gradient's memory, from the same cache
        dE, = torch.autograd.grad(swvr.embedding_lookup(tok, E, scale=0.5, padding_idx=pad), E, g)
        named = torch.zeros(V, dtype=torch.bool, device="cuda")
        named[tok] = True
        if pad is not None:
            named[pad] = False
        assert not bool(dE[~named].any())
        rows, where = torch.unique(tok, return_inverse=True)
        want = torch.zeros(len(rows), D, dtype=torch.float64, device="cuda").index_add_(0, where, 0.5 * g.double())
        most = torch.zeros_like(want).index_add_(0, where, 0.5 * g.double().abs())
        keep = named[rows]
        count = torch.bincount(where, minlength=len(rows))[:, None].double()
        acc = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
        # the sum of count terms in fp32 / fp64, the product with scale exact, rounded once
        bound = count * acc * most + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).tiny
        assert bool(((dE[rows].double() - want).abs() <= bound)[keep].all())
