"""GPU tests of sampling against its definition in 64 bits.

From given logits the token has to be the definition's: the kernel's weights are fixed point with 44 bits
below the largest, so a running sum of V of them is off by at most V 2^-45 of the largest weight, and a
token may differ only where u times the total lies that near a border of its interval (``near``).
From the head, scores carry the error of fp32 accumulation, e = 2^-20 (|s| |h| |W|^T + |b|), so weights
are off by e / T relatively: the token has to be one that some scores within e give."""
import math

import pytest
import torch

import swvr_b200 as swvr

pytestmark = pytest.mark.gpu
f64 = torch.float64


def col(v, N, off):
    return torch.full((N, 1), float(off if v is None else v), dtype=f64, device="cuda") if not isinstance(v, torch.Tensor) \
        else v.detach().to("cuda").double().reshape(N, 1)


def exact(x, u, T=1.0, k=None, p=None, m=None):
    """(token, kept mask, weights in index order) of 2-D x in 64 bits."""
    x = x.double()
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    N, V = x.shape
    T, k, p, m = col(T, N, 1), col(k, N, 0), col(p, N, 1), col(m, N, 0)
    u = u.double().reshape(N, 1)
    u = torch.where(u > 0, u, torch.zeros_like(u))
    greedy = ~(T > 0)
    top = x.max(1, keepdim=True).values
    z = torch.where(x == top, torch.zeros_like(x), (x - top) / torch.where(greedy, torch.ones_like(T), T))
    zs, order = z.sort(dim=1, descending=True, stable=True)
    w = zs.exp()
    keep = (w > 0) & ((torch.arange(V, device=x.device) < k) | (k <= 0))
    kept = w * keep
    ahead = kept.cumsum(1) - kept
    keep &= ~(p < 1) | (ahead < (p.clamp(min=0) * kept.sum(1, keepdim=True)).clamp(min=1e-300)) | (ahead == 0)
    keep &= ~(m > 0) | (zs >= m.clamp(max=1).log())
    index = torch.arange(V, device=x.device)
    kept_mask = torch.zeros_like(keep).scatter_(1, order, keep)
    w = z.exp() * kept_mask
    cdf = w.cumsum(1)
    goal = u * cdf[:, -1:]
    past = (cdf > goal) & (w > 0)
    last = torch.where(w > 0, index, -1).max(1).values
    token = torch.where(past, index, V).min(1).values
    token = torch.where(token == V, last, token)
    first = torch.where(x == top, index, V).min(1).values
    token = torch.where(greedy[:, 0], first, token)
    token = torch.where(torch.isneginf(top[:, 0]), torch.full_like(token, -1), token)
    return token, kept_mask, w


def near(got, want, w, u, V):
    """Rows where got differs: u times the total has to lie within V 2^-44 of got's interval."""
    for r in (got != want).nonzero().flatten().tolist():
        cdf = w[r].cumsum(0)
        g = int(got[r])
        goal, tol = float(u[r].double().clamp(0, 1) * cdf[-1]), V * 2.0 ** -44
        if g < 0 or float(w[r, g]) == 0 or not float(cdf[g] - w[r, g]) - tol <= goal <= float(cdf[g]) + tol:
            return False
    return True


def logits(N, V, dtype=torch.float32, scale=4.0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(N, V, generator=gen, device="cuda")).to(dtype)


def uniform(N, seed=1):
    return torch.rand(N, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def check(x, u, **kw):
    got = swvr.sample_logits(x, u, temperature=kw.get("T", 1.0), top_k=kw.get("k"), top_p=kw.get("p"), min_p=kw.get("m"))
    want, kept, w = exact(x, u, **kw)
    assert got.dtype == torch.int64 and got.shape == u.shape
    assert near(got, want, w, u, x.shape[1]), (got[got != want][:5], want[got != want][:5], kw)
    return got


SETTINGS = [dict(), dict(T=0.0), dict(T=0.6), dict(k=1), dict(k=50), dict(p=0.9), dict(m=0.05), dict(T=1.7, k=40, p=0.8, m=0.02),
            dict(T=0.8, k=2000, p=0.99), dict(p=0.999, m=1e-5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V", [(1, 1), (3, 2), (5, 33), (64, 1000), (150, 10007)])
@pytest.mark.parametrize("kw", SETTINGS)
def test_tokens(dtype, N, V, kw):
    check(logits(N, V, dtype), uniform(N), **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(1, 152064), (3, 50001), (20, 128256), (80, 70001), (2, 400003)])
@pytest.mark.parametrize("kw", SETTINGS[2:])
def test_long_rows(dtype, N, V, kw):
    """Rows over one CTA's shared memory: two to eight CTAs, and past eight."""
    check(logits(N, V, dtype, scale=5.0), uniform(N), **kw)


@pytest.mark.parametrize("V", [7, 1500, 5000, 60000])
@pytest.mark.parametrize("kw", [dict(), dict(k=3), dict(k=1400), dict(p=0.3), dict(p=0.97, k=1201), dict(m=1.0), dict(T=0.0),
                                dict(p=1e-9)])
def test_equal_scores(V, kw):
    """All scores equal, or a few values many times each: cuts inside runs of equal scores, runs longer than
    the list that is ranked at once."""
    u = uniform(6)
    same = torch.full((6, V), 2.5, device="cuda")
    check(same, u, **kw)
    steps = torch.randint(0, 3, (6, V), generator=torch.Generator().manual_seed(V)).float().cuda()
    check(steps, u, **kw)
    two = same.clone()
    two[:, V // 2] = 2.5000002
    check(two, u, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(k=2), dict(p=0.6), dict(m=0.3), dict(T=0.0), dict(T=1e-30), dict(T=1e6, k=5)])
def test_masked_and_non_finite_scores(kw):
    x = logits(12, 300)
    x[0] = -math.inf
    x[1, 1:] = -math.inf
    x[2, ::2] = -math.inf
    x[3, :] = math.nan
    x[4, 5:] = math.nan
    x[5] = torch.finfo(torch.float32).min
    x[6, 7] = math.inf
    x[7, 9:12] = math.inf
    x[8] = torch.finfo(torch.float32).min
    x[8, 20] = 0
    x[9] = 0.0
    x[9, ::2] = -0.0
    x[10] = torch.finfo(torch.float32).max
    x[11] = torch.finfo(torch.float32).tiny
    u = uniform(12)
    got = check(x, u, **kw)
    assert int(got[0]) == int(got[3]) == -1 and int(got[1]) == 0 and int(got[6]) == 7
    for dt in (torch.bfloat16, torch.float16):
        check(x.to(dt), u, **kw)


def test_uniform_numbers_at_and_past_the_ends():
    x = logits(7, 500)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -3.0, math.nan, 0.5], device="cuda")
    for kw in (dict(), dict(k=10), dict(p=0.5)):
        got = swvr.sample_logits(x, u, top_k=kw.get("k"), top_p=kw.get("p"))
        inside = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 1.0, 0.0, 0.0, 0.5], device="cuda")
        want, kept, w = exact(x, inside, **kw)
        assert near(got, want, w, inside, 500)
        assert bool(kept.gather(1, got[:, None]).all())


def test_settings_of_each_row():
    N, V = 40, 3000
    x, u = logits(N, V), uniform(N)
    gen = torch.Generator(device="cuda").manual_seed(4)
    T = 2 * torch.rand(N, generator=gen, device="cuda")
    k = torch.randint(1, 100, (N,), generator=gen, device="cuda")
    p, m = torch.rand(N, generator=gen, device="cuda"), 0.1 * torch.rand(N, generator=gen, device="cuda")
    T[:3] = torch.tensor([0.0, -1.0, math.nan])
    k[3:6] = torch.tensor([0, -1, 10 ** 12])
    p[6:10] = torch.tensor([1.0, 2.0, 0.0, -1.0])
    m[10:13] = torch.tensor([0.0, -1.0, 5.0])
    want, kept, w = exact(x, u, T, k, p, m)
    got = swvr.sample_logits(x, u, temperature=T, top_k=k, top_p=p, min_p=m)
    assert near(got, want, w, u, V)
    p[13:15], m[15] = math.nan, math.nan  # off
    off_p, off_m = torch.where(p.isnan(), 1.0, p), torch.where(m.isnan(), 0.0, m)
    want, kept, w = exact(x, u, T, k, off_p, off_m)
    got = swvr.sample_logits(x, u, temperature=T.double(), top_k=k.clamp(max=2 ** 31 - 1).int(), top_p=p, min_p=m.double())
    assert near(got, want, w, u, V)
    got = swvr.sample_logits(x, u, temperature=T.bfloat16(), top_p=0.9)
    want, kept, w = exact(x, u, T.bfloat16(), None, 0.9)
    assert near(got, want, w, u, V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_and_strides(dtype):
    big = logits(24, 1200, dtype)
    u = uniform(24)
    for x in (big[:, 5:900], big[:, ::2], big.t().contiguous().t()[:, :700], big[::2], big[:1].expand(24, 1200)):
        check(x, u[: x.shape[0]], k=30)
        check(x, u.double()[: x.shape[0]], p=0.9)
    x3, u3 = big.view(4, 6, 1200), u.view(6, 4).t()
    got = swvr.sample_logits(x3, u3, top_k=9)
    assert got.shape == (4, 6)
    assert torch.equal(got.reshape(-1), swvr.sample_logits(big, u3.reshape(-1), top_k=9))
    one = swvr.sample_logits(big[0], u[0])
    assert one.shape == () and int(one) == int(swvr.sample_logits(big[:1], u[:1])[0])
    assert swvr.sample_logits(big[:0], u[:0]).shape == (0,)
    assert swvr.sample_logits(big[:, :0], u).tolist() == [-1] * 24


@pytest.mark.parametrize("N,V", [(5, 100), (3, 60000)])
def test_logprobs(N, V):
    """Of the whole row at its temperature, rounded to fp32 once: half a step, and V 2^-44 of the sum."""
    x, u = logits(N, V), uniform(N)
    for T in (0.0, 0.7, 1.3):
        tok, lp = swvr.sample_logits(x, u, temperature=T, top_k=20, top_p=0.9, return_logprobs=True)
        assert torch.equal(tok, swvr.sample_logits(x, u, temperature=T, top_k=20, top_p=0.9))
        want = torch.log_softmax(x.double() / (T or 1.0), 1).gather(1, tok[:, None])[:, 0]
        assert lp.dtype == torch.float32
        assert bool(((lp.double() - want).abs() <= 2.0 ** -24 * want.abs() + V * 2.0 ** -43).all())
    dead = torch.full((1, V), -math.inf, device="cuda")
    assert float(swvr.sample_logits(dead, u[:1], return_logprobs=True)[1]) == -math.inf


def head(N, K, V, dtype, bias=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return (r(N, K).to(dtype).cuda(), (5 * K ** -0.5 * r(V, K)).to(dtype).cuda(),
            (0.5 * r(V)).to(dtype).cuda() if bias else None)


def check_head(got, h, W, b, u, s=1.0, T=1.0, k=None, p=None, m=None):
    """Some scores within e of the exact ones give the token: it may be kept when every threshold is loosened by what e
    moves, and u times the total lies within what e moves of its interval."""
    h, W = h.double(), W.double()
    x = s * (h @ W.T) + (0 if b is None else b.double())
    e = 2.0 ** -20 * (abs(s) * (h.abs() @ W.abs().T) + (0 if b is None else b.double().abs())).max()
    N, V = x.shape
    if T == 0:
        assert bool((x.gather(1, got[:, None])[:, 0] >= x.max(1).values - 2 * e).all())
        return
    f = float(torch.exp(4 * e / T))  # how far a ratio of two weights may be off
    _, kept, w = exact(x, u, T, k, p, m)
    low = torch.where(kept, x, math.inf).min(1, keepdim=True).values
    z = ((x - x.max(1, keepdim=True).values) / T).exp()
    # the cut may fall up to 2 e lower or higher: tokens there may or may not count
    sure, maybe = z * (x >= low + 2 * e), z * (x >= low - 2 * e)
    total_lo, total_hi = sure.sum(1), maybe.sum(1)
    if p is not None:  # a moved running sum shifts the nucleus by a token on either side
        slack = z.gather(1, torch.where(kept, x, math.inf).argmin(1, keepdim=True))[:, 0] * 2
        total_lo, total_hi = total_lo - slack, total_hi + slack
    else:
        slack = torch.zeros_like(total_lo)
    g = got[:, None]
    assert bool((x.gather(1, g) >= low - 2 * e).all()) or p is not None
    before = (sure.cumsum(1) - sure).gather(1, g)[:, 0] - slack
    after = maybe.cumsum(1).gather(1, g)[:, 0] + slack
    ud = u.double()
    assert bool((before <= (ud * f + 1e-12) * total_hi).all()), "the interval begins past u"
    assert bool((after * f >= (ud - 1e-12) * total_lo).all()), "the interval ends before u"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,V", [(1, 8, 1), (1, 64, 1000), (3, 100, 10007), (32, 256, 3001), (33, 64, 513), (65, 72, 2000),
                                   (130, 128, 5000), (300, 64, 700)])
@pytest.mark.parametrize("kw", [dict(k=40), dict(T=0.0), dict(T=0.7, k=50, p=0.9), dict(m=0.05)])
def test_head(dtype, N, K, V, kw):
    h, W, b = head(N, K, V, dtype, bias=N % 2 == 1)
    u = uniform(N)
    got = swvr.softmax_sample(h, W, u, b, temperature=kw.get("T", 1.0), top_k=kw.get("k"), top_p=kw.get("p"), min_p=kw.get("m"),
                              logit_scale=0.9)
    assert got.shape == (N,) and got.dtype == torch.int64 and bool(((got >= 0) & (got < V)).all())
    check_head(got, h, W, b, u, s=0.9, **kw)


def test_head_in_row_chunks():
    """500 rows of 152064 fp32 scores are 304 MB: two chunks.  Same tokens as one row at a time."""
    h, W, b = head(500, 16, 152064, torch.bfloat16)
    u = uniform(500)
    got = swvr.softmax_sample(h, W, u, b, top_k=20)
    check_head(got[430:], h[430:], W, b, u[430:], k=20)
    for i in (0, 440, 441, 499):
        assert int(swvr.softmax_sample(h[i], W, u[i], b, top_k=20)) == int(got[i])


def test_head_under_autocast_strides_and_leading_shape():
    h, W, b = head(12, 64, 900, torch.float32)
    u = uniform(12)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = swvr.softmax_sample(h.view(3, 4, 64), W.requires_grad_(True), u.view(3, 4), b, top_k=5, temperature=0.5)
    assert got.shape == (3, 4) and not got.requires_grad
    check_head(got.view(12), h.bfloat16(), W.detach().bfloat16(), b, u, T=0.5, k=5)
    wide = torch.randn(900, 80, device="cuda").bfloat16()
    one = torch.randn(64, device="cuda").bfloat16()
    got = swvr.softmax_sample(one.expand(12, 64), wide[:, 8:72], u, top_k=7)
    check_head(got, one.expand(12, 64), wide[:, 8:72], None, u, k=7)


def test_head_with_a_masked_vocabulary():
    h, W, b = head(9, 64, 2000, torch.bfloat16)
    b[:1500] = -math.inf
    got = swvr.softmax_sample(h, W, uniform(9), b, top_k=50)
    assert bool((got >= 1500).all())
    b[:] = -math.inf
    assert swvr.softmax_sample(h, W, uniform(9), b).tolist() == [-1] * 9


def test_offsets_past_32_bits():
    N, V = 15000, 152064  # 2.3e9 scores
    x = torch.zeros(N, V, dtype=torch.bfloat16, device="cuda")
    x[:, 77] = 1
    x[N - 1, V - 1] = 40
    got = swvr.sample_logits(x, torch.full((N,), 0.5, device="cuda"), top_k=1)
    assert int(got[N - 1]) == V - 1 and bool((got[:-1] == 77).all())


def test_side_stream_and_captured_call():
    x, (h, W, b) = logits(30, 5000), head(30, 64, 5000, torch.bfloat16)
    u, k = uniform(30), torch.full((30,), 25, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, c = swvr.sample_logits(x, u, top_k=k, top_p=0.9), swvr.softmax_sample(h, W, u, b, top_k=k)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a_g, c_g = swvr.sample_logits(x, u, top_k=k, top_p=0.9), swvr.softmax_sample(h, W, u, b, top_k=k)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, a_g) and torch.equal(c, c_g)
    u.copy_(uniform(30, seed=9))
    x.copy_(logits(30, 5000, seed=8))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a_g, swvr.sample_logits(x, u, top_k=k, top_p=0.9))
    assert torch.equal(c_g, swvr.softmax_sample(h, W, u, b, top_k=k))
    del graph


def test_compiled_whole():
    x, (h, W, b) = logits(8, 700), head(8, 64, 700, torch.bfloat16)
    u = uniform(8)

    def f(x, h, W, b, u):
        return swvr.sample_logits(x, u, top_k=9), swvr.softmax_sample(h, W, u, b, top_p=0.9)

    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x, h, W, b, u)
    assert all(torch.equal(a, c) for a, c in zip(got, f(x, h, W, b, u)))


@pytest.mark.parametrize("kw", [dict(), dict(k=30, p=0.9), dict(p=0.9999, T=1.3), dict(m=0.01)])
def test_very_long_rows(kw):
    """Past 2^20 scores: fixed-point weights of fewer bits, no fp32 sums."""
    check(logits(2, 1200007, scale=3.0), uniform(2), **kw)


def test_head_without_a_vocabulary():
    h, W, b = head(3, 64, 5, torch.bfloat16)
    assert swvr.softmax_sample(h, W[:0], uniform(3)).tolist() == [-1, -1, -1]
    assert swvr.softmax_sample(h[:0], W, uniform(0)).shape == (0,)


def test_scores_that_need_no_gradient_take_none():
    x = logits(4, 100).requires_grad_(True)
    tok, lp = swvr.sample_logits(x, uniform(4), return_logprobs=True)
    assert not tok.requires_grad and not lp.requires_grad
    h, W, b = head(4, 64, 100, torch.bfloat16)
    assert not swvr.softmax_sample(h.requires_grad_(True), W.requires_grad_(True), uniform(4), b).requires_grad


def test_rows_of_the_lowest_value_beside_minus_infinity():
    """A mask of the type's lowest value is a score like any other; one of -inf is not."""
    for dt in (torch.float32, torch.bfloat16):
        x = torch.full((6, 400), torch.finfo(dt).min, dtype=dt, device="cuda")
        x[:, ::2] = -math.inf
        for kw in (dict(), dict(T=1e30), dict(k=9), dict(p=0.5), dict(m=0.9)):
            got = check(x, uniform(6), **kw)
            assert bool((got % 2 == 1).all())


def test_a_row_gives_the_same_token_in_any_batch():
    """Many rows, which have few CTAs each, against the same rows in small batches: u on borders of the running weight
    (where fp32 sums leave the token open), temperatures at both ends, rows with nothing to choose from."""
    N, V = 310, 9001
    x = logits(N, V, torch.bfloat16)
    T = torch.where(torch.arange(N, device="cuda") % 7 < 5, 0.9, 1.0)
    T[::41], T[1::41], T[2::41] = 0.0, 1e-30, 1e30
    x[3::41] = -math.inf
    x[4::41, 100] = math.inf
    w = exact(x, uniform(N), T=T)[2].cumsum(1)
    u = uniform(N).double()
    u[::2] = (w.gather(1, torch.randint(0, V, (N, 1), generator=torch.Generator().manual_seed(3)).cuda())[:, 0] / w[:, -1])[::2]
    u = u.nan_to_num().clamp(0, 1 - 2.0 ** -53)
    call = lambda i, j: swvr.sample_logits(x[i:j], u[i:j], temperature=T[i:j], return_logprobs=True)  # noqa: E731
    got, lp = call(0, N)
    assert near(got, *exact(x, u, T=T)[::2], u, V)
    for i in range(0, N, 31):
        tok, part = call(i, i + 31)
        assert torch.equal(tok, got[i:i + 31]) and torch.equal(part, lp[i:i + 31])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again, lp2 = call(0, N)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, got) and torch.equal(lp2, lp)
    del graph


def test_fp32_sums_far_from_zero():
    """Scores whose integer part in octaves is large, or that rise along the row by more than fp32's range of weights."""
    V = 6000
    u = uniform(20)
    for shift in (0.0, 3e4, -3e4, 3e5, -3e5):
        x = (logits(20, V) + shift)
        for kw in (dict(), dict(p=0.9), dict(T=0.25)):
            check(x, u, **kw)
    ramp = torch.linspace(-4000, 4000, V, device="cuda").expand(20, V) + logits(20, V)
    for kw in (dict(), dict(p=0.9), dict(T=300.0), dict(T=300.0, p=0.9)):
        check(ramp, u, **kw)
        check(ramp.flip(1), u, **kw)
