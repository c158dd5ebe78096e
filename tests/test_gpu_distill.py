"""GPU tests of the distillation loss and its gradients against the formula in 64 bits.

Tolerances, element by element.  c is the relative error of a sum of products in the compute path
against the sum of their absolute values: 2^-20 for fp32 accumulation (tensor cores; three-term
split TF32 products), 2^-46 for fp64.  So a score is off by at most e = c (|s| |h| |W|^T + |b|) / T + c |z|, the logsumexp
by the p-weighted mean of e, a probability by twice the two, relatively, and the loss by T^2 sum q times them.  The
score gradient adds its rounding to 16 bits (half a step, r) where the products take 16-bit operands; the
products with W and h carry its error through their absolute values, add c, and round once more.  fp16
score gradients are scaled so that the largest lies within 2^12 .. 2^14, so the half step of its smallest numbers, 2^-25, is
2^-37 of the largest at most."""
import math

import pytest
import torch

import swvr_b200 as swvr
from swvr_b200 import _native as nat

pytestmark = pytest.mark.gpu
f64 = torch.float64


def make(N, K, V, Kt, dtype, bias=True, seed=0, spread=3.0, tdt=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=f64)  # noqa: E731
    put = lambda x: x.to(dtype).cuda().requires_grad_(True)  # noqa: E731
    h, W = put(r(N, K)), put(r(V, K) * spread / K ** 0.5)
    b = put(0.5 * r(V)) if bias else None
    ids = torch.stack([torch.randperm(V, generator=gen)[:Kt] for _ in range(N)]).reshape(N, min(Kt, V)).cuda()
    t = (3 * r(N, ids.shape[1])).to(tdt).cuda()
    return h, W, b, ids, t


class Exact:
    """The definition in 64 bits, with the bounds of the module's docstring."""

    def __init__(self, h, W, b, ids, t, T=1.0, s=1.0, t_lse=None, weight=None, reduction="mean", up=None, cdt=None):
        cdt = cdt or h.dtype
        self.r = torch.finfo(cdt).eps / 2 if cdt in (torch.bfloat16, torch.float16) else 0.0
        self.c = c = 2.0 ** -46 if cdt == f64 else 2.0 ** -20
        self.fp16 = cdt == torch.float16
        d = lambda x: x.detach().to(cdt).double() if x is not None else None  # noqa: E731
        h, W = d(h), d(W)
        b = torch.zeros(W.shape[0], dtype=f64, device=W.device) if b is None else b.detach().double()
        N, V = h.shape[0], W.shape[0]
        z = (s * (h @ W.T) + b) / T
        e = c * (abs(s) * (h.abs() @ W.abs().T) + b.abs()) / T
        e = torch.where(z.isfinite(), e + c * z.abs(), torch.zeros_like(e))
        lse = torch.logsumexp(z, 1)
        p = (z - lse[:, None]).exp()
        el = (p * e).sum(1) + c * (1 + lse.abs())
        live = (ids >= 0) & (t.double() != -math.inf)
        tt = torch.where(live, t.double() / T, torch.full_like(t, -math.inf, dtype=f64))
        L = torch.logsumexp(tt, 1, keepdim=True) if t_lse is None else t_lse.double()[:, None]
        logq = torch.where(live, tt - L, torch.full_like(tt, -math.inf))
        q = logq.exp()
        at = ids.clamp(min=0)
        term = torch.where(q > 0, q * (logq - z.gather(1, at) + lse[:, None]), torch.zeros_like(q))
        self.each = T * T * term.sum(1)
        lq_err = torch.where(q > 0, c * (1 + logq.abs() + tt.abs()), torch.zeros_like(q))  # an entry left out has none
        ee = torch.where(q > 0, q * (lq_err + e.gather(1, at) + el[:, None]
                                     + lq_err * (logq - z.gather(1, at) + lse[:, None]).abs()), torch.zeros_like(q))
        self.each_err = T * T * ee.sum(1)
        w = torch.ones(N, dtype=f64, device=z.device) if weight is None else weight.detach().double()
        we = torch.where(w == 0, torch.zeros_like(w), w * self.each)
        we_err = torch.where(w == 0, torch.zeros_like(w), w.abs() * self.each_err)
        den = w.sum() if reduction == "mean" else torch.ones((), dtype=f64, device=z.device)
        if reduction == "none":
            self.loss, self.loss_err = we, we_err + c * we.abs()
        else:
            self.loss, self.loss_err = we.sum() / den, we_err.sum() / den.abs() + c * we.abs().sum() / den.abs()
        up = torch.ones_like(self.loss) if up is None else up.double()
        g = up * w / den * T * torch.ones(N, dtype=f64, device=z.device)
        qsum = q.sum(1)
        g = torch.where((w == 0) | (qsum == 0), torch.zeros_like(g), g)
        teach = torch.zeros_like(p).scatter_add_(1, at, q)
        dS = g[:, None] * (p * qsum[:, None] - teach)
        dS = torch.where(g[:, None] == 0, torch.zeros_like(dS), dS)
        dS_err = g.abs()[:, None] * (p * qsum[:, None] * 2 * (e + el[:, None] + 4 * c) + 4 * c * teach * (1 + lq_err.amax(1, keepdim=True) / c))
        dS_err = torch.where(g[:, None] == 0, torch.zeros_like(dS), dS_err)
        self.db, self.db_err = dS.sum(0), dS_err.sum(0) + c * dS.abs().sum(0)
        dS, dS_err = s * dS, abs(s) * dS_err
        dS_err = dS_err + self.r * (dS.abs() + dS_err)
        if self.fp16:
            dS_err = dS_err + 2.0 ** -37 * abs(s) * (g.abs() * qsum.clamp(min=1)).max()
        self.dh, self.dh_err = dS @ W, dS_err @ W.abs() + c * (dS.abs() @ W.abs())
        self.dW, self.dW_err = dS.T @ h, dS_err.T @ h.abs() + c * (dS.abs().T @ h.abs())
        if reduction == "mean":
            self.dw = up * (self.each - self.loss) / den
            self.dw_err = up.abs() * (self.each_err + self.loss_err + 4 * c * (self.each.abs() + self.loss.abs())) / den.abs()
        else:
            self.dw, self.dw_err = up * self.each, up.abs() * (self.each_err + 4 * c * self.each.abs())


def close(got, want, err, name):
    r = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * r
    lim = err * (1 + r) + r * want.abs() + tiny
    bad = ~((got.double() - want).abs() <= lim)
    worst = ((got.double() - want).abs() / lim).max().item() if got.numel() else 0.0
    assert not bool(bad.any()), (name, int(bad.sum()), worst)


def run(h, W, b, ids, t, T=1.0, s=1.0, t_lse=None, weight=None, reduction="mean", up=None, chunk=None, want_w=False):
    loss = swvr.softmax_distill(h, W, ids, t, b, temperature=T, logit_scale=s, teacher_lse=t_lse, weight=weight,
                                reduction=reduction, chunk_size=chunk)
    leaves = [x for x in (h, W, b, weight if want_w else None) if x is not None]
    got = iter(torch.autograd.grad(loss, leaves, None if up is None else up.to(loss.dtype)))
    return loss.detach(), [next(got) if x is not None else None for x in (h, W, b, weight if want_w else None)]


def check(h, W, b, ids, t, **kw):
    chunk, want_w = kw.pop("chunk", None), kw.pop("want_w", False)
    loss, (dh, dW, db, dw) = run(h, W, b, ids, t, chunk=chunk, want_w=want_w, **kw)
    x = Exact(h, W, b, ids, t, **kw)
    assert loss.dtype == (f64 if h.dtype == f64 else torch.float32)
    close(loss, x.loss, x.loss_err, "loss")
    for name, got, leaf in (("dh", dh, h), ("dW", dW, W), ("db", db, b)):
        if got is not None:
            assert got.dtype == leaf.dtype and got.shape == leaf.shape
            close(got, getattr(x, name), getattr(x, name + "_err"), name)
    if want_w:
        close(dw, x.dw, x.dw_err, "dw")
    return loss, dh, dW, db


DTYPES = [torch.float32, torch.float64, torch.bfloat16, torch.float16]
SIZES = [(1, 8, 1, 1), (3, 16, 41, 5), (5, 12, 300, 4), (256, 64, 1000, 8), (130, 72, 513, 128), (300, 256, 3001, 33)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,K,V,Kt", SIZES)
@pytest.mark.parametrize("T,bias", [(1.0, False), (2.5, True)])
def test_loss_and_gradients(dtype, N, K, V, Kt, T, bias):
    h, W, b, ids, t = make(N, K, V, Kt, dtype, bias, tdt=torch.bfloat16 if dtype == torch.bfloat16 else torch.float32)
    check(h, W, b, ids, t, T=T, s=0.75 if bias else 1.0, chunk=256 if V > 1000 else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions_weights_and_upstream(dtype, reduction):
    h, W, b, ids, t = make(70, 64, 700, 9, dtype)
    gen = torch.Generator().manual_seed(1)
    w = torch.rand(70, generator=gen).cuda()
    w[::7] = 0
    w.requires_grad_(True)
    up = torch.randn(70 if reduction == "none" else (), generator=gen).cuda()
    check(h, W, b, ids.int(), t, weight=w, reduction=reduction, up=up, want_w=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_teacher_lse_leaves_mass_out(dtype):
    h, W, b, ids, t = make(40, 64, 500, 6, dtype)
    L = torch.logsumexp(t.double() / 1.5, 1).float() + torch.rand(40).cuda()
    check(h, W, b, ids, t, T=1.5, t_lse=L)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
def test_repeated_padded_and_masked_entries(dtype):
    """The same id up to Kt times, negative ids, logits of -inf and of the type's lowest value, rows with
    one entry left and with none."""
    h, W, b, ids, t = make(37, 64, 600, 12, dtype)
    ids[0] = 5
    ids[1, ::2] = 599
    ids[2, 3:] = -1
    ids[3] = -100
    t[4, 1:] = -math.inf
    t[5] = -math.inf
    ids[6, 4], t[6, 4] = 2 ** 40, -math.inf  # left out: nothing to look up
    t[7, :6] = torch.finfo(t.dtype).min
    loss, dh, *_ = check(h, W, b, ids.where(ids < 600, torch.full_like(ids, -1)), t)
    loss2, (dh2, *_) = run(h, W, b, ids, t)
    assert torch.equal(loss, loss2) and torch.equal(dh, dh2)
    assert bool((dh[3] == 0).all()) and bool((dh[5] == 0).all())
    each = swvr.softmax_distill(h, W, ids, t, b, reduction="none")
    assert float(each[3]) == 0 and float(each[5]) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_teacher_entries_at_all(dtype):
    h, W, b, ids, t = make(9, 16, 50, 1, dtype)
    loss, (dh, dW, db, _) = run(h, W, b, ids[:, :0], t[:, :0])
    assert float(loss) == 0 and all(bool((g == 0).all()) for g in (dh, dW, db))


@pytest.mark.parametrize("dtype", [torch.float64, torch.bfloat16])
def test_masked_vocabulary_and_dropped_tokens(dtype):
    """Vocabulary rows masked by a bias of -inf, whole tiles of them; a token whose teacher sits on a
    masked row has an infinite loss, which a zero weight drops."""
    h, W, b, ids, t = make(50, 64, 1500, 4, dtype)
    with torch.no_grad():
        b[200:900] = -math.inf
    ids[ids % 1500 >= 200] = 7
    ids[11, 0] = 300
    w = torch.ones(50, device="cuda")
    w[11] = 0
    each = swvr.softmax_distill(h, W, ids, t, b, reduction="none")
    assert float(each[11]) == math.inf and int(each.isinf().sum()) == 1
    loss, dh, dW, db = check(h, W, b, ids, t, weight=w)
    assert bool((dh[11] == 0).all()) and bool((dW[200:900] == 0).all()) and bool((db[200:900] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ids_out_of_range_are_reported(dtype):
    h, W, b, ids, t = make(8, 16, 50, 4, dtype)
    ids[2, 1] = 50
    each = swvr.softmax_distill(h, W, ids, t, b, reduction="none")
    assert bool(each[2].isnan()) and int(each.isnan().sum()) == 1
    dh = torch.autograd.grad(each.sum(), h)[0]
    assert bool(dh[2].isnan().all()) and int(dh.isnan().any(1).sum()) == 1
    with pytest.raises(RuntimeError, match=r"outside \[0, V\)"):
        nat.check_device_error()
    nat.check_device_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_student_that_has_learnt_the_teacher(dtype):
    """The teacher lists the student's own top probabilities: p - q vanishes on its entries, where a 16-bit p
    minus q would keep the rounding of p.  The bounds of the gradients shrink with it."""
    h, W, b, ids, t = make(64, 64, 400, 8, dtype, spread=6.0)
    z = h.detach().double() @ W.detach().double().T + b.detach().double()
    top = z.topk(8, dim=1)
    loss, dh, dW, db = check(h, W, b, top.indices, top.values.float(), t_lse=torch.logsumexp(z, 1).float())
    full = check(h, W, b, ids, t)[1]
    assert float(dh.double().norm()) < 0.3 * float(full.double().norm())


def test_small_fp16_gradients_do_not_vanish():
    """An upstream gradient of 1e-7: the fp32 gradients of an fp16 autocast keep their relative accuracy."""
    h, W, b, ids, t = make(64, 64, 900, 8, torch.float32)
    up = torch.tensor(1e-7).cuda()
    with torch.autocast("cuda", dtype=torch.float16):
        loss, (dh, dW, db, _) = run(h, W, b, ids, t, up=up)
    x = Exact(h, W, b, ids, t, up=up, cdt=torch.float16)
    for got, want, err in ((dh, x.dh, x.dh_err), (dW, x.dW, x.dW_err), (db, x.db, x.db_err)):
        assert got.dtype == torch.float32
        close(got, want, err, "autocast")
        assert float((got.double() - want).norm()) < 2e-3 * float(want.norm())


def test_autocast_over_fp32_parameters():
    h, W, b, ids, t = make(100, 100, 1111, 16, torch.float32)  # K = 100: rows padded to the kernels' alignment
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, (dh, dW, db, _) = run(h, W, b, ids, t)
    x = Exact(h, W, b, ids, t, cdt=torch.bfloat16)
    close(loss, x.loss, x.loss_err, "loss")
    for name, got in (("dh", dh), ("dW", dW), ("db", db)):
        close(got, getattr(x, name), getattr(x, name + "_err"), name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_leading_shape_strides_and_broadcast_rows(dtype):
    gen = torch.Generator().manual_seed(2)
    big = torch.randn(70, 80, generator=gen).to(dtype).cuda()
    W = big[:, 8:72].detach().requires_grad_(True)
    h = torch.randn(2, 9, 64, generator=gen).to(dtype).cuda().transpose(0, 1).detach().requires_grad_(True)
    ids = torch.randint(0, 70, (9, 2, 6), generator=gen).cuda()[..., ::2]
    t = torch.randn(3, 9, 2, generator=gen).cuda().permute(1, 2, 0)
    each = swvr.softmax_distill(h, W, ids, t, reduction="none")
    assert each.shape == (9, 2)
    x = Exact(h.reshape(18, 64), W, None, ids.reshape(18, 3), t.reshape(18, 3), reduction="none")
    close(each.reshape(18), x.loss, x.loss_err, "each")
    dh, dW = torch.autograd.grad(each.sum(), (h, W))  # the upstream gradient is expanded from one number
    close(dh.reshape(18, 64), x.dh, x.dh_err, "dh")
    close(dW, x.dW, x.dW_err, "dW")
    one = torch.randn(64, generator=gen).to(dtype).cuda().requires_grad_(True)
    rows = one.expand(18, 64)
    d = torch.autograd.grad(swvr.softmax_distill(rows, W, ids.reshape(18, 3), t.reshape(18, 3), reduction="sum"), one)[0]
    y = Exact(rows, W, None, ids.reshape(18, 3), t.reshape(18, 3), reduction="sum")
    r = torch.finfo(dtype).eps / 2
    lim = (y.dh_err + r * y.dh.abs()).sum(0) + 18 * r * y.dh.abs().sum(0)  # torch adds the rows in the parameter's type
    assert bool(((d.double() - y.dh.sum(0)).abs() <= lim).all())


@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_gradients_by_differences(reduction):
    h, W, b, ids, t = make(4, 6, 9, 3, f64)
    ids[1, 1] = ids[1, 0]
    w = torch.tensor([1.0, 0.5, 0.0, 2.0], dtype=f64, device="cuda", requires_grad=True)
    f = lambda h, W, b, w: swvr.softmax_distill(h, W, ids, t, b, temperature=1.7, weight=w, reduction=reduction,  # noqa: E731
                                                logit_scale=0.8)
    grads = torch.autograd.grad(f(h, W, b, w), (h, W, b, w))
    step = 1e-5
    for k, (x, g) in enumerate(zip((h, W, b, w), grads)):
        for i in range(x.numel()):
            if k == 3 and i == 2:
                continue  # at weight zero the token is dropped
            e = torch.zeros_like(x).reshape(-1)
            e[i] = step
            args = [h.detach(), W.detach(), b.detach(), w.detach()]
            hi, lo = list(args), list(args)
            hi[k], lo[k] = args[k] + e.view_as(x), args[k] - e.view_as(x)
            num = float(f(*hi) - f(*lo)) / (2 * step)
            # central difference: f''' step^2 / 6 and rounding 2^-52 |f| / step
            assert abs(num - float(g.reshape(-1)[i])) < 2e-8, (k, i)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_chunks_do_not_change_the_loss(dtype):
    h, W, b, ids, t = make(300, 64, 5000, 16, dtype)
    runs = [check(h, W, b, ids, t, chunk=c) for c in (100, 1024, 8192)]
    if dtype == torch.bfloat16:  # the forward has no chunks, dW one GEMM per row whatever its chunk
        assert all(torch.equal(r[0], runs[0][0]) and torch.equal(r[2], runs[0][2]) for r in runs)


def test_same_bits_on_every_run():
    h, W, b, ids, t = make(700, 128, 9000, 32, torch.bfloat16)
    ids[:, 0] = 17  # one row of the bias gradient takes an entry from every token
    runs = [run(h, W, b, ids, t) for _ in range(4)]
    for loss, grads in runs[1:]:
        assert torch.equal(loss, runs[0][0])
        assert all(torch.equal(a, c) for a, c in zip(grads[:3], runs[0][1][:3]))


def test_frozen_inputs_and_empty_batch():
    h, W, b, ids, t = make(60, 64, 700, 5, torch.bfloat16)
    full = run(h, W, b, ids, t)[1]
    for live in range(3):
        args = [x.detach().requires_grad_(i == live) for i, x in enumerate((h, W, b))]
        loss = swvr.softmax_distill(args[0], args[1], ids, t, args[2])
        assert torch.equal(torch.autograd.grad(loss, args[live])[0], full[live])
    loss = swvr.softmax_distill(h[:0], W, ids[:0], t[:0], b, reduction="sum")
    dW, db = torch.autograd.grad(loss, (W, b))
    assert float(loss) == 0 and bool((dW == 0).all()) and bool((db == 0).all())
    assert swvr.softmax_distill(h[:0], W, ids[:0], t[:0], b, reduction="none").shape == (0,)


def test_scores_are_never_held():
    """Peak memory of a step: one chunk of 16-bit score gradients, the fp32 dh and the gradients; the
    [N, V] scores alone would be 3.2 GB."""
    N, K, V = 8192, 256, 100000
    h, W, b, ids, t = make(4, K, 64, 4, torch.bfloat16)
    h = torch.randn(N, K, device="cuda").bfloat16().requires_grad_(True)
    W = torch.randn(V, K, device="cuda").bfloat16().requires_grad_(True)
    ids, t = torch.randint(0, V, (N, 8), device="cuda"), torch.randn(N, 8, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    loss = swvr.softmax_distill(h, W, ids, t, chunk_size=4096)
    torch.autograd.grad(loss, (h, W))
    assert torch.cuda.max_memory_allocated() - base < 8192 * N * 2 + 3 * (N + V) * K * 4


def test_side_stream_and_captured_step():
    """Captured with .backward() while an eager graph of the same leaves lives, then replayed on new inputs."""
    h, W, b, ids, t = make(200, 64, 3000, 8, torch.bfloat16)
    leaves = (h, W, b)

    def step():
        loss = swvr.softmax_distill(h, W, ids, t, b, temperature=1.5)
        return loss, torch.autograd.grad(loss, leaves)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            alive = step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss_g, grads_g = step()
    for seed in (5, 6):
        with torch.no_grad():
            h.copy_(torch.randn(200, 64, generator=torch.Generator().manual_seed(seed)))
        t.copy_(torch.randn(200, 8, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [loss_g.clone()] + [g.clone() for g in grads_g]
        loss_e, grads_e = step()
        assert all(torch.equal(a, e) for a, e in zip(got, [loss_e, *grads_e]))
    x = Exact(h, W, b, ids, t, T=1.5)
    close(got[0], x.loss, x.loss_err, "loss")
    del graph, alive


def test_compiled_checkpointed_and_module():
    from torch.utils.checkpoint import checkpoint
    head = torch.nn.Linear(64, 500).cuda().bfloat16()
    m = swvr.SoftmaxDistill(head, temperature=2.0)
    h, _, _, ids, t = make(30, 64, 500, 6, torch.bfloat16)
    leaves = (h, head.weight, head.bias)
    want = torch.autograd.grad(m(h, ids, t), leaves)
    for f in (torch.compile(m, fullgraph=True, backend="aot_eager"), lambda *a: checkpoint(m, *a, use_reentrant=False)):
        got = torch.autograd.grad(f(h, ids, t), leaves)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_wide_teacher_rows():
    """1024 entries per token, and a vocabulary no wider than that."""
    h, W, b, ids, t = make(6, 32, 1024, 1024, torch.bfloat16)
    check(h, W, b, ids, t)
    check(h.detach().double().requires_grad_(True), W.detach().double().requires_grad_(True),
          b.detach().double().requires_grad_(True), ids, t)


def test_the_teacher_is_a_constant():
    h, W, b, ids, t = make(9, 16, 60, 4, torch.float32)
    t.requires_grad_(True)
    L = torch.logsumexp(t, 1)
    loss = swvr.softmax_distill(h.detach(), W.detach(), ids, t, teacher_lse=L)
    assert not loss.requires_grad
    loss = swvr.softmax_distill(h, W, ids, t, teacher_lse=L)
    assert torch.autograd.grad(loss, t, allow_unused=True)[0] is None
