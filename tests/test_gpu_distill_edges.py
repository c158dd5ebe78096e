"""GPU tests of the distillation loss where a teacher's logits reach the ends of their type, and of its repeatability."""
import math

import pytest
import torch

import swvr_b200 as swvr
from test_gpu_distill import Exact, check, close, make, run

pytestmark = pytest.mark.gpu


def check_shifted(h, W, b, ids, t, T):
    """Against the definition of the logits less each row's largest, the same teacher: its bounds then go by differences."""
    top = t.double().amax(1, keepdim=True)
    x = Exact(h, W, b, ids, torch.where(top.isneginf(), top, t.double() - top), T=T)
    loss, grads = run(h, W, b, ids, t, T=T)
    close(loss, x.loss, x.loss_err, "loss")
    for name, got in zip(("dh", "dW", "db"), grads):
        close(got, getattr(x, name), getattr(x, name + "_err"), name)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tdt", [torch.float64, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [0.25, 1.0, 3.0])
def test_rows_of_the_lowest_and_the_largest_value(dtype, tdt, T):
    """A mask of the type's lowest value is a logit like any other, whatever the temperature: a row of nothing else is an
    even teacher, not an empty one; only -inf is left out."""
    h, W, b, ids, t = make(12, 64, 300, 6, dtype, tdt=tdt)
    low, high = torch.finfo(tdt).min, torch.finfo(tdt).max
    t[0] = low
    t[1, 1:] = low
    t[2, ::2] = -math.inf
    t[2, 1::2] = low
    t[3] = high
    t[4, :2] = high
    t[5] = -math.inf
    t[6, 3:] = high
    t[6, :3] = low
    check_shifted(h, W, b, ids, t, T)
    each = swvr.softmax_distill(h, W, ids, t, b, temperature=T, reduction="none")
    assert bool(each.isfinite().all()) and float(each[5]) == 0
    even = swvr.softmax_distill(h, W, ids, torch.zeros_like(t), b, temperature=T, reduction="none")
    assert torch.equal(each[:1], even[:1]) and torch.equal(each[3:4], even[3:4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_logits_at_low_temperatures(dtype):
    """Logits of a few thousand with differences of a few units, T below one."""
    h, W, b, ids, t = make(30, 64, 400, 7, dtype)
    t = (t + 3000).detach()
    check_shifted(h, W, b, ids, t, 0.3)
    L = torch.logsumexp(t.double() / 0.3, 1).float()
    check(h, W, b, ids, t, T=0.3, t_lse=L)


@pytest.mark.parametrize("dtype,N,K,V", [(torch.float16, 517, 512, 10007), (torch.float32, 517, 64, 10007),
                                         (torch.bfloat16, 2048, 512, 40000)])
def test_same_bits_at_sizes_whose_sums_are_split(dtype, N, K, V):
    """dh summed over slices, dW and db over many chunks: the same bits whatever ran before."""
    h, W, b, ids, t = make(N, K, 64, 20, dtype)
    gen = torch.Generator(device="cuda").manual_seed(3)
    W = (K ** -0.5 * torch.randn(V, K, generator=gen, device="cuda")).to(dtype).requires_grad_(True)
    b = torch.randn(V, generator=gen, device="cuda").to(dtype).requires_grad_(True)
    ids = torch.randint(0, V, ids.shape, generator=gen, device="cuda")
    first = run(h, W, b, ids, t)
    for _ in range(3):
        torch.randn(1 << 24, device="cuda").sum()
        loss, grads = run(h, W, b, ids, t)
        assert torch.equal(loss, first[0]) and all(torch.equal(a, c) for a, c in zip(grads[:3], first[1][:3]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ["entries", "tokens"])
def test_small_gradients_of_the_bias_keep_their_bits(dtype, case):
    """Rows of the bias whose student and teacher probabilities are e^-30 and less, or which get entries only of
    tokens with a small upstream gradient: to the same relative accuracy as the others."""
    N, K, V = 40, 64, 500
    h, W, b, ids, t = make(N, K, V, 24, dtype, spread=4.0)
    b = b.detach().float().requires_grad_(True)
    if case == "entries":
        t = 8 * t
        check(h, W, b, ids, t, T=0.5)
        return
    with torch.no_grad():  # each half of the vocabulary is what half of the tokens know
        b[: V // 2] = 0
        half = (torch.arange(N, device="cuda") % 2 == 0)
        h[:, 0] = torch.where(half, 6.0, -6.0).to(dtype)
        W[:, 0] = torch.where(torch.arange(V, device="cuda") < V // 2, 4.0, -4.0).to(dtype)
    ids = ids % (V // 2) + torch.where(half, 0, V // 2)[:, None]
    up = torch.where(half, 1.0, 2.0 ** -50).cuda()
    check(h, W, b, ids, t, reduction="none", up=up)
