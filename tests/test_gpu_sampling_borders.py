"""GPU tests of sampling where the fp32 sums leave a token open under a cut, and of the head against given scores."""
import pytest
import torch

import swvr_b200 as swvr
from test_gpu_sampling import check, exact, near, uniform

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kw", [dict(k=2000), dict(m=1e-9), dict(p=0.999999), dict(k=3000, p=0.99999)])
def test_wide_filters_on_borders_of_the_running_weight(dtype, kw):
    """Over 1024 tokens left, one large score among every eight, u on borders of the running weight: the definition's token,
    and the same in batches of few rows (many CTAs each) as of many (one each)."""
    N, V = 310, 9001
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(N, V, generator=gen, device="cuda") - 9
    x[:, 3::8] += 9
    x = x.to(dtype)
    w = exact(x, uniform(N), **kw)[2].cumsum(1)
    at = torch.randint(0, V, (N, 1), generator=gen, device="cuda")
    u = (w.gather(1, at)[:, 0] / w[:, -1]).clamp(0, 1 - 2.0 ** -53)
    got = check(x, u, **kw)
    for i in range(0, N, 31):
        assert torch.equal(check(x[i:i + 31], u[i:i + 31], **kw), got[i:i + 31])


@pytest.mark.parametrize("kw", [dict(), dict(m=1e-7), dict(k=1500), dict(p=0.99999)])
def test_borders_of_the_longest_rows_with_fp32_sums(kw):
    """734 000 scores and up to 2^20, where the fixed point has its fewest bits under fp32 sums."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    for V in (734003, 1 << 20):
        x = (2 * torch.randn(4, V, generator=gen, device="cuda")).bfloat16()
        w = exact(x, uniform(4), **kw)[2].cumsum(1)
        at = torch.randint(0, V, (4, 1), generator=gen, device="cuda")
        check(x, (w.gather(1, at)[:, 0] / w[:, -1]).clamp(0, 1 - 2.0 ** -53), **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,V", [(1, 64, 5000), (33, 72, 2001), (140, 64, 10007)])
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.7, top_k=50, top_p=0.9), dict(top_p=0.6), dict(min_p=0.03, top_p=0.8),
                                dict(temperature=0.0), dict(top_k=1300, top_p=0.97)])
def test_head_of_small_integers_samples_as_its_scores_do(dtype, N, K, V, kw):
    """Scores of small integers are exact in every compute dtype, so the head has to choose what its scores choose."""
    gen = torch.Generator().manual_seed(N)
    h = torch.randint(-3, 4, (N, K), generator=gen).to(dtype).cuda()
    W = torch.randint(-2, 3, (V, K), generator=gen).to(dtype).cuda()
    b = torch.randint(-8, 9, (V,), generator=gen).to(dtype).cuda()
    u = uniform(N)
    x = (0.125 * (h.double() @ W.double().T) + b.double()).float()  # multiples of 1/8 below 2^10: exact
    got = swvr.softmax_sample(h, W, u, b, logit_scale=0.125, **kw)
    assert torch.equal(got, swvr.sample_logits(x, u, **kw))
    names = dict(temperature="T", top_k="k", top_p="p", min_p="m")
    want, _, w = exact(x, u, **{names[k]: v for k, v in kw.items()})
    assert near(got, want, w, u, V)
