"""CPU tests of sampling: argument validation before any device work, the C ABI's host-side checks
and the custom ops' fake impls."""
import ctypes

import pytest
import torch

import swvr_b200 as swvr
from swvr_b200 import _native as nat


def test_sampling_validates_before_any_device_work():
    x, u = torch.randn(3, 2, 40), torch.rand(3, 2)
    f = swvr.sample_logits
    with pytest.raises(ValueError, match="vocabulary dimension"):
        f(x[0, 0, 0], u[0, 0])
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        f(x.double(), u)
    with pytest.raises(ValueError, match="u must have shape"):
        f(x, u[0])
    with pytest.raises(ValueError, match="unsupported dtype"):
        f(x, u.long())
    for T in (-0.1, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            f(x, u, temperature=T)
    for k in (0, -1):
        with pytest.raises(ValueError, match="top_k"):
            f(x, u, top_k=k)
    for p in (0.0, 1.1, float("nan")):
        with pytest.raises(ValueError, match="top_p"):
            f(x, u, top_p=p)
    for m in (-0.1, 1.1):
        with pytest.raises(ValueError, match="min_p"):
            f(x, u, min_p=m)
    with pytest.raises(ValueError, match="top_k"):
        f(x, u, top_k=torch.ones(3, 2))
    for name in ("temperature", "top_k", "top_p", "min_p"):
        with pytest.raises(ValueError, match=name):
            f(x, u, **{name: torch.ones(3, dtype=torch.int32)})
    with pytest.raises(RuntimeError, match="CUDA devices only"):  # no CPU fallback
        f(x, u)
    h, W = torch.randn(3, 2, 8), torch.randn(40, 8)
    g = swvr.softmax_sample
    with pytest.raises(ValueError, match="2-D"):
        g(h, W[0], u)
    with pytest.raises(ValueError, match="hidden size"):
        g(h, W[:, 1:], u)
    with pytest.raises(ValueError, match="bias"):
        g(h, W, u, torch.randn(39))
    with pytest.raises(ValueError, match="computes in"):
        g(h.double(), W.double(), u)
    with pytest.raises(ValueError, match="u must have shape"):
        g(h, W, u[0])
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        g(h, W, u)


def test_sampling_is_reached_under_both_package_names():
    import swvr as alias
    assert alias.softmax_sample is swvr.softmax_sample and alias.sample_logits is swvr.sample_logits


def _sampling(buf=1 << 20, **kw):
    s = nat.Sampling()
    s.temperature, s.top_p, s.min_p, s.top_k, s.u, s.u_dtype, s.tokens = 1.0, 1.0, 0.0, 0, buf, nat.F32, buf
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("bad", [
    dict(temperature=-1.0), dict(temperature=float("inf")), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.5),
    dict(min_p=2.0), dict(top_k=-1), dict(u=None), dict(tokens=None), dict(u_dtype=7),
    dict(temperatures=1 << 20, temperatures_dtype=9), dict(top_ks=1 << 20, top_ks_bits=8)])
def test_sampling_abi_checks_settings(bad):
    lib, buf = nat.lib(), 1 << 20
    assert lib.swvr_sample_logits(4, 100, buf, nat.F32, 100, _sampling(**bad), None) == nat.ERR_INVALID_ARGUMENT
    assert nat.last_error()


def test_sampling_abi_rejects_before_any_launch():
    lib, buf, n = nat.lib(), 1 << 20, ctypes.c_size_t(0)
    f = lambda N=4, V=100, x=buf, dt=nat.F32, ld=100, s=None: lib.swvr_sample_logits(N, V, x, dt, ld, s or _sampling(), None)
    assert f(N=-1) == f(V=-1) == f(ld=99) == f(x=None) == nat.ERR_INVALID_ARGUMENT
    assert f(dt=nat.F64) == f(N=1 << 28) == f(V=1 << 31, ld=1 << 31) == nat.ERR_UNSUPPORTED
    assert f(N=0) == nat.OK
    p = nat.Problem()
    p.n_tokens, p.hidden, p.vocab, p.compute_dtype, p.bias_dtype = 4, 64, 1000, nat.BF16, nat.F32
    p.h = p.W = buf
    p.ldh = p.ldw = 64
    p.logit_scale = 1.0
    assert lib.swvr_sample_workspace_size(p, ctypes.byref(n)) == nat.OK and n.value == 4 * 1000 * 4
    assert lib.swvr_sample(p, _sampling(), buf, n.value - 1, None) == nat.ERR_WORKSPACE
    assert lib.swvr_sample(p, _sampling(), None, n.value, None) == nat.ERR_INVALID_ARGUMENT
    assert lib.swvr_sample(p, _sampling(top_p=0.0), buf, n.value, None) == nat.ERR_INVALID_ARGUMENT
    for field, value, code in (("compute_dtype", nat.F64, nat.ERR_UNSUPPORTED), ("h", buf + 2, nat.ERR_UNSUPPORTED),
                               ("ldh", 32, nat.ERR_INVALID_ARGUMENT), ("W", None, nat.ERR_INVALID_ARGUMENT),
                               ("hidden", 60, nat.ERR_UNSUPPORTED), ("vocab", -1, nat.ERR_INVALID_ARGUMENT)):
        old = getattr(p, field)
        setattr(p, field, value)
        assert lib.swvr_sample_workspace_size(p, ctypes.byref(n)) == code, field
        setattr(p, field, old)
    p.n_tokens, p.vocab = 100000, 152064
    assert lib.swvr_sample_workspace_size(p, ctypes.byref(n)) == nat.OK and n.value <= 256 * 2 ** 20


def test_sampling_fake_impls_give_shapes():
    m = lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
    rest = (1.0, 0, 1.0, 0.0, None, None, None, None)
    tok, lp = torch.ops.swvr_b200.sample_logits(m(5, 90), m(5), *rest, True)
    assert tok.shape == lp.shape == (5,) and tok.dtype == torch.int64 and lp.dtype == torch.float32
    tok, lp = torch.ops.swvr_b200.sample(m(5, 16), m(90, 16), None, m(5), 1.0, torch.bfloat16, *rest, False)
    assert tok.shape == (5,) and lp.shape == (0,)


def test_a_vocabulary_within_a_tile_of_2_31_is_refused():
    """A tile's last row index has to fit an int."""
    lib, n = nat.lib(), ctypes.c_size_t(0)
    p = nat.Problem()
    p.n_tokens, p.hidden, p.compute_dtype, p.bias_dtype = 1, 64, nat.BF16, nat.F32
    p.h = p.W = 1 << 20
    p.ldh = p.ldw = 64
    p.logit_scale = 1.0
    for vocab, code in ((2 ** 31 - 512, nat.OK), (2 ** 31 - 511, nat.ERR_UNSUPPORTED)):
        p.vocab = vocab
        assert lib.swvr_sample_workspace_size(p, ctypes.byref(n)) == code
