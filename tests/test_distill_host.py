"""CPU tests of the distillation loss: argument validation before any device work, the C ABI's
host-side checks and workspace planning, and the custom ops' fake impls."""
import ctypes

import pytest
import torch

import swvr_b200 as swvr
from swvr_b200 import _native as nat


def _args(N=6, K=12, V=41, Kt=3):
    return torch.randn(N, K), torch.randn(V, K), torch.randint(0, V, (N, Kt)), torch.randn(N, Kt)


def test_distill_validates_before_any_device_work():
    h, W, ids, t = _args()
    f = swvr.softmax_distill
    with pytest.raises(ValueError, match="2-D"):
        f(h, W[0], ids, t)
    with pytest.raises(ValueError, match="hidden size"):
        f(h, W[:, :-1], ids, t)
    with pytest.raises(ValueError, match="no vocabulary"):
        f(h, W[:0], ids, t)
    with pytest.raises(ValueError, match="bias"):
        f(h, W, ids, t, torch.randn(40))
    with pytest.raises(ValueError, match="teacher_ids and teacher_logits"):
        f(h, W, ids[:-1], t[:-1])
    with pytest.raises(ValueError, match="teacher_ids and teacher_logits"):
        f(h, W, ids, t[:, :-1])
    with pytest.raises(ValueError, match="int64 or int32"):
        f(h, W, ids.float(), t)
    with pytest.raises(ValueError, match="at most 1024"):
        f(h, W, ids.repeat(1, 400), t.repeat(1, 400))
    with pytest.raises(ValueError, match="teacher_lse"):
        f(h, W, ids, t, teacher_lse=torch.zeros(5))
    with pytest.raises(ValueError, match="weight"):
        f(h, W, ids, t, weight=torch.zeros(6, 1))
    with pytest.raises(ValueError, match="reduction"):
        f(h, W, ids, t, reduction="max")
    for T in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            f(h, W, ids, t, temperature=T)
    with pytest.raises(ValueError, match="chunk_size"):
        f(h, W, ids, t, chunk_size=-1)
    with pytest.raises(ValueError, match="unsupported dtype"):
        f(h, W, ids, t.long())
    with pytest.raises(RuntimeError, match="CUDA devices only"):  # no CPU fallback
        f(h, W, ids, t)


def test_distill_is_reached_under_both_package_names():
    import swvr as alias
    assert alias.softmax_distill is swvr.softmax_distill and alias.SoftmaxDistill is swvr.SoftmaxDistill
    head = torch.nn.Linear(12, 41)
    m = swvr.SoftmaxDistill(head, temperature=2.0)
    assert m.head is head
    h, _, ids, t = _args()
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        m(h, ids, t)


def _problem(N=256, K=64, V=1000, Kt=8, dt=nat.BF16, buf=1 << 20, **kw):
    p = nat.Distill()
    p.n_tokens, p.hidden, p.vocab, p.teacher = N, K, V, Kt
    p.compute_dtype, p.bias_dtype, p.teacher_dtype, p.id_bits = dt, nat.F32, nat.F32, 64
    p.h = p.W = p.teacher_ids = p.teacher_logits = p.slogq = p.z = p.lse = p.lse_lo = p.qsum = p.each = p.stats = p.sid = buf
    p.ldh = p.ldw = K
    p.logit_scale = p.temperature = 1.0
    p.chunk, p.reduction = 8192, nat.REDUCE_MEAN
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("bad,code", [
    (dict(N=-1), nat.ERR_INVALID_ARGUMENT), (dict(Kt=-1), nat.ERR_INVALID_ARGUMENT), (dict(Kt=1025), nat.ERR_UNSUPPORTED),
    (dict(dt=7), nat.ERR_INVALID_ARGUMENT), (dict(teacher_dtype=9), nat.ERR_INVALID_ARGUMENT),
    (dict(id_bits=16), nat.ERR_INVALID_ARGUMENT), (dict(chunk=0), nat.ERR_INVALID_ARGUMENT),
    (dict(temperature=0.0), nat.ERR_INVALID_ARGUMENT), (dict(temperature=float("nan")), nat.ERR_INVALID_ARGUMENT),
    (dict(reduction=5), nat.ERR_INVALID_ARGUMENT), (dict(ldh=32), nat.ERR_INVALID_ARGUMENT),
    (dict(V=0), nat.ERR_UNSUPPORTED), (dict(K=12), nat.ERR_UNSUPPORTED), (dict(h=(1 << 20) + 2), nat.ERR_UNSUPPORTED),
    (dict(sid=None), nat.ERR_INVALID_ARGUMENT), (dict(lse=None), nat.ERR_INVALID_ARGUMENT),
    (dict(stats=None), nat.ERR_INVALID_ARGUMENT), (dict(V=(1 << 31) - 1), nat.ERR_UNSUPPORTED),
])
def test_distill_abi_argument_validation(bad, code):
    n = ctypes.c_size_t(0)
    assert nat.lib().swvr_distill_fwd_workspace_size(_problem(**bad), ctypes.byref(n)) == code
    assert nat.last_error()


def test_distill_abi_rejects_before_any_launch():
    lib, buf, n = nat.lib(), 1 << 20, ctypes.c_size_t(0)
    p = _problem()
    assert lib.swvr_distill_fwd_workspace_size(p, ctypes.byref(n)) == nat.OK and n.value > 0
    assert lib.swvr_distill_fwd(p, None, buf, n.value, None) == nat.ERR_INVALID_ARGUMENT
    assert lib.swvr_distill_fwd(p, buf, None, n.value, None) == nat.ERR_INVALID_ARGUMENT
    assert lib.swvr_distill_fwd(p, buf, buf, n.value - 1, None) == nat.ERR_WORKSPACE
    g = nat.DistillGrads()
    assert lib.swvr_distill_bwd(p, g, buf, 1 << 40, None) == nat.ERR_INVALID_ARGUMENT  # no grad_out
    g.grad_out, g.grad_W, g.grad_W_dtype, g.ld_grad_W = buf, buf, nat.BF16, 64
    assert lib.swvr_distill_bwd_workspace_size(p, g, ctypes.byref(n)) == nat.OK
    assert lib.swvr_distill_bwd(p, g, buf, n.value - 1, None) == nat.ERR_WORKSPACE
    g.grad_W_dtype = nat.F16
    assert lib.swvr_distill_bwd(p, g, buf, 1 << 40, None) == nat.ERR_UNSUPPORTED
    g.grad_W_dtype, g.grad_W = nat.BF16, buf + 8
    assert lib.swvr_distill_bwd(p, g, buf, 1 << 40, None) == nat.ERR_UNSUPPORTED
    g.grad_W, g.ld_grad_W = buf, 32
    assert lib.swvr_distill_bwd(p, g, buf, 1 << 40, None) == nat.ERR_INVALID_ARGUMENT
    g.grad_W, g.grad_weight = None, buf
    assert lib.swvr_distill_bwd(p, g, buf, 1 << 40, None) == nat.ERR_INVALID_ARGUMENT  # no weight
    g.grad_weight, g.grad_h, g.grad_h_dtype = None, buf, 11
    assert lib.swvr_distill_bwd(p, g, buf, 1 << 40, None) == nat.ERR_INVALID_ARGUMENT


def test_distill_workspace_holds_chunks_not_scores():
    lib, n = nat.lib(), ctypes.c_size_t(0)
    p = _problem(N=8192, K=2560, V=152064, Kt=64)
    assert lib.swvr_distill_fwd_workspace_size(p, ctypes.byref(n)) == nat.OK and n.value < 16 * 2 ** 20
    g = nat.DistillGrads()
    g.grad_out = g.grad_h = g.grad_W = 1 << 20
    g.grad_W_dtype, g.ld_grad_W = nat.BF16, 2560
    assert lib.swvr_distill_bwd_workspace_size(p, g, ctypes.byref(n)) == nat.OK
    assert n.value < 16384 * 8192 * 2 + 8192 * 2560 * 4 + 2 ** 20  # one dS chunk and the fp32 dh


@pytest.mark.parametrize("dtype,adt", [(torch.bfloat16, torch.float32), (torch.float64, torch.float64)])
def test_distill_fake_impls_give_shapes(dtype, adt):
    m = lambda *s, dt=dtype: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
    h, W, b, ids, t, w = m(6, 16), m(100, 16), m(100), m(6, 5, dt=torch.int64), m(6, 5, dt=torch.float32), m(6, dt=adt)
    out, *saved = torch.ops.swvr_b200.distill(h, W, b, ids, t, None, w, 2.0, 1.0, 8192, dtype, nat.REDUCE_MEAN)
    assert out.shape == () and out.dtype == adt
    assert [tuple(s.shape) for s in saved] == [(6, 5), (2 * 30 + 4 * 6 + 2,)] and saved[0].dtype == torch.int32
    none = torch.ops.swvr_b200.distill(h, W, b, ids, t, None, w, 2.0, 1.0, 8192, dtype, nat.REDUCE_NONE)[0]
    assert none.shape == (6,)
    grads = torch.ops.swvr_b200.distill_bwd(out, h, W, b, ids, t, None, w, *saved, 2.0, 1.0, 8192, dtype, nat.REDUCE_MEAN,
                                            True, False, True, True)
    assert [tuple(g.shape) for g in grads] == [(6, 16), (0,), (100,), (6,)] and grads[3].dtype == adt


@pytest.mark.parametrize("field", ["N", "V"])
def test_sizes_within_a_tile_of_2_31_are_refused(field):
    """A tile's last row index has to fit an int."""
    lib, n = nat.lib(), ctypes.c_size_t(0)
    small = dict(N=1, V=1, Kt=1)
    for size, code in ((2 ** 31 - 512, nat.OK), (2 ** 31 - 511, nat.ERR_UNSUPPORTED)):
        assert lib.swvr_distill_fwd_workspace_size(_problem(**{**small, field: size}), ctypes.byref(n)) == code
    assert lib.swvr_distill_bwd_workspace_size(_problem(**small, chunk=2 ** 62), nat.DistillGrads(), ctypes.byref(n)) == nat.OK
