"""CPU tests of the sizes at which the token operators' launches and workspaces have to give way."""
import ctypes

import pytest

from swvr_b200 import _native as nat
from test_distill_host import _problem


def test_fp32_head_takes_tiny_vocabularies_in_chunks_of_rows():
    """The fp32 product has at most 65535 row tiles of 128 in a launch."""
    lib, n = nat.lib(), ctypes.c_size_t(0)
    p = nat.Problem()
    p.hidden, p.compute_dtype, p.bias_dtype = 8, nat.F32, nat.F32
    p.h = p.W = 1 << 20
    p.ldh = p.ldw = 8
    p.logit_scale = 1.0
    for vocab in (1, 4, 8):
        p.vocab = vocab
        for rows in (65535 * 128, 65535 * 128 + 1, (1 << 28) - 1):
            p.n_tokens = rows
            assert lib.swvr_sample_workspace_size(p, ctypes.byref(n)) == nat.OK
            assert n.value == min(65535 * 128, (256 << 20) // (16 * ((vocab + 3) // 4))) * 16 * ((vocab + 3) // 4)


@pytest.mark.parametrize("dt", [nat.F32, nat.F64])
def test_exact_path_takes_what_its_products_can_launch(dt):
    """At most 65535 row tiles of 128: tokens past that are refused, chunks of the vocabulary are kept to it, and the
    largest sizes that are taken do not wrap the workspace's."""
    lib, n, most = nat.lib(), ctypes.c_size_t(0), 65535 * 128
    g = nat.DistillGrads()
    g.grad_out = g.grad_h = g.grad_W = 1 << 20
    g.ld_grad_W = 1
    for N, code in ((most, nat.OK), (most + 1, nat.ERR_UNSUPPORTED), (2 ** 31 - 512, nat.ERR_UNSUPPORTED)):
        p = _problem(N=N, K=1, V=2 ** 31 - 512, Kt=1, dt=dt, chunk=2 ** 62)
        assert lib.swvr_distill_fwd_workspace_size(p, ctypes.byref(n)) == code
        assert lib.swvr_distill_bwd_workspace_size(p, g, ctypes.byref(n)) == code
    p = _problem(N=most, K=1, V=2 ** 31 - 512, Kt=1, dt=dt, chunk=2 ** 62)
    assert lib.swvr_distill_fwd_workspace_size(p, ctypes.byref(n)) == nat.OK
    assert n.value >= most * most * (8 if dt == nat.F64 else 4)
    p = _problem(N=2 ** 31 - 512, K=8, V=1000, Kt=1, dt=nat.BF16)  # the tensor-core path has no such tiles
    assert lib.swvr_distill_fwd_workspace_size(p, ctypes.byref(n)) == nat.OK


def test_exact_forward_asks_for_no_split_sums():
    """The scores' product is never split along its sum: the forward's workspace is the staged scores, the scaled bias, two
    numbers a token and a counter; the backward adds the gradients of the tokens, dh, and slices of dh and dW where asked for."""
    lib, n = nat.lib(), ctypes.c_size_t(0)
    N, K, V, slack = 1024, 64, 10007, 8192
    p = _problem(N=N, K=K, V=V, Kt=8, dt=nat.F32)
    assert lib.swvr_distill_fwd_workspace_size(p, ctypes.byref(n)) == nat.OK
    fwd = 4 * (N * 8192 + V + 2 * N)
    assert fwd <= n.value <= fwd + slack

    def bwd(h=None, W=None):
        g = nat.DistillGrads()
        g.grad_out, g.grad_h, g.grad_W, g.ld_grad_W = 1 << 20, h, W, K
        assert lib.swvr_distill_bwd_workspace_size(p, g, ctypes.byref(n)) == nat.OK
        return n.value - fwd

    both = 4 * 2 * N  # g T and g T sum q
    assert both <= bwd() <= both + slack
    assert both + 4 * 17 * N * K <= bwd(h=1 << 20) <= both + 4 * 17 * N * K + slack  # dh and 16 slices of it
    assert both + 4 * 16 * 8192 * K <= bwd(W=1 << 20) <= both + 4 * 16 * 8192 * K + slack
    assert both + 4 * (16 * 8192 + N) * K <= bwd(h=1 << 20, W=1 << 20) <= both + 4 * (16 * 8192 + N) * K + slack


def test_workspaces_have_to_be_aligned():
    """The kernels read and write them 16 bytes at a time: one that starts elsewhere is refused before any launch."""
    lib, buf, n = nat.lib(), 1 << 20, ctypes.c_size_t(0)
    for off in (1, 4, 8):
        assert lib.swvr_embed_bwd(4, 9, 8, buf, 64, buf, 8, 1.0, -1, buf, nat.BF16, 8, buf + off, 1 << 30, None) == nat.ERR_UNSUPPORTED
        for dt in (nat.BF16, nat.F32, nat.F64):
            p, g = _problem(dt=dt), nat.DistillGrads()
            g.grad_out = g.grad_bias = p.bias = buf
            assert lib.swvr_distill_fwd(p, buf, buf + off, 1 << 40, None) == nat.ERR_UNSUPPORTED
            assert lib.swvr_distill_bwd(p, g, buf + off, 1 << 40, None) == nat.ERR_UNSUPPORTED
        p, s = nat.Problem(), nat.Sampling()
        p.n_tokens, p.hidden, p.vocab, p.compute_dtype, p.bias_dtype = 4, 64, 1000, nat.BF16, nat.F32
        p.h = p.W = buf
        p.ldh = p.ldw = 64
        p.logit_scale = s.temperature = s.top_p = 1.0
        s.u, s.u_dtype, s.tokens = buf, nat.F32, buf
        assert lib.swvr_sample(p, s, buf + off, 1 << 30, None) == nat.ERR_UNSUPPORTED
    assert "aligned" in nat.last_error()
