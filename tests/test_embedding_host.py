"""CPU tests of the embedding lookup: argument validation before any device work, the C ABI's
host-side checks and the custom ops' fake impls."""
import ctypes

import pytest
import torch

import swvr_b200 as swvr
from swvr_b200 import _native as nat


def test_lookup_validates_before_any_device_work():
    E, tok = torch.randn(11, 4), torch.tensor([1, 2])
    with pytest.raises(ValueError, match="2-D"):
        swvr.embedding_lookup(tok, E[0])
    with pytest.raises(ValueError, match="int64 or int32"):
        swvr.embedding_lookup(tok.float(), E)
    with pytest.raises(ValueError, match="int64 or int32"):
        swvr.embedding_lookup(tok.to(torch.int16), E)
    for bad in (11, -12):
        with pytest.raises(ValueError, match="padding_idx"):
            swvr.embedding_lookup(tok, E, padding_idx=bad)
    with pytest.raises(ValueError, match="unsupported dtype"):
        swvr.embedding_lookup(tok, E.to(torch.int8))
    with pytest.raises(RuntimeError, match="CUDA devices only"):  # no CPU fallback
        swvr.embedding_lookup(tok, E)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        swvr.embedding_lookup(tok, E.requires_grad_(True))


def test_lookup_is_reached_under_both_package_names():
    import swvr as alias
    assert alias.embedding_lookup is swvr.embedding_lookup


def test_embed_abi_rejects_bad_arguments_on_the_host():
    lib = nat.lib()
    buf, bad = 1 << 20, nat.ERR_INVALID_ARGUMENT
    fwd = lambda n=4, V=9, D=8, tok=buf, bits=64, E=buf, dt=nat.BF16, ld=8, out=buf: lib.swvr_embed_fwd(
        n, V, D, tok, bits, E, dt, ld, 1.0, out, None)
    assert fwd(n=-1) == bad and fwd(V=-1) == bad and fwd(D=-1) == bad
    assert fwd(bits=16) == bad and fwd(dt=9) == bad and fwd(ld=7) == bad
    assert fwd(tok=None) == bad and fwd(E=None) == bad and fwd(out=None) == bad
    assert fwd(n=1 << 31) == nat.ERR_UNSUPPORTED and fwd(V=(1 << 31) - 1) == nat.ERR_UNSUPPORTED
    assert fwd(n=0) == nat.OK and fwd(D=0, ld=0) == nat.OK  # nothing to do, nothing launched
    size = ctypes.c_size_t(0)
    assert lib.swvr_embed_bwd_workspace_size(4, 9, 8, nat.BF16, ctypes.byref(size)) == nat.OK and size.value > 0
    assert lib.swvr_embed_bwd_workspace_size(4, 9, 8, nat.BF16, None) == bad
    need = size.value
    bwd = lambda n=4, V=9, D=8, bits=64, g=buf, ldg=8, dE=buf, dt=nat.BF16, ld=8, ws=buf, nb=need: lib.swvr_embed_bwd(
        n, V, D, buf, bits, g, ldg, 1.0, -1, dE, dt, ld, ws, nb, None)
    assert bwd(nb=need - 1) == nat.ERR_WORKSPACE
    assert bwd(ldg=7) == bad and bwd(ld=7) == bad and bwd(g=None) == bad and bwd(dE=None) == bad and bwd(ws=None) == bad
    assert bwd(bits=8) == bad and bwd(dt=-1) == bad
    assert bwd(V=0, dE=None) == nat.OK


def test_embed_workspace_stays_small():
    """The sort's pairs twice, its counters and one pair of partial rows per chunk, not a [V, D] copy."""
    size = ctypes.c_size_t(0)
    assert nat.lib().swvr_embed_bwd_workspace_size(16384, 152064, 2560, nat.BF16, ctypes.byref(size)) == nat.OK
    assert size.value < 40 * 2 ** 20


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float64])
def test_embed_fake_impls_give_shapes(dtype):
    E = torch.empty(9, 5, dtype=dtype, device="meta")
    tok = torch.empty(6, dtype=torch.int64, device="meta")
    out = torch.ops.swvr_b200.embed(tok, E, 2.0, -1)
    assert out.shape == (6, 5) and out.dtype == dtype
    dE = torch.ops.swvr_b200.embed_bwd(out, tok, 9, 2.0, -1)
    assert dE.shape == (9, 5) and dE.dtype == dtype
