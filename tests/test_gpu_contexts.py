"""The library in several CUDA contexts of one device, one after another, as a host without torch may use it."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CHILD = r"""
import ctypes as c, struct
from swvr_b200 import _native as nat
cu = c.CDLL("libcuda.so.1")
def ok(rc):
    assert rc == 0, rc
ok(cu.cuInit(0))
dev = c.c_int(0)
ok(cu.cuDeviceGet(c.byref(dev), 0))
def alloc(n, host=None):
    p = c.c_uint64(0)
    ok(cu.cuMemAlloc_v2(c.byref(p), c.c_size_t(n)))
    ok(cu.cuMemcpyHtoD_v2(p, host if host is not None else bytes(n), c.c_size_t(n)))
    return p.value
def fetch(p, n):
    b = c.create_string_buffer(n)
    ok(cu.cuMemcpyDtoH_v2(b, c.c_uint64(p), c.c_size_t(n)))
    return b.raw
for turn in range(3):
    ctx = c.c_void_p()
    ok(cu.cuCtxCreate_v2(c.byref(ctx), 0, dev))
    # the lookup's gradient: tokens 2, 0, 2 of a 4 x 2 table
    g = alloc(24, struct.pack("6f", 1, 2, 3, 4, 5, 6))
    tok = alloc(24, struct.pack("3q", 2, 0, 2))
    n, dE = c.c_size_t(0), alloc(32)
    nat.check(nat.lib().swvr_embed_bwd_workspace_size(3, 4, 2, nat.F32, c.byref(n)), "size")
    ws = alloc(n.value)
    nat.check(nat.lib().swvr_embed_bwd(3, 4, 2, tok, 64, g, 2, 1.0, -1, dE, nat.F32, 2, ws, n.value, None), "embed_bwd")
    ok(cu.cuCtxSynchronize())
    assert struct.unpack("8f", fetch(dE, 32)) == (3, 4, 0, 0, 6, 8, 0, 0), turn
    # the head: one row, two tokens, the second the larger score
    p, s = nat.Problem(), nat.Sampling()
    p.n_tokens, p.hidden, p.vocab, p.compute_dtype, p.ldh, p.ldw, p.logit_scale = 1, 8, 2, nat.F16, 8, 8, 1.0
    p.h = alloc(16, struct.pack("8e", *[1] * 8))
    p.W = alloc(32, struct.pack("16e", *[0] * 8, *[1] * 8))
    s.temperature, s.top_p, s.u, s.u_dtype, s.tokens = 0.0, 1.0, alloc(4), nat.F32, alloc(8)
    nat.check(nat.lib().swvr_sample_workspace_size(p, c.byref(n)), "size")
    nat.check(nat.lib().swvr_sample(p, s, alloc(n.value), n.value, None), "sample")
    ok(cu.cuCtxSynchronize())
    assert struct.unpack("q", fetch(s.tokens, 8)) == (1,), turn
    ok(cu.cuCtxDestroy_v2(ctx))
print("three contexts")
"""


def test_kernel_attributes_are_those_of_the_current_context():
    """Shared memory beyond 48 KiB is allowed per context, not per device."""
    res = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=120,
                         env={**os.environ, "PYTHONPATH": ROOT})
    assert res.returncode == 0 and "three contexts" in res.stdout, res.stderr[-2000:]
