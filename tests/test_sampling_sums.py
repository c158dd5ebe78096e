"""The bound on the sampler's fp32 sums, tried on the host: csrc/sample_sums.cuh is plain C++ as well as CUDA."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from conftest import ROOT

SOURCE = """
#include "sample_sums.cuh"
using namespace swvr::sample;
extern "C" {
float tree4(float* v) { return tree_sum<4>(*reinterpret_cast<float(*)[4]>(v)); }
float tree8(float* v) { return tree_sum<8>(*reinterpret_cast<float(*)[8]>(v)); }
int lg_one(long long V) { return lg_one_of(V); }
unsigned long long error(unsigned long long total) { return rough_error(total); }
int most() { return kRoughMost; }
}
"""


@pytest.fixture(scope="module")
def sums(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    at = tmp_path_factory.mktemp("sums")
    (at / "sums.cpp").write_text(SOURCE)
    out = str(at / "libsums.so")
    subprocess.run([cxx, "-O1", "-std=c++17", "-Wno-unknown-pragmas", "-ffp-contract=off", "-shared", "-fPIC", "-o", out,
                    "-I", os.path.join(ROOT, "swvr_b200", "csrc"), str(at / "sums.cpp")], check=True, capture_output=True)
    lib = ctypes.CDLL(out)
    lib.tree4.restype = lib.tree8.restype = ctypes.c_float
    lib.lg_one.argtypes, lib.error.argtypes, lib.error.restype = [ctypes.c_longlong], [ctypes.c_ulonglong], ctypes.c_ulonglong
    return lib


def packs(vec):
    """One dominant weight with others of half a step of it and a little more or less, at each place; and plain ones."""
    rng = np.random.default_rng(0)
    for at in range(vec):
        for top in (1.0, 1.0 + 2.0 ** -23, 1.4, 0.75):
            for part in (0.49, 0.501, 0.75, 1.49, 1.501):
                v = np.full(vec, part * np.spacing(np.float32(top)), dtype=np.float32)
                v[at] = top
                yield v
    for _ in range(500):
        yield np.exp2(-rng.uniform(0, 26, vec)).astype(np.float32)


@pytest.mark.parametrize("vec", [4, 8])
def test_a_pack_is_summed_in_few_roundings(sums, vec):
    f, depth = getattr(sums, f"tree{vec}"), vec.bit_length() - 1
    for v in packs(vec):
        got = float(f(v.copy().ctypes.data_as(ctypes.POINTER(ctypes.c_float))))
        want = float(np.sum(v.astype(np.float64)))
        assert abs(got - want) <= ((1 + 2.0 ** -24) ** depth - 1) * want


def test_weights_stay_below_the_sign(sums):
    for V in (1, 2, 1 << 18, (1 << 18) + 1, 1 << 19, 734000, 1 << 20, 1 << 24, (1 << 31) - 1):
        assert sums.lg_one(V) <= 44 and V << sums.lg_one(V) <= 1 << 62


def test_the_bound_holds_up_to_the_longest_row(sums):
    """The terms in rough_error's comment, against it, at totals from the least (the largest weight alone, which is
    2^-1/2 of its power of two) up."""
    most = sums.most()
    for V in {1, 1000, 1 << 18, (1 << 18) + 1, 1 << 19, (1 << 19) + 1, 734000, most - 1, most}:
        # units cut off: one a thread of up to eight CTAs of 512, one a thread of the CTA that looks closer, one a score of
        # the 256th of a share at the end
        cut = 8 * 512 + 512 + V // 256 + 256
        for total in (2.0 ** 39.5, 2.0 ** 41 + 12345, V * 2.0 ** 40):
            if total > V * 2.0 ** 40.5:
                continue
            # half a unit a score, the unit being 2^-lg_one of the largest weight, which is part of the total
            fixed = V * 2.0 ** -(sums.lg_one(V) + 1) * min(total, 2.0 ** 40.5)
            assert (0.6 + 4 + 3) * 2.0 ** -24 * total + fixed + cut <= sums.error(int(total)), (V, total)
