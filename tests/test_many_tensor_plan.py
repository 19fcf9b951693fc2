"""The arithmetic by which the many-tensor operators are launched (csrc/plan.h), compiled by itself: no GPU needed."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r'''
#include "plan.h"
extern "C" int past_last_level(int count, const GsrGrad* g) { return gsr::past_last_level(count, g); }
extern "C" void quotients(uint32_t d, const uint32_t* n, uint32_t* q, uint64_t count) {
  const gsr::Divisor by = gsr::divisor(d);
  for (uint64_t i = 0; i < count; i++) q[i] = by.quotient(n[i]);
}
extern "C" int lies_in_two_rows(uint32_t units, uint32_t unit) { return gsr::lies_in_two_rows(units, unit); }
'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(SOURCE)
    out = str(where / "libplan.so")
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-shared", "-fPIC",
                           "-I", os.path.join(ROOT, "gaussian-splatting-own_amd", "csrc"), str(where / "plan.cpp"), "-o", out])
    return C.CDLL(out)


def test_what_outgrows_the_last_level_cache_is_counted_in_bytes(plan):
    def past(*tensors):
        return plan.past_last_level(len(tensors), (C.c_uint64 * (3 * max(1, len(tensors))))(*[w for t in tensors for w in t]))

    F32, F16, BF16 = 0, 1, 2
    mib = 1 << 20
    assert not past() and not past((0x1000, 64 * mib, F32)) and past((0x1000, 64 * mib + 1, F32))
    for half in (F16, BF16):
        assert not past((0x1000, 128 * mib, half)) and past((0x1000, 128 * mib + 1, half))
    assert past((0x1000, 32 * mib, F32), (0, 0, F32), (0x1000, 64 * mib, BF16), (0x1000, 1, F16))
    assert past((0x1000, 1 << 44, F32)) and past(*[(0x1000, 1 << 40, F32)] * 1000)
    assert not past(*[(0x1000, 3, F32)] * 50_000)                  # 600 KB in many pieces


def test_the_division_of_the_row_kernels_is_exact(plan):
    """Row lengths up to 2^31 - 1 units, numerators over all 32 bits and around every kind of multiple."""
    rng = np.random.default_rng(0)
    spread = np.concatenate([np.arange(70_000), 2 ** 32 - 1 - np.arange(2000), 2 ** 31 + np.arange(-2000, 2000),
                             rng.integers(0, 2 ** 32, 50_000)])
    plan.quotients.argtypes = [C.c_uint32, C.c_void_p, C.c_void_p, C.c_uint64]
    plan.quotients.restype = None
    lengths = list(range(1, 300)) + [1023, 1024, 1025, 4099, 65535, 65536, 65537, 1_000_003, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1,
                                     2 ** 31 - 2, 2 ** 31 - 1] + [int(x) for x in rng.integers(2, 2 ** 31, 100)]
    for d in lengths:
        multiples = (spread // d) * d
        n = np.concatenate([spread, multiples, np.maximum(multiples, 1) - 1, np.minimum(multiples + d - 1, 2 ** 32 - 1)])
        n = np.ascontiguousarray(n, dtype=np.uint32)
        q = np.empty_like(n)
        plan.quotients(d, n.ctypes.data, q.ctypes.data, n.size)
        assert np.array_equal(q, n // np.uint32(d)), d


def test_vectors_that_reach_into_a_third_row_are_told_apart(plan):
    """Against every column that a vector of 16 bytes can begin at."""
    for unit in (1, 2, 4):
        k = 16 // unit
        for units in range(1, 70):
            never = all((v * k) % units + k <= 2 * units for v in range(units))
            wide = bool(plan.lies_in_two_rows(units, unit))
            assert not wide or never, (units, unit)
            assert wide or units < k - 1, (units, unit)
        assert plan.lies_in_two_rows(k // 2, unit)
        assert all(plan.lies_in_two_rows(u, unit) for u in (2 ** 30, 2 ** 31 - 1))
