"""The arithmetic by which the many-tensor operators are launched (csrc/plan.h), compiled by itself: no GPU needed."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r'''
#include "plan.h"
extern "C" int past_last_level(int count, const GsrGrad* g) { return gsr::past_last_level(count, g); }
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
