"""What the 8-bit and mixture-of-experts launches decide from sizes (csrc/i8_plan.h), compiled for the host and checked
over the sizes that the entry points accept."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

from webllm_b200.build_ext import CSRC

SOURCE = """
#include "i8_plan.h"
extern "C" {
void plan_shape(int64_t slots, int E, int most, int* out) {
    const wllm::PlanShape p = wllm::plan_shape(slots, E, most);
    out[0] = p.warps, out[1] = p.ctas, out[2] = p.smem;
}
int piece_bytes(int K, int k) { return wllm::piece_bytes(K, k); }
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("i8_plan")
    src, lib = os.path.join(d, "plan.cpp"), os.path.join(d, "libplan.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", CSRC, "-o", lib, src], check=True)
    return ctypes.CDLL(lib)


def test_gathered_pieces_end_with_the_row(host):
    """Of a row of K bytes its 16-byte pieces read every byte once and none behind it."""
    for K in [*range(1, 300), 1000, 1536, 131071]:
        pieces = [host.piece_bytes(K, k) for k in range(0, K + 256, 16)]
        assert sum(pieces) == K
        assert all(p == 16 for p in pieces[: K // 16]) and all(k + host.piece_bytes(K, k) <= max(K, k) for k in range(0, K + 256, 16))


@pytest.mark.parametrize("most", [8, 16])
def test_plan_cluster_is_one_that_the_device_places(host, most):
    """From no slot to the most that are accepted: at most `most` CTAs (8 where no cluster of 16 can be placed), each with
    work while there are slots for it, and shared memory within what the kernel is allowed."""
    out = (ctypes.c_int * 3)()
    for slots in [*range(0, 2000, 7), 16384, 16385, 65536, 8192 * 8, 10 ** 7, 2 ** 31 - 1024]:
        for E in (1, 60, 360, 1024):
            host.plan_shape(ctypes.c_int64(slots), E, most, out)
            warps, ctas, smem = out
            assert 4 <= warps <= 32 and 1 <= ctas <= most and (ctas == 1 or warps == 32)
            assert smem == (warps + 2) * (E + 1) * 4 <= 227 * 1024 - 1024
            assert ctas == most or 64 * warps * ctas >= slots
