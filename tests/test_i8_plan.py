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
