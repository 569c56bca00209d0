"""What the 8-bit and mixture-of-experts launches decide from sizes (csrc/i8_plan.h), compiled for the host and checked
over the sizes that the entry points accept."""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest

from webllm_b200.build_ext import CSRC

SOURCE = """
#include "i8_plan.h"
extern "C" {
void plan_shape(int64_t slots, int E, int most, int* out) {
    const wllm::PlanShape p = wllm::plan_shape(slots, E, most);
    out[0] = p.warps, out[1] = p.ctas, out[2] = p.smem;
}
void plan(int grouped, int M, int K, int N, int E, int64_t slots, int64_t* out) {
    const wllm::I8Shape o{M, K, N, E, slots};
    const wllm::Plan p = grouped ? wllm::plan<true>(o, 148) : wllm::plan<false>(o, 148);
    out[0] = p.mode, out[1] = p.tile_n, out[2] = p.splits, out[3] = p.items;
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


SINGLE, SPLIT, PAIR, PAIR_SHORT = range(4)


def product_plan(host, M, K, N):
    out = (ctypes.c_int64 * 4)()
    host.plan(0, M, K, N, 1, ctypes.c_int64(0), out)
    return tuple(out)


def grouped_plan(host, M, K, E, slots):
    out = (ctypes.c_int64 * 4)()
    host.plan(1, M, K, slots, E, ctypes.c_int64(slots), out)
    return tuple(out)


def check(plan, M, K, most_tiles):
    """What the kernel takes for granted of a plan."""
    mode, tile_n, splits, items = plan
    pair = mode in (PAIR, PAIR_SHORT)
    assert tile_n > 0 and tile_n % (32 if pair else 16) == 0
    assert tile_n <= {SINGLE: 64, SPLIT: 64, PAIR: 256, PAIR_SHORT: 128}[mode]
    assert (mode == SPLIT) == (splits > 1) and splits in (1, 2, 4, 8) and splits <= max(1, -(-K // 256))
    assert not pair or M > 128
    assert 1 <= items <= -(-M // (256 if pair else 128)) * most_tiles(tile_n)
    assert mode != SPLIT or items * splits < 2 ** 31  # a grid of one item a cluster


def test_product_plans(host):
    """Over the sizes that are accepted, their ends among them."""
    rng = np.random.default_rng(11)
    top = 2 ** 31 - 1024
    shapes = [(M, K, N) for M in (1, 128, 129, 50000, top) for K in (1, 16, 4096, 131071) for N in (1, 16, 17, 300, 65537, top)]
    shapes += [tuple(int(np.exp(rng.uniform(0, np.log(hi)))) for hi in (300000, 131071, 100000)) for _ in range(2000)]
    for M, K, N in shapes:
        check(product_plan(host, M, K, N), M, K, lambda t: -(-N // t))  # noqa: B023


def test_grouped_plans(host):
    rng = np.random.default_rng(12)
    top = 2 ** 31 - 1024
    shapes = [(M, K, E, s) for M in (1, 129, top) for K in (1, 2048, 131071) for E in (1, 60, 1024) for s in (1, 8, 5000, top)]
    shapes += [tuple(int(np.exp(rng.uniform(0, np.log(hi)))) for hi in (20000, 20000, 1024, 300000)) for _ in range(2000)]
    for M, K, E, s in shapes:
        check(grouped_plan(host, M, K, E, s), M, K, lambda t: min(s, s // t + E))  # noqa: B023


# A product of each mode, split and token tile that the plan chooses: mode, splits, tile, M, K, N.
PRODUCTS = [
    (SINGLE, 1, 16, 102, 101, 2), (SINGLE, 1, 32, 108, 100, 163), (SINGLE, 1, 48, 101, 115, 563),
    (SINGLE, 1, 64, 100, 121, 1500), (SPLIT, 2, 16, 881, 3388, 146), (SPLIT, 2, 32, 571, 3455, 292),
    (SPLIT, 2, 48, 259, 3967, 828), (SPLIT, 2, 64, 553, 5150, 711), (SPLIT, 4, 16, 139, 2354, 117),
    (SPLIT, 4, 32, 169, 2337, 301), (SPLIT, 4, 48, 296, 2850, 371), (SPLIT, 4, 64, 276, 2909, 674),
    (SPLIT, 8, 16, 103, 1830, 1), (SPLIT, 8, 32, 100, 1830, 171), (SPLIT, 8, 48, 138, 3092, 264),
    (SPLIT, 8, 64, 267, 5363, 199), (PAIR, 1, 160, 132, 123, 138), (PAIR, 1, 192, 132, 111, 164),
    (PAIR, 1, 224, 157, 107, 201), (PAIR, 1, 256, 129, 106, 244), (PAIR_SHORT, 1, 32, 133, 143, 191),
    (PAIR_SHORT, 1, 64, 159, 135, 513), (PAIR_SHORT, 1, 96, 1009, 130, 883), (PAIR_SHORT, 1, 128, 945, 143, 1199),
]
# The same of grouped ones: .., M, K, E, tokens, experts of each.
GROUPS = [
    (SINGLE, 1, 16, 105, 100, 3, 2, 1), (SINGLE, 1, 32, 109, 107, 5, 271, 5), (SINGLE, 1, 48, 104, 117, 3, 868, 3),
    (SINGLE, 1, 64, 286, 132, 4, 362, 4), (SPLIT, 2, 16, 136, 3365, 12, 28, 7), (SPLIT, 2, 32, 207, 4562, 3, 502, 1),
    (SPLIT, 2, 48, 167, 6417, 4, 183, 4), (SPLIT, 2, 64, 262, 6475, 3, 627, 1), (SPLIT, 4, 16, 130, 2488, 3, 29, 2),
    (SPLIT, 4, 32, 130, 3287, 3, 178, 1), (SPLIT, 4, 48, 129, 2891, 6, 106, 2), (SPLIT, 4, 64, 135, 3656, 4, 92, 4),
    (SPLIT, 8, 16, 104, 1835, 3, 2, 3), (SPLIT, 8, 32, 135, 1885, 3, 13, 3), (SPLIT, 8, 48, 135, 3187, 3, 107, 1),
    (SPLIT, 8, 64, 137, 3488, 4, 62, 2), (PAIR, 1, 192, 151, 109, 3, 45, 3), (PAIR, 1, 256, 260, 127, 15, 342, 7),
    (PAIR_SHORT, 1, 32, 156, 131, 3, 198, 3), (PAIR_SHORT, 1, 64, 259, 153, 4, 247, 3),
    (PAIR_SHORT, 1, 128, 270, 144, 3, 501, 3),
]

# Of every mode one whose items' MMAs take 10 us and more, one or two items a CTA: mode, splits, M, K, E (0: dense), tokens.
LONG = [
    (SINGLE, 1, 17920, 65536, 0, 16), (SPLIT, 8, 128, 131056, 0, 1), (SPLIT, 8, 256, 131056, 0, 256),
    (PAIR, 1, 17920, 16384, 0, 256), (PAIR_SHORT, 1, 17920, 32768, 0, 64),
    (SINGLE, 1, 128, 16384, 200, 200), (SPLIT, 8, 128, 131056, 1, 3), (PAIR, 1, 17920, 16384, 1, 256),
    (PAIR_SHORT, 1, 17920, 32768, 1, 64),
]


def test_products_of_every_mode(host):
    """The sizes that the GPU tests run, so that each of the kernel's forms is reached."""
    for *form, M, K, N in PRODUCTS:
        assert product_plan(host, M, K, N)[:3] == (form[0], form[2], form[1])
    for *form, M, K, E, T, k in GROUPS:
        assert grouped_plan(host, M, K, E, T * k)[:3] == (form[0], form[2], form[1])
    every = {(SINGLE, 1), (SPLIT, 2), (SPLIT, 4), (SPLIT, 8), (PAIR, 1), (PAIR_SHORT, 1)}
    assert {(c[0], c[1]) for c in PRODUCTS} == every and {(c[0], c[1]) for c in GROUPS} == every
    for mode, splits, M, K, E, N in LONG:
        plan = grouped_plan(host, M, K, E, N) if E else product_plan(host, M, K, N)
        assert (plan[0], plan[2]) == (mode, splits)
