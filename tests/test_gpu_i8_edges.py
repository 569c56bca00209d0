"""GPU tests of the 8-bit and mixture-of-experts operators at the ends of what they accept, against plain implementations
in 64 bits."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_fresh(code, *args):
    """`code` in a new process, where no call has set a kernel's attributes yet."""
    r = subprocess.run([sys.executable, "-c", code, *map(str, args)], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as expected" in r.stdout, r.stdout[-1500:] + r.stderr[-1500:]


FIRST_PLAN = """
import sys
import numpy as np
import torch
from webllm_b200 import jsep
jsep.install_jsep_callbacks(0)
slots, E = map(int, sys.argv[1:])
ids = np.random.default_rng(slots).integers(-1, E + 1, (slots, 1), dtype=np.int32)
dev, offsets, order = torch.from_numpy(ids).cuda(), torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty(slots, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
jsep.moe_plan(dev.data_ptr(), slots, 1, E, offsets.data_ptr(), order.data_ptr(), stream=jsep.STREAM_LEGACY)
torch.cuda.synchronize()
key = np.where((ids < 0) | (ids >= E), E, ids).flatten().astype(np.int64)
assert np.array_equal(order.cpu().numpy(), np.argsort(key, kind="stable"))
assert np.array_equal(offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]))
print("as expected")
"""


@pytest.mark.parametrize("slots,E", [(2048, 360), (1408, 511), (1900, 383), (16384, 360)])
def test_first_plan_of_a_process(slots, E):
    """Sizes whose shared memory is within 48 KB only without what the kernel holds statically: as the first plan of a
    process (a larger one before it raises the kernel's limit for the rest)."""
    run_fresh(FIRST_PLAN, slots, E)
