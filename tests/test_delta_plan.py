"""The chunked delta rule's arithmetic of launches (csrc/delta_plan.h, which host and device share), built for the CPU:
no launch reads a record that its workspace does not hold, and the GPU tests' shapes reach every width of the chain.
No GPU needed."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "df-ssm_amd", "csrc")
SOURCE = """
#include "delta_plan.h"
extern "C" void pass_chunks(int64_t first, int64_t nch, int64_t slot0, int64_t slot1, int64_t* out) {
  const dfssm::PassChunks p = dfssm::pass_chunks(first, nch, slot0, slot1);
  out[0] = p.begin;
  out[1] = p.count;
}
extern "C" int chain_tiles(int64_t heads, int64_t tiles) { return dfssm::chain_tiles(heads, tiles); }
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + CSRC, str(d / "plan.cpp"),
                    "-o", str(d / "plan.so")], check=True)
    return ctypes.CDLL(str(d / "plan.so"))


def pass_chunks(plan, *args):
    out = (ctypes.c_int64 * 2)()
    plan.pass_chunks(*(ctypes.c_int64(x) for x in args), out)
    return out[0], out[1]


LENS = {"empty last": [80000, 0], "empty first": [0, 80000], "empty all round": [0, 15000, 0, 0, 9000, 0, 0],
        "short": [1, 0, 63, 64, 65, 0, 128, 1000] * 40, "one": [100000], "none": [0] * 300 + [7] + [0] * 300}


@pytest.mark.parametrize("per", [1, 3, 64, 303, 1213])
@pytest.mark.parametrize("name", LENS)
def test_records_of_a_pass(plan, name, per):
    """Sequence b has its chunks from slot floor(t0 / 64) + b on. Over the passes every chunk comes once and in order,
    and what a launch reads of the records lies in the `per` slots that it holds."""
    lens = LENS[name]
    first = np.concatenate([[0], np.cumsum(lens)])
    slots = int(first[-1]) // 64 + len(lens)
    for b, n in enumerate(lens):
        at, nch, done = int(first[b]) // 64 + b, (n + 63) // 64, 0
        for slot0 in range(0, slots, per):
            slot1 = min(slot0 + per, slots)
            begin, count = pass_chunks(plan, at, nch, slot0, slot1)
            assert count >= 0, (b, slot0)
            if count:
                assert begin == done and slot0 <= at + begin and at + begin + count <= slot1, (b, slot0)
                done += count
        assert done == nch


def tiles_of(plan, lens, Hv, Dv):
    return plan.chain_tiles(ctypes.c_int64(len(lens) * Hv), ctypes.c_int64(Dv // 16))


def test_shapes_of_the_gpu_tests(plan):
    """A change of the rule must not leave a width without a test."""
    import test_gpu_delta_nonfinite as nonfinite
    import test_gpu_delta_overwrite as overwrite
    import test_gpu_delta_widths as widths
    for want, (lens, _, Hv, Dv) in widths.SHAPES:
        assert tiles_of(plan, lens, Hv, Dv) == want
    for module in (nonfinite, overwrite):
        assert {(tiles_of(plan, lens, Hv, Dv)) for lens, _, Hv, _, Dv in module.SHAPES} == {1, 2, 4}
