"""The lookup of a place's sequence in the chunked operators' launches (csrc/places.h and csrc/scan_plan.h, which host and device
share), built for the CPU: every token of a sequence is in one place, rows of no sequence are in none, and an empty sequence has one
place, wherever the first sequence begins. No GPU needed."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "df-ssm_amd", "csrc")
SOURCE = """
#include "scan_plan.h"
using namespace dfssm;
extern "C" int64_t segment(int64_t n, int n_seq, int64_t w) { return scan_segment(n, n_seq, w); }
extern "C" int64_t places(int64_t n, int n_seq, int64_t seg) { return scan_places(n, n_seq, seg); }
// The sequence that the launch takes for a place, or -1, and the segment of it.
extern "C" int lookup(int64_t place, const int32_t* cu, int n_seq, int seg, int64_t* segment) {
  const int b = last_started(n_seq, [&](int lo, int step, int end) {
    int count = 0;
    for (int lane = 0; lane < 64; ++lane) {
      const int i = lo + lane * step;
      count += i < end && place_of(cu[i], i, seg) <= place;
    }
    return count;
  });
  const int64_t first = place_of(cu[b], b, seg);
  *segment = place - first;
  return scan_holds(place, first, cu[b + 1] - cu[b], seg) ? b : -1;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("places")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + CSRC, str(d / "plan.cpp"),
                    "-o", str(d / "plan.so")], check=True)
    lib = ctypes.CDLL(str(d / "plan.so"))
    lib.segment.restype = lib.places.restype = ctypes.c_int64
    return lib


LENS = {"short": [0, 3, 1, 2] * 160, "even": [30] * 600, "long ones": [5] * 100 + [9000] + [0] * 300 + [700, 0, 65] * 60,
        "few": [700, 0, 3], "one": [5000], "empty": [0] * 520}


@pytest.mark.parametrize("before,behind", [(0, 0), (1000, 0), (6000, 50), (256, 4000), (255, 1)])
@pytest.mark.parametrize("first_empty", [False, True])
@pytest.mark.parametrize("name", LENS)
def test_every_token_once(plan, name, first_empty, before, behind):
    lens = ([0] if first_empty else []) + LENS[name]
    n = len(lens)
    cu = np.cumsum([before] + lens).astype(np.int32)
    T = int(cu[-1]) + behind
    for wgs in (1, 32):
        seg = plan.segment(ctypes.c_int64(T), n, ctypes.c_int64(wgs))
        times, empty = np.zeros(T, dtype=int), np.zeros(n, dtype=int)
        for place in range(plan.places(ctypes.c_int64(T), n, ctypes.c_int64(seg))):
            s = ctypes.c_int64()
            b = plan.lookup(ctypes.c_int64(place), cu.ctypes.data_as(ctypes.c_void_p), n, int(seg), ctypes.byref(s))
            if b < 0:
                continue
            t0 = cu[b] + s.value * seg
            times[max(t0, 0):min(t0 + seg, cu[b + 1])] += 1
            assert s.value >= 0 and (t0 < cu[b + 1] or lens[b] == 0)
            empty[b] += lens[b] == 0
        assert (times[cu[0]:cu[-1]] == 1).all() and not times[:cu[0]].any() and not times[cu[-1]:].any()
        assert (empty[np.array(lens) == 0] == 1).all()
