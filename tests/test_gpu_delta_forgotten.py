"""Large values beside small ones in one chunk, forgotten in between (a decay of -inf): what comes after them is as exact as
without them, up to 2^-32 of the largest value.

Where that comes from: a chunk's v - S' k and its u are pairs of halves with one scale per value column, so one of a size
below 2^-17 of the column's largest, M, is off by up to 2^-39 M. A state or output sums at most 64 of them, with
factors whose sum stays below 64 (keys of norm 1, beta below 1), and M is at most twice the largest value: 2^-39 2 64.
On top what test_gpu_delta.py allows, of the small values' own size.
"""
import pytest
import torch

from test_gpu_delta import ATOL, gpu, make, prefill, recurrence

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,ratio", [(torch.float16, 10), (torch.float16, 20), (torch.bfloat16, 10), (torch.bfloat16, 20)])
@pytest.mark.parametrize("shape", [([64], 1, 2, 128, 64), ([50, 64, 64], 16, 64, 64, 64), ([60] * 5, 16, 64, 128, 64)],
                         ids=["16", "32", "64"])
def test_forgotten(shape, dtype, ratio):
    lens, Hk, Hv, Dk, Dv = shape
    big = 4                                                            # tokens of each sequence, then the decay
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=ratio)
    first = [sum(lens[:b]) for b in range(len(lens))]
    small = torch.ones(sum(lens), dtype=torch.bool)
    v = x["v"].float() * 2.0 ** (8 - ratio)
    for t in first:
        v[t:t + big] *= 2.0 ** ratio
        x["g"][t + big] = float("-inf")
        small[t:t + big] = False
    x["v"] = v.to(dtype)
    x["state"] *= 2.0 ** 8
    ref, ref_state = recurrence(gpu(x), lens, True)
    ref_state = ref_state.cpu()
    d = gpu(x)
    out = prefill(d, lens, l2norm=True).cpu()
    most = float(x["v"].float().abs().max())
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0               # half a step of the subnormal halves
    for got, want, dims, half in ((out[small], ref[small], (0, 2), torch.finfo(dtype).eps / 2),
                                  (d["state"].cpu(), ref_state, (-1, -2), 0.0)):
        assert torch.isfinite(got).all()
        err, top = (got.double() - want).abs(), want.abs().amax(dims, keepdim=True)
        bad = err > half * want.abs() * (1 + 2.0 ** -7) + ATOL * top + 2.0 ** -32 * most + tiny
        assert not bad.any(), (int(bad.sum()), float(err.max()))
