"""gated_delta_prefill with a value that is not finite. The recurrence in 64 bits says what it reaches. In the operator
it may also reach tokens before it in its own 64 (of its value column, or of the heads that read it): they are not
finite then. What is finite is right, and nothing else is touched: earlier chunks, other sequences, other heads,
for v and the state other value columns. (Tolerances: test_gpu_delta.py.)
"""
import numpy as np
import pytest
import torch

from test_gpu_delta import ATOL, gpu, make, prefill, recurrence

pytestmark = pytest.mark.gpu

# sequences' lengths, heads and dimensions: 16, 32 and 64 value columns to a workgroup
SHAPES = [([150, 20], 1, 2, 128, 64), ([150, 20, 70], 16, 64, 64, 64), ([150, 20, 70, 1, 9], 16, 64, 128, 64)]
AT, HEAD, COLUMN = 100, 1, 21       # a token of the first sequence's second chunk
POISON = [("v", "inf"), ("v", "nan"), ("k", "inf"), ("k", "nan"), ("q", "inf"), ("q", "nan"), ("g", "nan"), ("beta", "inf"),
          ("beta", "nan"), ("state", "inf"), ("state", "nan")]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=["16", "32", "64"])
@pytest.mark.parametrize("name,value", POISON)
def test_not_finite(name, value, shape, dtype):
    lens, Hk, Hv, Dk, Dv = shape
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=7)
    rep, value = Hv // Hk, float(value)
    mine = torch.zeros(sum(lens), Hv, Dv, dtype=torch.bool)            # outputs that it may reach
    state = torch.zeros(len(lens), Hv, Dv, Dk, dtype=torch.bool)
    heads = slice(0, rep) if name in ("q", "k") else slice(HEAD, HEAD + 1)
    columns = slice(COLUMN, COLUMN + 1) if name in ("v", "state") else slice(None)
    chunk = slice(0 if name == "state" else 64, lens[0])
    if name == "q":
        x["q"][AT, 0, 5] = value
        mine[AT, heads] = True
    else:
        if name == "v":
            x["v"][AT, HEAD, COLUMN] = value
        elif name == "k":
            x["k"][AT, 0, 5] = value
        elif name == "state":
            x["state"][0, HEAD, COLUMN, 5] = value
        else:
            x[name][AT, HEAD] = value
        mine[chunk, heads, columns] = True
        state[0, heads, columns] = True
    ref, ref_state = recurrence(x, lens, True)
    d = gpu(x)
    out = prefill(d, lens, l2norm=True).cpu()
    for got, want, reached, dims, half in ((out, ref, mine, (0, 2), torch.finfo(dtype).eps / 2),
                                           (d["state"].cpu(), ref_state, state, (-1, -2), 0.0)):
        finite = torch.isfinite(got)
        assert (finite | reached).all()
        assert torch.isfinite(want)[finite].all()
        got, want = got.double(), want.where(torch.isfinite(want), torch.zeros_like(want))
        top = want.abs().amax(dims, keepdim=True).clamp_min(1e-3)
        bad = finite & ((got - want).abs() > half * want.abs() * (1 + 2.0 ** -7) + ATOL * top + 2.0 ** -25)
        assert not bad.any(), int(bad.sum())
