"""gated_delta_prefill at each of the chain's widths (16, 32 and 64 value columns to a workgroup, by the number of heads) and
each key dimension and type, against the recurrence in 64 bits: ragged batches with empty sequences, decays of any size,
slots, strides. (Tolerances: test_gpu_delta.py. Which shape has which width: test_delta_plan.py.)
"""
import numpy as np
import pytest
import torch

from dfssm import ops
from test_gpu_delta import DEV, check, gpu, make, prefill, recurrence

pytestmark = pytest.mark.gpu

# tiles of 16 value columns to a workgroup; sequences' lengths, key and value heads, value columns (5 tiles leave a part of
# a workgroup's waves idle)
SHAPES = [(1, ([130, 0, 5, 64, 1], 1, 2, 80)), (2, ([129, 0, 65], 16, 64, 64)), (2, ([64, 1, 0], 64, 64, 48)),
          (4, ([150, 0, 63, 17, 64], 16, 64, 64)), (4, ([1, 129, 0, 16, 70], 8, 64, 80)), (4, ([200, 70, 0, 3, 65], 1, 64, 256))]


@pytest.fixture(params=SHAPES, ids=lambda s: f"{s[0]}-{s[1][3]}")
def shape(request):
    return request.param[1]


def steps(x, lens, *args, **kw):
    """The recurrence, its tensors on the GPU."""
    out, state = recurrence(gpu(x), lens, *args, **kw)
    return out, state.cpu()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Dk", [64, 128])
def test_ragged(shape, Dk, dtype):
    lens, Hk, Hv, Dv = shape
    for l2norm in (True, False):
        x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=Dk + sum(lens), l2norm=l2norm)
        ref, ref_state = steps(x, lens, l2norm)
        d = gpu(x)
        check(prefill(d, lens, l2norm=l2norm), ref, "out")
        check(d["state"], ref_state, "state")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Dk", [64, 128])
def test_extremes(shape, Dk, dtype):
    """-inf decays (first, last and in the middle of a chunk), long decays, beta 0 and 1, zero keys and queries, a state
    far larger than the values."""
    lens, Hk, Hv, Dv = shape
    T = sum(lens)
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=Dv + sum(lens))
    x["state"] *= 100.0
    x["g"][0, 0] = float("-inf")
    x["g"][T // 2, 1::3] = float("-inf")
    x["g"][T - 1, 0] = -300.0
    x["g"][:, 1::4] -= 20.0
    x["beta"][::3] = 0.0
    x["beta"][1::3] = 1.0
    x["k"][T // 3] = 0.0
    x["q"][T // 4] = 0.0
    ref, ref_state = steps(x, lens, True)
    d = gpu(x)
    check(prefill(d, lens, l2norm=True), ref, "out")
    check(d["state"], ref_state, "state")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Dk", [64, 128])
def test_slots_and_strides(shape, Dk, dtype):
    """Sequences in a larger pool, one of them padding, one past its end and one in a slot that is taken; q, k and v as
    parts of packed rows with NaN behind the last sequence, out in a wider buffer of which nothing else is written."""
    lens, Hk, Hv, Dv = shape
    n, T = len(lens), sum(lens)
    slots = [4, -1, 9, 4, 0][:n] if lens[1] else [4, 0, 4, -1, 9][:n]
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=3, pool=7)
    first = np.concatenate([[0], np.cumsum(lens)])
    keep = [b for b in range(n) if 0 <= slots[b] < 7 and slots[b] not in slots[:b]]
    ref_state = x["state"].double().clone()
    ref = torch.zeros(T, Hv, Dv, dtype=torch.float64)
    for b in keep:
        one = {m: (t if m == "state" else t[first[b]:first[b + 1]]) for m, t in x.items()}
        ref[first[b]:first[b + 1]], state = steps(one, [lens[b]], True, slots=[slots[b]])
        ref_state[slots[b]] = state[slots[b]]
    d = gpu(x)
    wide = torch.cat([d[m].flatten(1) for m in ("q", "k", "v")] + [torch.zeros(T, 8, device=DEV, dtype=dtype)], 1)
    wide = torch.cat([wide, torch.full((70, wide.shape[1]), float("nan"), device=DEV, dtype=dtype)])
    q, k, v = (t.view(T + 70, -1, w) for t, w in zip(wide.split([Hk * Dk, Hk * Dk, Hv * Dv, 8], 1), (Dk, Dk, Dv)))
    gb = torch.full((T + 70, 2 * Hv + 3), float("nan"), device=DEV)
    gb[:T, :Hv], gb[:T, Hv:2 * Hv] = d["g"], d["beta"]
    buffer = torch.full((T + 70, Hv * Dv + 16), 5.0, device=DEV, dtype=dtype)
    out = buffer[:, 8:8 + Hv * Dv].view(T + 70, Hv, Dv)
    so = torch.full_like(d["state"], 7.0)
    cu = torch.tensor(first, dtype=torch.int32, device=DEV)
    ops.gated_delta_prefill(q, k, v, gb[:, :Hv], gb[:, Hv:2 * Hv], d["state"], cu_seqlens=cu, l2norm=True, out=out,
                            slots=torch.tensor(slots, dtype=torch.int32, device=DEV), state_out=so)
    assert torch.equal(d["state"].cpu(), x["state"])
    assert (buffer[T:] == 5).all() and (buffer[:, :8] == 5).all() and (buffer[:, 8 + Hv * Dv:] == 5).all()
    for b in range(n):
        got = out[first[b]:first[b + 1]].contiguous()
        if b in keep:
            if lens[b]:
                check(got, ref[first[b]:first[b + 1]], f"out {b}")
        else:
            assert (got == 0).all() if slots[b] < 0 else torch.isnan(got).all()
    touched = [slots[b] for b in keep]
    check(so[touched], ref_state[touched], "state_out")
    assert (so[[i for i in range(7) if i not in touched]] == 7).all()
