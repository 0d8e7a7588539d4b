"""Packed sequences that do not begin at row 0 (cu_seqlens[0] > 0): other rows lie before and behind them, which no operator reads
or writes. The convolution, the selective scan and the gated delta rule, with few and many sequences, against their formulas
in 64 bits with the tolerances of their own tests."""
import pytest
import torch

import layer_math as lm
import test_gpu_conv as conv
import test_gpu_delta as delta
import test_gpu_scan as scan
from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BEHIND = 70


def lengths(n, first_empty):
    gen = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 4, (n,), generator=gen).tolist()
    lens[n // 2], lens[n - 1], lens[1] = 900, 300, 70
    lens[0] = 0 if first_empty else 3
    return lens


def between(t, before):
    """t's rows between rows of NaN, which show in every result that they enter."""
    fill = lambda k: torch.full((k, *t.shape[1:]), float("nan"), dtype=t.dtype)
    return torch.cat([fill(before), t, fill(BEHIND)]).to(DEV)


def places(n, seed):
    """Slots of a pool with one more, in any order."""
    return torch.randperm(n + 1, generator=torch.Generator().manual_seed(seed))[:n]


cases = [pytest.mark.parametrize("before", [1, 1030, 4096]), pytest.mark.parametrize("first_empty", [False, True]),
         pytest.mark.parametrize("n", [5, 512, 513, 700])]


def each(f):
    for c in cases:
        f = c(f)
    return f


def run(op, names, x, lens, before, slots, out_like):
    rows = {k: between(x[k], before) for k in names}
    cu = (torch.tensor([0] + lens).cumsum(0) + before).int().to(DEV)
    into = torch.full((before + sum(lens) + BEHIND, *out_like.shape[1:]), 5.0, dtype=out_like.dtype, device=DEV)
    so = torch.full_like(x["state"], 7.0).to(DEV)
    op(rows, cu, slots.int().to(DEV), into, so)
    rest = [i for i in range(len(lens) + 1) if i not in set(slots.tolist())]
    assert (into[:before] == 5).all() and (into[before + sum(lens):] == 5).all() and (so[rest] == 7).all()
    return into[before:before + sum(lens)], so[slots.to(DEV)]


@each
def test_convolution(n, first_empty, before):
    lens, slots = lengths(n, first_empty), places(n, 1)
    x = conv.make(lens, 24, 4, torch.float16, pool=n + 1)
    ref, mag, state = lm.conv(x["x"], x["weight"], x["bias"], x["state"], lens, slots.tolist())
    g = conv.gpu(x)
    out, so = run(lambda r, cu, s, o, so: ops.causal_conv_prefill(r["x"], g["weight"], g["bias"], g["state"], cu_seqlens=cu, slots=s,
                                                                  out=o, state_out=so), ["x"], x, lens, before, slots, x["x"])
    conv.check(out, ref, mag, True, "out")
    assert torch.equal(so.cpu(), state[slots])


@each
def test_scan(n, first_empty, before):
    lens, slots = lengths(n, first_empty), places(n, 2)
    x = scan.make(lens, 2, 1, 32, 64, torch.bfloat16, pool=n + 1)
    y, mag, s, smag = scan.reference(x, lens, slots.tolist())
    g = scan.gpu(x)
    out, so = run(lambda r, cu, sl, o, so: ops.selective_scan_prefill(r["x"], r["dt"], g["A_log"], r["B"], r["C"], g["state"], D=g["D"],
                                                                      dt_bias=g["dt_bias"], cu_seqlens=cu, slots=sl, out=o, state_out=so),
                  ["x", "dt", "B", "C"], x, lens, before, slots, x["x"])
    scan.check(out, so, (y, mag, s[slots], smag[slots]))


@each
def test_delta_rule(n, first_empty, before):
    lens, slots = lengths(n, first_empty), places(n, 3)
    x = delta.make(lens, 1, 2, 64, 32, torch.float16, pool=n + 1)
    ref, state = delta.recurrence(x, lens, True, slots.tolist())
    g = delta.gpu(x)
    out, so = run(lambda r, cu, s, o, so: ops.gated_delta_prefill(r["q"], r["k"], r["v"], r["g"], r["beta"], g["state"], cu_seqlens=cu,
                                                                  slots=s, l2norm=True, out=o, state_out=so),
                  ["q", "k", "v", "g", "beta"], x, lens, before, slots, x["v"])
    delta.check(out, ref, "out")
    delta.check(so, state[slots], "state")


@pytest.mark.parametrize("offsets", [[3000, 0], [0, 3000], [2999, 64, 1 << 30, -5]])
def test_falling_offsets_of_many_sequences_stay_inside(offsets):
    """Results are not specified, but nothing outside the tensors is written (more than 512 sequences)."""
    T, n, H, P, N = 3000, 600, 4, 32, 64
    x = scan.gpu(scan.make([T], H, 1, P, N, torch.float16, pool=n))
    around = torch.full((3 * T, H, P), 5.0, dtype=torch.float16, device=DEV)
    states = torch.full((3 * n, H, P, N), 7.0, device=DEV)
    states[n:2 * n] = x["state"]
    cu = torch.tensor((offsets * n)[:n + 1], dtype=torch.int32, device=DEV)
    ops.selective_scan_prefill(x["x"], x["dt"], x["A_log"], x["B"], x["C"], states[n:2 * n], D=x["D"], dt_bias=x["dt_bias"],
                               cu_seqlens=cu, out=around[T:2 * T])
    torch.cuda.synchronize()
    assert (around[:T] == 5).all() and (around[2 * T:] == 5).all() and (states[:n] == 7).all() and (states[2 * n:] == 7).all()
