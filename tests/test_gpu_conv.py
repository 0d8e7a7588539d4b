"""The short causal convolution (ops.causal_conv_step, ops.causal_conv_prefill) against its formula in 64 bits.

Tolerance: a sum of at most W + 1 = 5 terms in fp32 is off by at most 5 roundings of 2^-24 of the terms' magnitudes, and
SiLU's slope is at most 1.1; SiLU itself is off by (1 + |y|) 2^-22 of its result (twice what its comment states). Outputs
are rounded to their type on top: half a step. States are copies."""
import pytest
import torch

import layer_math as lm
from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(lens, C, W, dtype, seed=0, pool=None):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    return {"x": r(sum(lens), C).to(dtype), "weight": (0.5 * r(C, W)).to(dtype), "bias": (0.2 * r(C)).to(dtype),
            "state": r(pool or len(lens), C, W - 1).to(dtype)}


def gpu(x):
    return {n: t.to(DEV) for n, t in x.items()}


def check(got, ref, mag, act, what):
    got = got.cpu()
    assert torch.isfinite(got.double()).all(), what
    rel, tiny = lm.half_step(got.dtype)
    y = mag  # (bounds |y|)
    tol = 1.1 * 5 * 2.0 ** -24 * mag + (rel * (1 + 2.0 ** -7) + ((1 + y) * 2.0 ** -22 if act else 0.0)) * ref.abs() + tiny
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} values off"


LENS = [[1], [2], [15, 16, 17, 0, 1, 3, 2, 33], [0, 0, 5, 0], [100], [1] * 70, [0]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("C", [1, 7, 8, 130, 520])
def test_prefill(C, lens, W, dtype):
    x = make(lens, C, W, dtype)
    ref, mag, state = lm.conv(x["x"], x["weight"], x["bias"], x["state"], lens)
    g = gpu(x)
    so = torch.full_like(g["state"], 7.0)
    out = ops.causal_conv_prefill(g["x"], g["weight"], g["bias"], g["state"], cu_seqlens=lm.offsets(lens, DEV), state_out=so)
    check(out, ref, mag, True, "out")
    assert torch.equal(so.cpu(), state) and torch.equal(g["state"].cpu(), x["state"])
    out2 = ops.causal_conv_prefill(g["x"], g["weight"], g["bias"], g["state"], cu_seqlens=lm.offsets(lens, DEV))
    assert torch.equal(out, out2) and torch.equal(g["state"].cpu(), state)      # in place


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("B,C", [(1, 4352), (3, 5), (33, 512), (65, 24), (5, 1027)])
def test_step(B, C, W, dtype):
    x = make([1] * B, C, W, dtype, pool=B + 3)
    slots = torch.randperm(B + 3, generator=torch.Generator().manual_seed(1))[:B].int()
    for act, bias in ((True, x["bias"]), (False, None)):
        ref, mag, state = lm.conv(x["x"], x["weight"], bias, x["state"], [1] * B, slots.tolist(), act)
        g = gpu(x)
        out = ops.causal_conv_step(g["x"], g["weight"], None if bias is None else g["bias"], g["state"],
                                   slots=slots.to(DEV), silu=act)
        check(out, ref, mag, act, "out")
        assert torch.equal(g["state"].cpu(), state)
        g2 = gpu(x)
        ops.causal_conv_step(g2["x"], g2["weight"], None if bias is None else g2["bias"], g2["state"], slots=slots.to(DEV),
                             silu=act, out=g2["x"])
        assert torch.equal(g2["x"], out) and torch.equal(g2["state"].cpu(), state)


@pytest.mark.parametrize("C,W,dtype", [(264, 4, torch.float16), (33, 3, torch.bfloat16), (72, 2, torch.float16)])
def test_tokens_parts_and_batches_agree(C, W, dtype):
    """Prompts in one call, cut anywhere, token by token and as a padless batch: the same bits."""
    B, T = 3, 41
    x = make([T] * B, C, W, dtype)
    g = gpu(x)
    s = [g["state"].clone() for _ in range(4)]
    one = ops.causal_conv_prefill(g["x"], g["weight"], g["bias"], s[0], cu_seqlens=lm.offsets([T] * B, DEV))
    batch = ops.causal_conv_prefill(g["x"].view(B, T, C), g["weight"], g["bias"], s[1])
    parts, steps, at = torch.empty_like(one).view(B, T, C), torch.empty_like(one).view(B, T, C), 0
    for n in (1, 2, 17, 20, 1):
        parts[:, at:at + n] = ops.causal_conv_prefill(g["x"].view(B, T, C)[:, at:at + n], g["weight"], g["bias"], s[2])
        at += n
    for t in range(T):
        steps[:, t] = ops.causal_conv_step(g["x"].view(B, T, C)[:, t], g["weight"], g["bias"], s[3])
    for y in (batch, parts, steps):
        assert torch.equal(y.view(-1, C), one)
    for y in s[1:]:
        assert torch.equal(y, s[0])


@pytest.mark.parametrize("C", [8, 24, 37])
def test_strided_rows(C):
    """Columns of a wider row in and out, at odd addresses too; what lies beside them stays."""
    lens, W = [5, 0, 40], 4
    x = make(lens, C, W, torch.float16)
    ref, mag, state = lm.conv(x["x"], x["weight"], x["bias"], x["state"], lens)
    g = gpu(x)
    for before in (0, 3, 8):
        wide = torch.full((45, C + 13), 3.0, dtype=torch.float16, device=DEV)
        wide[:, before:before + C] = g["x"]
        into = torch.full((45, C + 11), 5.0, dtype=torch.float16, device=DEV)
        s = g["state"].clone()
        out = ops.causal_conv_prefill(wide[:, before:before + C], g["weight"], g["bias"], s,
                                      cu_seqlens=lm.offsets(lens, DEV), out=into[:, before:before + C])
        check(out, ref, mag, True, "out")
        assert (into[:, :before] == 5).all() and (into[:, before + C:] == 5).all() and torch.equal(s.cpu(), state)
    column = ops.causal_conv_prefill(g["x"].t().contiguous().t(), g["weight"], g["bias"], g["state"].clone(),
                                     cu_seqlens=lm.offsets(lens, DEV))       # channels not contiguous: copied
    check(column, ref, mag, True, "out")


def test_padding_bad_slots_and_rows_of_no_sequence():
    lens, C, W = [20, 18, 3, 0, 17], 40, 4
    x = make(lens, C, W, torch.bfloat16, pool=4)
    slots = [2, -1, 2, 9, 0]                          # the third has the first one's, the fourth is past the state
    g = gpu(x)
    rows = torch.cat([g["x"], g["x"][:6]])            # six rows behind the last sequence
    into = torch.full_like(rows, 5.0)
    so = torch.full_like(g["state"], 7.0)
    ops.causal_conv_prefill(rows, g["weight"], g["bias"], g["state"], cu_seqlens=lm.offsets(lens, DEV),
                            slots=torch.tensor(slots, dtype=torch.int32, device=DEV), out=into, state_out=so)
    good = [20, 17]
    xs = torch.cat([x["x"][:20], x["x"][41:58]])
    ref, mag, state = lm.conv(xs, x["weight"], x["bias"], x["state"], good, [2, 0])
    check(torch.cat([into[:20], into[41:58]]), ref, mag, True, "out")
    assert (into[20:38] == 0).all() and into[38:41].isnan().all() and (into[58:] == 5).all()
    assert torch.equal(so[[0, 2]].cpu(), state[[0, 2]]) and (so[[1, 3]] == 7).all()
    so.fill_(7.0)
    step = ops.causal_conv_step(g["x"][:5], g["weight"], g["bias"], g["state"],
                                slots=torch.tensor(slots, dtype=torch.int32, device=DEV), state_out=so)
    assert (step[1] == 0).all() and step[2:4].isnan().all() and step[[0, 4]].isfinite().all() and (so[[1, 3]] == 7).all()


def test_values_that_are_not_finite_stay_in_their_window():
    lens, C = [40, 40], 16
    x = make(lens, C, 4, torch.float16)
    x["x"][50, 3], x["x"][39, 5], x["state"][1, 7, 2] = float("nan"), float("inf"), float("nan")
    g = gpu(x)
    out = ops.causal_conv_prefill(g["x"], g["weight"], g["bias"], g["state"], cu_seqlens=lm.offsets(lens, DEV))
    bad = torch.zeros(80, C, dtype=torch.bool)
    bad[50:54, 3] = True
    bad[40:43, 7] = True
    bad[39, 5] = True
    assert torch.equal(out.cpu()[:, [3, 7]].isnan(), bad[:, [3, 7]])
    assert out.cpu()[~bad].isfinite().all()


def test_rows_past_32_bits():
    C, W, T = 8192, 4, (1 << 18) + 40
    x = torch.zeros(T, C, dtype=torch.float16, device=DEV)
    tail = make([40], C, W, torch.float16)
    x[-40:] = tail["x"].to(DEV)
    g = gpu(tail)
    state = torch.zeros(2, C, W - 1, dtype=torch.float16, device=DEV)
    state[1] = g["state"][0]
    cu = torch.tensor([0, T - 40, T], dtype=torch.int32, device=DEV)
    out = ops.causal_conv_prefill(x, g["weight"], g["bias"], state, cu_seqlens=cu)
    ref, mag, after = lm.conv(tail["x"], tail["weight"], tail["bias"], tail["state"], [40])
    check(out[-40:], ref, mag, True, "out")
    assert torch.equal(state[1].cpu(), after[0])


@pytest.mark.parametrize("offsets", [[0, 300, 0, 300], [-5, 400, 1 << 30, 7], [300, 200, 100, 0]])
def test_bad_offsets_stay_inside(offsets):
    T, C = 300, 40
    x = gpu(make([T], C, 4, torch.float16, pool=3))
    around = torch.full((3 * T, C), 5.0, dtype=torch.float16, device=DEV)
    states = torch.full((9, C, 3), 7.0, dtype=torch.float16, device=DEV)
    ops.causal_conv_prefill(x["x"], x["weight"], x["bias"], states[3:6], out=around[T:2 * T],
                            cu_seqlens=torch.tensor(offsets, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert (around[:T] == 5).all() and (around[2 * T:] == 5).all() and (states[:3] == 7).all() and (states[6:] == 7).all()
