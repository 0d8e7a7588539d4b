"""The selective state space scan (ops.selective_scan_step, ops.selective_scan_prefill) against its recurrence in 64 bits.

Tolerance. Relative to the sums over magnitudes (layer_math.scan): a state is off by the roundings of d (8 of 2^-24), of
each decay (an exponent t off by 2^-22 t, and t e^-t < 0.4), of factors in parts (at worst 22 bits) and of the sums over
64 tokens: below 64 roundings, 2^-18. An output has its factors in two parts of 8 bits, each off by 2^-17, on two ways,
and the state's error: below 2^-16, and half a step of its type."""
import pytest
import torch

import layer_math as lm
from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(lens, H, G, P, N, dtype, seed=0, pool=None, dt32=False):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    T = sum(lens)
    return {"x": r(T, H, P).to(dtype), "dt": r(T, H).to(torch.float32 if dt32 else dtype),
            "A_log": torch.log(1 + 15 * torch.rand(H, generator=gen)), "B": r(T, G, N).to(dtype), "C": r(T, G, N).to(dtype),
            "D": 1 + 0.2 * r(H), "dt_bias": 4 * torch.rand(H, generator=gen) - 5,
            "state": 0.3 * r(pool or len(lens), H, P, N)}


def gpu(x):
    return {n: t.to(DEV) for n, t in x.items()}


def reference(x, lens, slots=None, **kw):
    return lm.scan(x["x"], x["dt"], x["A_log"], x["B"], x["C"], x["state"], x["D"], x["dt_bias"], lens, slots, **kw)


def check(out, state, ref, what=""):
    y, ymag, s, smag = ref
    out, state = out.cpu(), state.cpu()
    assert torch.isfinite(out.double()).all() and torch.isfinite(state).all(), what
    rel, tiny = lm.half_step(out.dtype)
    bad = (out.double() - y).abs() > rel * (1 + 2.0 ** -7) * y.abs() + 2.0 ** -16 * ymag + tiny
    assert not bad.any(), f"{what} out: {int(bad.sum())} off, worst {float(((out.double() - y).abs() / (ymag + 1e-30)).max()):.3g}"
    bad = (state.double() - s).abs() > 2.0 ** -18 * smag + 1e-37
    assert not bad.any(), f"{what} state: {int(bad.sum())} off, worst {float(((state.double() - s).abs() / (smag + 1e-30)).max()):.3g}"


def prefill(g, lens, **kw):
    return ops.selective_scan_prefill(g["x"], g["dt"], g["A_log"], g["B"], g["C"], kw.pop("state", g["state"]), D=g["D"],
                                      dt_bias=g["dt_bias"], cu_seqlens=lm.offsets(lens, DEV), **kw)


STEP = [(1, 64, 1, 64, 128), (3, 6, 2, 208, 64), (33, 8, 8, 32, 128), (64, 4, 1, 16, 64), (2, 3, 3, 256, 128), (40, 64, 8, 64, 128)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,G,P,N", STEP)
def test_step(B, H, G, P, N, dtype):
    x = make([1] * B, H, G, P, N, dtype, pool=B + 2, dt32=B % 2 == 0)
    slots = torch.randperm(B + 2, generator=torch.Generator().manual_seed(1))[:B].int()
    ref = reference(x, [1] * B, slots.tolist())
    g = gpu(x)
    so = torch.full_like(g["state"], 7.0)
    out = ops.selective_scan_step(g["x"], g["dt"], g["A_log"], g["B"], g["C"], g["state"], D=g["D"], dt_bias=g["dt_bias"],
                                  slots=slots.to(DEV), state_out=so)
    mine = slots.long()
    check(out, so[mine.to(DEV)], (ref[0], ref[1], ref[2][mine], ref[3][mine]))
    rest = [i for i in range(B + 2) if i not in slots.tolist()]
    assert (so[rest] == 7).all() and torch.equal(g["state"].cpu(), x["state"])
    ops.selective_scan_step(g["x"], g["dt"], g["A_log"], g["B"], g["C"], g["state"], D=g["D"], dt_bias=g["dt_bias"],
                            slots=slots.to(DEV))
    assert torch.equal(g["state"][mine.to(DEV)], so[mine.to(DEV)])


SHAPES = [([1], 2, 1, 64, 128), ([45], 8, 1, 64, 128), ([64], 4, 2, 32, 64), ([65, 0, 1, 63, 128, 200], 6, 3, 64, 128),
          ([130, 17], 3, 1, 48, 64), ([300], 5, 5, 208, 64), ([700, 3], 2, 1, 16, 128), ([90, 70], 4, 1, 256, 128),
          ([0, 0, 77, 0], 8, 8, 80, 64), ([40] * 20, 21, 3, 64, 64), ([0], 2, 1, 64, 128), ([1500], 3, 3, 32, 128)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,H,G,P,N", SHAPES, ids=lambda v: str(v)[:14])
def test_prefill(lens, H, G, P, N, dtype):
    x = make(lens, H, G, P, N, dtype, dt32=len(lens) % 2 == 0)
    ref = reference(x, lens)
    g = gpu(x)
    so = torch.full_like(g["state"], 7.0)
    out = prefill(g, lens, state_out=so)
    check(out, so, ref)
    assert torch.equal(g["state"].cpu(), x["state"])
    out2 = prefill(g, lens)
    assert torch.equal(out2, out) and torch.equal(g["state"], so)               # in place


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_without_d_bias_or_softplus(dtype):
    lens = [70, 9]
    x = make(lens, 4, 2, 64, 64, dtype)
    x["dt"] = (0.2 * x["dt"]).to(dtype)                                         # half of them negative: no time passes
    g = gpu(x)
    for D, b, soft in ((None, None, False), (x["D"], None, True), (None, x["dt_bias"], True)):
        ref = lm.scan(x["x"], x["dt"], x["A_log"], x["B"], x["C"], x["state"], D, b, lens, softplus=soft)
        s = g["state"].clone()
        out = ops.selective_scan_prefill(g["x"], g["dt"], g["A_log"], g["B"], g["C"], s, D=None if D is None else g["D"],
                                         dt_bias=None if b is None else g["dt_bias"], cu_seqlens=lm.offsets(lens, DEV),
                                         softplus=soft)
        check(out, s, ref)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parts_batches_and_steps_agree(dtype):
    """Prompts in one call, in parts and token by token, within each form's rounding."""
    B, T, H, G, P, N = 2, 150, 4, 1, 64, 128
    x = make([T] * B, H, G, P, N, dtype)
    ref = reference(x, [T] * B)
    g = gpu(x)
    v = {n: g[n].view(B, T, *g[n].shape[1:]) for n in ("x", "dt", "B", "C")}
    part = lambda a, b: {n: t[:, a:b] for n, t in v.items()}
    for cuts in ([150], [1, 12, 64, 73], [77, 73], [1] * 150):
        s, at, out = g["state"].clone(), 0, torch.empty_like(v["x"])
        for n in cuts:
            p = part(at, at + n)
            if len(cuts) == T:
                out[:, at] = ops.selective_scan_step(p["x"][:, 0], p["dt"][:, 0], g["A_log"], p["B"][:, 0], p["C"][:, 0], s,
                                                     D=g["D"], dt_bias=g["dt_bias"])
            else:
                out[:, at:at + n] = ops.selective_scan_prefill(p["x"], p["dt"], g["A_log"], p["B"], p["C"], s, D=g["D"],
                                                               dt_bias=g["dt_bias"])
            at += n
        check(out.view(B * T, H, P), s, ref, str(cuts[:4]))


def test_strided_rows():
    """x, B and C as columns of one row, as the convolution leaves them; out as columns of a wider one."""
    lens, H, G, P, N = [33, 90], 4, 1, 64, 128
    x = make(lens, H, G, P, N, torch.float16)
    ref = reference(x, lens)
    g = gpu(x)
    row = torch.cat([g["x"].flatten(1), g["B"].flatten(1), g["C"].flatten(1)], 1)
    wide = torch.full((123, H * P + 16), 5.0, dtype=torch.float16, device=DEV)
    s = g["state"].clone()
    a, b = H * P, H * P + G * N
    out = ops.selective_scan_prefill(row[:, :a].unflatten(1, (H, P)), g["dt"], g["A_log"], row[:, a:b].unflatten(1, (G, N)),
                                     row[:, b:].unflatten(1, (G, N)), s, D=g["D"], dt_bias=g["dt_bias"],
                                     cu_seqlens=lm.offsets(lens, DEV), out=wide[:, 8:8 + a].unflatten(1, (H, P)))
    check(out, s, ref)
    assert (wide[:, :8] == 5).all() and (wide[:, 8 + a:] == 5).all()


@pytest.mark.parametrize("n", [3, 80])
def test_padding_bad_slots_and_rows_of_no_sequence(n):
    lens = [n, 2 * n, 5, 0, n + 1]
    x = make(lens, 4, 2, 64, 128, torch.bfloat16, pool=4)
    slots = [2, -1, 2, 9, 0]
    g = gpu(x)
    T, off = sum(lens), lm.offsets(lens).tolist()
    for k in ("x", "dt", "B", "C"):
        g[k] = torch.cat([g[k], torch.full_like(g[k][:7], float("nan"))])       # rows behind the last sequence
    into = torch.full_like(g["x"], 5.0)
    so = torch.full_like(g["state"], 7.0)
    prefill(g, lens, slots=torch.tensor(slots, dtype=torch.int32, device=DEV), out=into, state_out=so)
    keep = torch.cat([torch.arange(off[0], off[1]), torch.arange(off[4], off[5])])
    y = dict(x, **{k: x[k][keep] for k in ("x", "dt", "B", "C")})
    ref = reference(y, [lens[0], lens[4]], [2, 0])
    check(into[:T][keep.to(DEV)], so[[0, 2]], (ref[0], ref[1], ref[2][[0, 2]], ref[3][[0, 2]]))
    assert (into[off[1]:off[2]] == 0).all() and into[off[2]:off[3]].isnan().all() and (into[T:] == 5).all()
    assert (so[[1, 3]] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decays_of_any_size(dtype):
    """Tokens that wipe the state beside tokens that hardly move it: differences of the decays' sums keep their digits."""
    lens = [256]
    x = make(lens, 4, 1, 64, 128, dtype, dt32=True)
    x["dt"][::7] = 900.0
    x["dt"][3::11] = -20.0
    x["x"][::7] *= 2.0 ** -9                                                    # (d x in range)
    ref = reference(x, lens)
    g = gpu(x)
    check(prefill(g, lens), g["state"], ref)


def test_repeats_are_equal():
    lens = [500, 64, 1000, 3]
    g = gpu(make(lens, 16, 2, 64, 128, torch.float16))
    first = None
    for _ in range(3):
        s = g["state"].clone()
        out = prefill(g, lens, state=s)
        first = first or (out, s)
        assert torch.equal(out, first[0]) and torch.equal(s, first[1])


@pytest.mark.parametrize("n", [63, 64, 65, 511, 512, 513, 700])
def test_many_sequences(n):
    """Both numberings of the segments (counted up to 512 sequences), with empty and long ones among them."""
    gen = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 4, (n,), generator=gen).tolist()
    lens[n // 2], lens[n - 1], lens[1] = 900, 300, 70
    x = make(lens, 2, 1, 32, 64, torch.bfloat16)
    ref = reference(x, lens)
    g = gpu(x)
    check(prefill(g, lens), g["state"], ref)


@pytest.mark.parametrize("offsets", [[0, 3000, 0, 3000, 0, 3000], [-5, 4000, 1 << 30, 0, 64, 63], [3000, 2000, 1000, 0, 0, 0]])
def test_bad_offsets_stay_inside(offsets):
    """Offsets that fall or lie outside: results are not specified, but nothing outside the tensors is written."""
    T, H, P, N = 3000, 4, 32, 64
    x = gpu(make([T], H, 1, P, N, torch.float16, pool=8))
    around = torch.full((3 * T, H, P), 5.0, dtype=torch.float16, device=DEV)
    states = torch.full((24, H, P, N), 7.0, device=DEV)
    states[8:16] = x["state"]
    cu = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    for _ in range(2):
        ops.selective_scan_prefill(x["x"], x["dt"], x["A_log"], x["B"], x["C"], states[8:16], D=x["D"], dt_bias=x["dt_bias"],
                                   cu_seqlens=cu, out=around[T:2 * T])
    torch.cuda.synchronize()
    assert (around[:T] == 5).all() and (around[2 * T:] == 5).all() and (states[:8] == 7).all() and (states[16:] == 7).all()


def test_states_past_32_bits():
    H, P, N = 64, 64, 128
    pool = 4200                                                                 # 2.2 * 10^9 values
    state = torch.zeros(pool, H, P, N, device=DEV)
    for lens in ([70], [5]):
        x = make(lens, H, 1, P, N, torch.float16)
        state[pool - 1] = x["state"][0].to(DEV)
        g = gpu(x)
        slots = torch.tensor([pool - 1], dtype=torch.int32, device=DEV)
        out = prefill(g, lens, state=state, slots=slots)
        check(out, state[pool - 1:], reference(x, lens))
    assert not state[:pool - 1].any()


def test_a_value_that_is_not_finite():
    """It stays in its sequence, its column of x or its head, and the tokens from 63 before it on; NaN comes back as NaN."""
    lens = [200, 100]
    x = make(lens, 2, 1, 64, 64, torch.bfloat16)
    x["x"][150, 0, 5] = float("nan")
    x["dt"][230, 1] = float("nan")
    g = gpu(x)
    out = prefill(g, lens).cpu()
    bad = out.isnan()
    assert bad[150:200, 0, 5].all() and bad[230:, 1].all()
    bad[87:200, 0, 5] = False
    bad[200:, 1] = False
    assert not bad.any() and not g["state"].cpu()[0, 1].isnan().any() and g["state"].cpu()[1, 1].isnan().all()
    assert g["state"].cpu()[0, 0, 5].isnan().all() and not g["state"].cpu()[0, 0, 6].isnan().any()
