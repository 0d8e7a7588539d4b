"""The gated delta rule (ops.gated_delta_step, ops.gated_delta_prefill) against its recurrence in 64 bits.

Tolerance: the operators work in fp32 (products of the chunked form in pairs of halves, 22 bits), so the state
may be off by a few hundred roundings of 2^-24 of the head's largest value, taken as 2^-17 of it (a product
with operands of 16 bits would be off by 2^-9 to 2^-12). Outputs are rounded to their type on top: half a step.
"""
import numpy as np
import pytest
import torch

from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ATOL = 2.0 ** -17


def make(lens, Hk, Hv, Dk, Dv, dtype, seed=0, pool=None, l2norm=True):
    gen = torch.Generator().manual_seed(seed)
    T, n = sum(lens), len(lens)
    size = 1.0 if l2norm else Dk ** -0.5
    x = {"q": (size * torch.randn(T, Hk, Dk, generator=gen)).to(dtype),
         "k": (size * torch.randn(T, Hk, Dk, generator=gen)).to(dtype),
         "v": torch.randn(T, Hv, Dv, generator=gen).to(dtype),
         "g": -torch.nn.functional.softplus(2 * torch.randn(T, Hv, generator=gen) - 3),
         "beta": torch.sigmoid(torch.randn(T, Hv, generator=gen)),
         "state": 0.3 * torch.randn(pool or n, Hv, Dv, Dk, generator=gen)}
    return x


def recurrence(x, lens, l2norm, slots=None, scale=None):
    """Token by token in fp64: out (T, Hv, Dv) and the states (pool, ...) afterwards."""
    q, k, v, g, beta = (x[n].double() for n in ("q", "k", "v", "g", "beta"))
    Hk, Hv, Dk = q.shape[1], v.shape[1], q.shape[2]
    if l2norm:
        q = q / (q.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()
        k = k / (k.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()
    q, k = (t.repeat_interleave(Hv // Hk, 1) for t in (q, k))
    state = x["state"].double().clone()
    out = torch.zeros(v.shape, dtype=torch.float64)
    t = 0
    for b, n in enumerate(lens):
        S = state[b if slots is None else slots[b]]
        for _ in range(n):
            S.mul_(torch.exp(g[t])[:, None, None])
            u = beta[t][:, None] * (v[t] - (S * k[t][:, None]).sum(-1))
            S.add_(u[..., None] * k[t][:, None])
            out[t] = (S * q[t][:, None]).sum(-1)
            t += 1
    return out * (Dk ** -0.5 if scale is None else scale), state


def check(got, ref, what, roundings=1):
    got, ref = got.cpu(), ref
    assert torch.isfinite(got.double()).all(), what
    half = roundings * torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    err = (got.double() - ref).abs()
    if got.dtype == torch.float32:                                     # states (slots, heads, Dv, Dk)
        top = ref.abs().amax((-1, -2), keepdim=True).clamp_min(1e-3)
    else:                                                              # outputs (tokens, heads, Dv)
        top = ref.abs().amax((0, 2), keepdim=True).clamp_min(1e-3)
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0           # half a step of the subnormal halves
    bad = err > half * ref.abs() * (1 + 2.0 ** -7) + ATOL * top + tiny
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float((err / top).max()):.3g} of the largest"


def gpu(x):
    return {n: t.to(DEV) for n, t in x.items()}


def prefill(x, lens, **kw):
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    return ops.gated_delta_prefill(x["q"], x["k"], x["v"], x["g"], x["beta"], x["state"], cu_seqlens=cu, **kw)


# batch, heads, key and value dimensions; 208 leaves a part of a 64-row block
STEP = [(1, 1, 1, 128, 16), (1, 16, 64, 128, 64), (3, 2, 6, 64, 208), (5, 1, 8, 128, 256), (33, 4, 8, 64, 32),
        (64, 8, 8, 128, 64), (2, 3, 3, 64, 112), (33, 4, 8, 64, 208), (64, 4, 16, 128, 48)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("l2norm", [True, False])
@pytest.mark.parametrize("shape", STEP)
def test_step(shape, l2norm, dtype):
    B, Hk, Hv, Dk, Dv = shape
    x = make([1] * B, Hk, Hv, Dk, Dv, dtype, seed=B + Dv, l2norm=l2norm)
    ref, ref_state = recurrence(x, [1] * B, l2norm)
    d = gpu(x)
    out = ops.gated_delta_step(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], l2norm=l2norm)
    check(out, ref, "out")
    check(d["state"], ref_state, "state")


LENS = [[1], [2], [15], [16], [17], [63], [64], [65], [129], [0, 5, 0], [200, 1, 64, 0, 33], [1] * 9, [257, 300]]
HEADS = [(1, 1, 128, 64), (2, 4, 128, 64), (1, 3, 64, 48), (2, 2, 64, 256), (1, 2, 128, 208)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("lens", LENS, ids=lambda l: "-".join(map(str, l)))
def test_prefill(lens, heads, dtype):
    Hk, Hv, Dk, Dv = heads
    l2norm = (len(lens) + Dv // 16) % 2 == 0
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=sum(lens), l2norm=l2norm)
    ref, ref_state = recurrence(x, lens, l2norm)
    d = gpu(x)
    out = prefill(d, lens, l2norm=l2norm)
    check(out, ref, "out")
    check(d["state"], ref_state, "state")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_long(dtype):
    """Many chunks: the state is carried on without losing bits."""
    lens = [2500]
    x = make(lens, 1, 2, 128, 64, dtype, seed=9)
    x["g"] = x["g"] * 0.05                                             # a state that remembers
    ref, ref_state = recurrence(x, lens, True)
    d = gpu(x)
    check(prefill(d, lens, l2norm=True), ref, "out")
    check(d["state"], ref_state, "state")


def test_prefill_batch_form_and_scale():
    """(B, T, ...) without offsets is the packed form with equal lengths; scale is a factor of the output."""
    B, T = 3, 70
    x = make([T] * B, 2, 4, 128, 64, torch.float16, seed=4)
    ref, ref_state = recurrence(x, [T] * B, True, scale=0.5)
    d = gpu(x)
    s = lambda t: t.view(B, T, *t.shape[1:])
    out = ops.gated_delta_prefill(s(d["q"]), s(d["k"]), s(d["v"]), s(d["g"]), s(d["beta"]), d["state"], scale=0.5,
                                  l2norm=True)
    assert out.shape == (B, T, 4, 64)
    check(out.flatten(0, 1), ref, "out")
    check(d["state"], ref_state, "state")


@pytest.mark.parametrize("kind", ["step", "prefill"])
def test_slots(kind):
    """Sequences in a larger pool: padding gives zeros, a slot past the pool or taken twice NaN, and no other
    slot is touched; in place and into state_out."""
    lens = [1] * 6 if kind == "step" else [70, 3, 0, 65, 2, 20]
    slots = [4, -1, 2, 9, 4, 0]                                        # sequences 1 padding, 3 past the end, 4 twice
    x = make(lens, 2, 4, 128, 64, torch.bfloat16, seed=11, pool=7)
    keep = [b for b in (0, 2, 5)]
    ref, ref_state = torch.zeros(sum(lens), 4, 64, dtype=torch.float64), x["state"].double().clone()
    first = np.concatenate([[0], np.cumsum(lens)])
    for b in keep:
        one = {n: (t if n == "state" else t[first[b]:first[b + 1]]) for n, t in x.items()}
        o, st = recurrence(one, [lens[b]], True, slots=[slots[b]])
        ref[first[b]:first[b + 1]] = o
        ref_state[slots[b]] = st[slots[b]]
    for in_place in (True, False):
        d = gpu(x)
        st = torch.tensor(slots, dtype=torch.int32, device=DEV)
        so = None if in_place else torch.full_like(d["state"], 7.0)
        if kind == "step":
            out = ops.gated_delta_step(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], slots=st, l2norm=True,
                                       state_out=so)
        else:
            out = prefill(d, lens, slots=st, l2norm=True, state_out=so)
        out = out.cpu()
        assert (out[first[1]:first[2]] == 0).all()
        for b in (3, 4):
            assert torch.isnan(out[first[b]:first[b + 1]]).all()
        for b in keep:
            if lens[b]:
                check(out[first[b]:first[b + 1]], ref[first[b]:first[b + 1]], f"out {b}")
        touched = [slots[b] for b in keep]
        if in_place:
            check(d["state"][touched], ref_state[touched], "state")
        else:
            assert torch.equal(d["state"].cpu(), x["state"])
            check(so[touched], ref_state[touched], "state_out")
        rest = [i for i in range(7) if i not in touched]
        after = (d["state"] if in_place else so)[rest].cpu()
        assert torch.equal(after, x["state"][rest] if in_place else torch.full_like(after, 7.0))


@pytest.mark.parametrize("lens", [[1], [5], [100]])
def test_strided(lens):
    """q, k and v as parts of packed rows, g and beta as columns of one projection, out into a wider buffer whose
    rows behind the last sequence and other columns stay as they were."""
    T, Hk, Hv, Dk, Dv = sum(lens), 2, 4, 128, 64
    x = make(lens, Hk, Hv, Dk, Dv, torch.float16, seed=21)
    ref, ref_state = recurrence(x, lens, True)
    d = gpu(x)
    packed = torch.cat([d["q"].flatten(1), d["k"].flatten(1), d["v"].flatten(1), torch.zeros(T, 8, device=DEV).half()], 1)
    packed = torch.cat([packed, torch.full((3, packed.shape[1]), float("nan"), device=DEV).half()])
    gb = torch.cat([d["g"], d["beta"], torch.zeros(T, 3, device=DEV)], 1)
    gb = torch.cat([gb, torch.full((3, gb.shape[1]), float("nan"), device=DEV)])
    a, b = Hk * Dk, 2 * Hk * Dk
    wide = torch.full((T + 3, Hv * Dv + 16), 5.0, device=DEV, dtype=torch.float16)
    out = wide[:, :Hv * Dv].view(T + 3, Hv, Dv)
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
    ops.gated_delta_prefill(packed[:, :a].view(-1, Hk, Dk), packed[:, a:b].view(-1, Hk, Dk),
                            packed[:, b:b + Hv * Dv].view(-1, Hv, Dv), gb[:, :Hv], gb[:, Hv:2 * Hv], d["state"],
                            cu_seqlens=cu, l2norm=True, out=out)
    check(out[:T].contiguous(), ref, "out")
    check(d["state"], ref_state, "state")
    assert (wide[T:] == 5).all() and (wide[:, Hv * Dv:] == 5).all()
    d = gpu(x)                                                        # rows that no 16-byte load can take
    odd = lambda t: torch.cat([t, t[..., :1]], -1)[..., :-1]
    ops.gated_delta_prefill(odd(d["q"]), odd(d["k"]), odd(d["v"]), odd(d["g"]), odd(d["beta"]), d["state"],
                            cu_seqlens=cu, l2norm=True, out=out[:T])
    check(out[:T].contiguous(), ref, "out")


@pytest.mark.parametrize("lens", [[1], [40], [150]])
def test_extremes(lens):
    """-inf decays (a forgotten state, first, last and in the middle of a chunk), beta 0 and 1, zero keys and
    queries, and a long decay beside short ones."""
    T = sum(lens)
    x = make(lens, 1, 3, 128, 64, torch.bfloat16, seed=31)
    x["g"][0, 0] = float("-inf")
    x["g"][T // 2, 1] = float("-inf")
    x["g"][T - 1, 2] = -300.0
    x["g"][:, 2] -= 20.0
    x["beta"][::3] = 0.0
    x["beta"][1::3] = 1.0
    x["k"][T // 3] = 0.0
    x["q"][T // 4] = 0.0
    ref, ref_state = recurrence(x, lens, True)
    d = gpu(x)
    check(prefill(d, lens, l2norm=True), ref, "out")
    check(d["state"], ref_state, "state")


@pytest.mark.parametrize("size", [2.0 ** -18, 2.0 ** 14])
def test_ranges(size):
    """Values, keys and states far from 1, without normalisation (k v stays within the recurrence's own range:
    keys shrink as values grow)."""
    lens = [100]
    x = make(lens, 1, 2, 128, 64, torch.bfloat16, seed=41, l2norm=False)
    x["v"] = (x["v"].float() * size).bfloat16()
    x["state"] = x["state"] * size
    ref, ref_state = recurrence(x, lens, False)
    d = gpu(x)
    out = prefill(d, lens)
    check(out.float().cpu().div(size).bfloat16(), ref / size, "out")
    check(d["state"] / size, ref_state / size, "state")


def test_prefill_equals_steps():
    """A prompt in one call, in two calls, and token by token leave the same state."""
    lens = [90]
    x = make(lens, 2, 4, 64, 64, torch.float16, seed=51)
    d = gpu(x)
    st0 = d["state"].clone()
    whole = prefill(d, lens, l2norm=True)
    state = st0.clone()
    parts = []
    for lo, hi in ((0, 37), (37, 90)):
        y = {n: (t if n == "state" else t[lo:hi]) for n, t in dict(d, state=state).items()}
        parts.append(prefill(y, [hi - lo], l2norm=True))
    # both sides are rounded here: two fp32 values a hair apart may fall to either side of a border, one whole
    # step (half a step from each) apart
    check(torch.cat(parts), whole.double().cpu(), "two calls", roundings=2)
    check(state, d["state"].double().cpu(), "state of two calls")
    state = st0.clone()
    for t in range(90):
        o = ops.gated_delta_step(*(d[n][t:t + 1] for n in ("q", "k", "v", "g", "beta")), state, l2norm=True)
    check(state, d["state"].double().cpu(), "state of steps")
    check(o, whole[-1:].double().cpu(), "last token", roundings=2)


def test_bad_offsets_stay_inside():
    """Offsets outside the tensors or running backwards are held to them: nothing else is written."""
    x = make([70], 1, 2, 128, 64, torch.float16, seed=61, pool=4)
    d = gpu(x)
    buf = torch.full((90, 2, 64), 3.0, device=DEV, dtype=torch.float16)
    cu = torch.tensor([-5, 60, 40, 1000, 1000], dtype=torch.int32, device=DEV)
    ops.gated_delta_prefill(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], cu_seqlens=cu, l2norm=True,
                            out=buf[10:80])
    torch.cuda.synchronize()
    assert (buf[:10] == 3).all() and (buf[80:] == 3).all()


def test_streams_and_graph():
    """On a side stream, two calls at once on two streams, and captured and replayed with new inputs."""
    lens = [150, 70]
    x = make(lens, 1, 2, 128, 64, torch.float16, seed=71)
    y = make(lens, 1, 2, 128, 64, torch.float16, seed=72)
    refs = [recurrence(t, lens, True) for t in (x, y)]
    ds = [gpu(x), gpu(y)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for d, s in zip(ds, streams):
        with torch.cuda.stream(s):
            outs.append(prefill(d, lens, l2norm=True))
    torch.cuda.synchronize()
    for d, o, (ref, ref_state) in zip(ds, outs, refs):
        check(o, ref, "out")
        check(d["state"], ref_state, "state")

    cu = torch.tensor([0, 150, 220], dtype=torch.int32, device=DEV)
    s = {n: t.clone() for n, t in gpu(x).items()}
    so = torch.zeros_like(s["state"])
    tok = {n: s[n][:2] for n in ("q", "k", "v", "g", "beta")}

    def both():
        o = ops.gated_delta_prefill(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], cu_seqlens=cu, l2norm=True,
                                    state_out=so)
        return o, ops.gated_delta_step(tok["q"], tok["k"], tok["v"], tok["g"], tok["beta"], so, l2norm=True)
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for z in (y, x, y):
        for n, t in gpu(z).items():
            s[n].copy_(t)
        eager = [t.clone() for t in both()]
        eager_state = so.clone()
        so.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1]) and torch.equal(so, eager_state)


def test_refusals():
    x = gpu(make([4], 2, 4, 128, 64, torch.float16))
    step = lambda **kw: ops.gated_delta_step(**{**x, **kw})
    with pytest.raises(TypeError):
        step(q=x["q"].float())
    with pytest.raises(TypeError):
        step(k=x["k"].bfloat16())
    with pytest.raises(TypeError):
        step(g=x["g"].half())
    with pytest.raises(TypeError):
        step(state=x["state"].half())
    with pytest.raises(ValueError):
        step(v=x["v"][:, :3])                                          # 3 value heads of 2 key heads
    with pytest.raises(ValueError):
        step(k=x["k"][:2])
    with pytest.raises(ValueError):
        step(state=x["state"])                                         # one slot for four sequences
    with pytest.raises(ValueError):
        step(state=x["state"].transpose(-1, -2))
    with pytest.raises(ValueError):
        step(q=x["q"][..., :96], k=x["k"][..., :96])
    with pytest.raises(TypeError):
        step(slots=torch.zeros(4, dtype=torch.int64, device=DEV))
    big = torch.zeros(6, 4, 64, 128, device=DEV)
    with pytest.raises(ValueError):
        step(state=big[:4], state_out=big[1:5])                        # overlaps
    with pytest.raises(TypeError):
        prefill(x, [4], out=torch.zeros(4, 4, 64, device=DEV))
    with pytest.raises(ValueError):
        ops.gated_delta_prefill(**x)                                   # packed without offsets
    assert ops.gated_delta_step(*(x[n][:0] for n in ("q", "k", "v", "g", "beta")), x["state"]).shape == (0, 4, 64)


@pytest.mark.parametrize("n", [255, 256, 257, 300])
def test_many_sequences(n):
    """Around the number up to which sequences are taken by length."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 140, n) * (rng.random(n) < 0.3) + rng.integers(0, 3, n)]
    x = make(lens, 1, 2, 64, 32, torch.float16, seed=n)
    ref, ref_state = recurrence(x, lens, True)
    d = gpu(x)
    out = prefill(d, lens, l2norm=True)
    check(out, ref, "out")
    check(d["state"], ref_state, "state")


def test_more_chunks_than_one_pass_holds():
    """A workspace's worth of chunks and the rest: bit for bit the same prompt in two calls, each of one pass."""
    lens, Hk, Hv, Dk, Dv = [15000, 9000], 4, 256, 64, 16
    x = gpu(make(lens, Hk, Hv, Dk, Dv, torch.bfloat16, seed=91))
    states = [x["state"].clone(), x["state"].clone()]
    whole = prefill({**x, "state": states[0]}, lens, l2norm=True)
    parts = torch.empty_like(whole)
    for b, first, last in ((0, 0, 6400), (1, 15000, 21400), (0, 6400, 15000), (1, 21400, 24000)):
        ops.gated_delta_prefill(*(x[n][first:last] for n in ("q", "k", "v", "g", "beta")), states[1],
                                cu_seqlens=torch.tensor([0, last - first], dtype=torch.int32, device=DEV),
                                slots=torch.tensor([b], dtype=torch.int32, device=DEV), l2norm=True,
                                out=parts[first:last])
    assert torch.equal(whole, parts) and torch.equal(states[0], states[1])


def test_offsets_past_32_bits():
    """Slots behind 2^31 values of the state, and tokens so far apart that they pass 2^31 elements: the same bits as
    close together."""
    lens, (Hk, Hv, Dk, Dv), ld = [290, 3], (1, 2, 128, 64), 1 << 23
    x = gpu(make(lens, Hk, Hv, Dk, Dv, torch.float16, seed=97))
    pool = (1 << 31) // (Hv * Dv * Dk) + 3
    near, state = x["state"].clone(), torch.zeros(pool, Hv, Dv, Dk, device=DEV)
    slots = torch.tensor([pool - 1, pool - 2], dtype=torch.int32, device=DEV)
    state[slots.long()] = near
    want = prefill({**x, "state": near}, lens, l2norm=True)
    wide, wide32 = torch.empty(sum(lens) * ld, dtype=torch.float16, device=DEV), torch.empty(sum(lens) * ld, device=DEV)
    at, far = 0, {}
    for n in ("q", "k", "v", "out"):
        t = x[n] if n in x else want
        far[n] = wide.as_strided(t.shape, (ld, t.shape[2], 1), at)
        at += t.shape[1] * t.shape[2]
    for i, n in enumerate(("g", "beta")):
        far[n] = wide32.as_strided(x[n].shape, (ld, 1), i * Hv)
    for n in ("q", "k", "v", "g", "beta"):
        far[n].copy_(x[n])
    out = prefill({**far, "state": state}, lens, l2norm=True, slots=slots, out=far["out"])
    assert torch.equal(out, want) and torch.equal(state[slots.long()], near) and not state[:pool - 2].any()
    # one token of each, which are 290 tokens apart
    step = {n: far[n][::290][:2] for n in ("q", "k", "v", "g", "beta")}
    assert step["q"].stride(0) > 1 << 31
    a = ops.gated_delta_step(*(step[n] for n in ("q", "k", "v", "g", "beta")), state, slots=slots, l2norm=True)
    b = ops.gated_delta_step(*(step[n].contiguous() for n in ("q", "k", "v", "g", "beta")), near, l2norm=True)
    assert torch.equal(a, b) and torch.equal(state[slots.long()], near)
