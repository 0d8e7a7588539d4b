"""ops.sample_filtered against the draw on the sorted row in 64 bits. Tokens must be equal; the logarithms of
the probabilities are fp32 roundings of 64-bit values (masses kept to 2^-44 of the largest): 2^-23 of the
value and of 1.
"""
import numpy as np
import pytest
import torch

from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(l, u, T, k, tp, mp):
    """One row: (token, log of its share)."""
    l = l.astype(np.float64)
    l = np.where(np.isnan(l), -np.inf, l) + 0.0
    order = np.argsort(-l, kind="stable")
    s = l[order]
    if s[0] == -np.inf:
        return -1, -np.inf
    if not T > 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.where(s == s[0], 1.0, np.exp((s - s[0]) / T))
        e = np.where((s < s[0]) & ((s == -np.inf) | (s[0] == np.inf)), 0.0, e)   # (at T = inf too: -inf / inf is NaN)
    nk = k if 0 < k < len(l) else len(l)
    above = np.concatenate([[0.0], np.cumsum(e)])
    Z = above[nk]
    n = nk
    if tp < 1:
        n = min(n, int((above[:nk] <= max(tp, 0.0) * Z).sum()))
    n = max(1, min(n, int((e >= mp).sum())))
    S = above[n]
    u = min(max(u, 0.0), np.float64(np.float32(1) - np.float32(2.0 ** -24))) if u == u else 0.0
    j = int((above[1:n + 1] <= u * S).sum())
    return int(order[j]), float(np.log(e[j] / S))


def run_check(logits, u, T, k, tp, mp, as_tensors=True):
    d = logits.to(DEV)
    B = logits.shape[0]
    t = lambda x, dt: (torch.as_tensor(np.broadcast_to(np.asarray(x), (B,)).copy(), dtype=dt).to(DEV)
                       if as_tensors else x)
    args = dict(temperature=t(T, torch.float32), top_k=t(k, torch.int32), top_p=t(tp, torch.float32),
                min_p=t(mp, torch.float32))
    u32 = torch.as_tensor(np.asarray(u, np.float32)).to(DEV)
    tok, lp = ops.sample_filtered(d, u32, want_logprob=True, **args)
    assert torch.equal(tok, ops.sample_filtered(d, u32, **args))
    f32 = lambda x: np.broadcast_to(np.asarray(x, np.float32), (B,)).astype(np.float64)
    Tb, tpb, mpb, kb = f32(T), f32(tp), f32(mp), np.broadcast_to(np.asarray(k), (B,))
    rows = logits.float().numpy()
    tok, lp, us = tok.cpu().numpy(), lp.cpu().numpy(), u32.cpu().numpy().astype(np.float64)
    for b in range(B):
        rt, rl = reference(rows[b], us[b], Tb[b], int(kb[b]), tpb[b], mpb[b])
        assert tok[b] == rt, (b, int(tok[b]), rt, us[b], Tb[b], kb[b], tpb[b], mpb[b])
        if np.isfinite(rl):
            assert abs(lp[b] - rl) <= 2.0 ** -23 * (1 + abs(rl)), (b, lp[b], rl)
        else:
            assert lp[b] == rl


def settings(rng, B):
    pick = rng.random((4, B))
    T = np.where(pick[0] < 0.1, 0.0, 0.3 + 1.2 * rng.random(B))
    k = np.where(pick[1] < 0.4, 0, rng.integers(1, 300, B))
    tp = np.where(pick[2] < 0.3, 1.0, rng.random(B))
    mp = np.where(pick[3] < 0.5, 0.0, 0.2 * rng.random(B))
    return T, k, tp, mp


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1024, 2049, 50288, 131071])
def test_random(V, dtype):
    rng = np.random.default_rng([V, 3])
    B = 40 if V < 10000 else 12
    l = torch.from_numpy(rng.normal(0, 2.5, (B, V)).astype(np.float32)).to(dtype)
    run_check(l, rng.random(B).astype(np.float32), *settings(rng, B))


def test_largest_vocabulary_and_many_rows():
    rng = np.random.default_rng(5)
    l = torch.from_numpy(rng.normal(0, 3, (3, 262144)).astype(np.float32))
    run_check(l, rng.random(3).astype(np.float32), *settings(rng, 3))
    l = torch.from_numpy(rng.normal(0, 3, (700, 777)).astype(np.float32)).half()
    run_check(l, rng.random(700).astype(np.float32), *settings(rng, 700))


@pytest.mark.parametrize("V", [5, 3000, 50288])
def test_ties(V):
    """Equal logits rank by index: all equal, two levels, and -0 beside +0; more ties than fit one search."""
    rng = np.random.default_rng([V, 7])
    B = 12
    l = np.zeros((B, V), np.float32)
    l[1::3] = rng.integers(0, 2, (4, V)) * 0.25
    l[2::3] = np.where(rng.random((4, V)) < 0.5, -0.0, 0.0)
    T, k, tp, mp = settings(rng, B)
    run_check(torch.from_numpy(l).half(), (np.arange(B) / B).astype(np.float32), T, k, tp, mp)


def test_masks_and_special_values():
    """-inf masks up to the whole row, NaN logits, +inf logits, the type's lowest value as a mask."""
    rng = np.random.default_rng(11)
    V, B = 3001, 12
    l = rng.normal(0, 2, (B, V)).astype(np.float32)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, :] = -np.inf
    l[2, 1777] = -3.0
    l[3, rng.random(V) < 0.9] = -np.inf
    l[4, [5, 900]] = np.inf
    l[5, ::2] = np.nan
    l[6] = -65504.0
    l[7, rng.random(V) < 0.95] = -65504.0
    l[8, 100] = 65504.0
    l[9, :] = np.inf
    l[10, 1:] = -np.inf
    for T, k, tp, mp in [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.05), (0.0, 0, 1.0, 0.0), (1.3, 2000, 0.99, 0.0)]:
        run_check(torch.from_numpy(l).half(), rng.random(B).astype(np.float32), T, k, tp, mp)
        run_check(torch.from_numpy(l), rng.random(B).astype(np.float32), T, k, tp, mp, as_tensors=False)


@pytest.mark.parametrize("T", [1e-30, 1e-3, 40.0, 1e30, float("inf"), -1.0, float("nan")])
def test_temperatures(T):
    rng = np.random.default_rng(13)
    l = torch.from_numpy(rng.normal(0, 4, (6, 5000)).astype(np.float32)).bfloat16()
    run_check(l, rng.random(6).astype(np.float32), T, np.array([0, 40, 0, 4999, 5000, 9999]), 0.9, 0.0)


def test_borders():
    """u at both ends and outside, filters that keep one token or everything."""
    rng = np.random.default_rng(17)
    l = torch.from_numpy(rng.normal(0, 2, (8, 4097)).astype(np.float32)).half()
    u = np.array([0.0, 1.0 - 2.0 ** -24, 1.0, -1.0, 2.0, np.nan, 2.0 ** -24, 0.5], np.float32)
    for k, tp, mp in [(0, 1.0, 0.0), (1, 1.0, 0.0), (0, 0.0, 0.0), (0, 1.0, 1.0), (4097, 2.0, -1.0), (-3, -1.0, 0.0),
                      (7, 0.6, 0.3)]:
        run_check(l, u, 0.8, k, tp, mp)


def test_peaked_far_from_the_rest():
    """One token far above: what lies below shares few bins of the search, which goes over the row."""
    rng = np.random.default_rng(19)
    l = rng.normal(0, 1, (6, 50288)).astype(np.float32)
    l[:, 77] = 200.0
    l[3:, 4000:4004] = 190.0
    run_check(torch.from_numpy(l), rng.random(6).astype(np.float32), 0.9, np.array([0, 20, 30000, 0, 3, 50000]),
              np.array([1.0, 1.0, 1.0, 0.5, 0.9, 1.0]), 0.0)


def test_strided_rows_and_scalars():
    """Rows of a wider buffer (odd row length: no alignment), and numbers instead of tensors."""
    rng = np.random.default_rng(23)
    wide = torch.from_numpy(rng.normal(0, 2, (9, 2011)).astype(np.float32)).half()
    l = wide[:, 3:2004]
    u = rng.random(9).astype(np.float32)
    run_check(l, u, 0.8, 20, 0.95, 0.01, as_tensors=False)
    d, ud = wide.to(DEV), torch.from_numpy(u).to(DEV)
    a = ops.sample_filtered(d[:, 3:2004], ud, temperature=0.8, top_k=20)
    b = ops.sample_filtered(d[:, 3:2004].contiguous(), ud, temperature=0.8, top_k=20)
    c = ops.sample_filtered(d[:, 3:2004].t().contiguous().t(), ud, temperature=0.8, top_k=20)
    assert torch.equal(a, b) and torch.equal(a, c)
    one = ops.sample_filtered(d[:1, 3:2004].expand(9, -1), ud, temperature=0.8, top_k=20)   # stride 0
    assert one[0] == a[0]


def test_streams_and_graph():
    rng = np.random.default_rng(29)
    rows = [torch.from_numpy(rng.normal(0, 2, (3, 50288)).astype(np.float32)).half().to(DEV) for _ in range(3)]
    us = [torch.from_numpy(rng.random(3).astype(np.float32)).to(DEV) for _ in range(3)]
    kw = dict(temperature=0.8, top_k=100, top_p=0.95, min_p=0.001, want_logprob=True)
    want = [ops.sample_filtered(l, u, **kw) for l, u in zip(rows, us)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in rows]
    got = []
    for l, u, s in zip(rows, us, streams):
        with torch.cuda.stream(s):
            got.append(ops.sample_filtered(l, u, **kw))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    l, u = rows[0].clone(), us[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.sample_filtered(l, u, **kw)
    for i in (1, 2, 0, 1):
        l.copy_(rows[i])
        u.copy_(us[i])
        ops.sample_filtered(rows[2], us[2], **kw)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


def test_refusals():
    l, u = torch.zeros(2, 8, device=DEV), torch.zeros(2, device=DEV)
    with pytest.raises(TypeError):
        ops.sample_filtered(l.double(), u)
    with pytest.raises(TypeError):
        ops.sample_filtered(l, u.half())
    with pytest.raises(ValueError):
        ops.sample_filtered(l, u[:1])
    with pytest.raises(ValueError):
        ops.sample_filtered(l[0], u)
    with pytest.raises(ValueError):
        ops.sample_filtered(torch.zeros(2, 262145, device=DEV), u)
    with pytest.raises(TypeError):
        ops.sample_filtered(l, u, top_k=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError):
        ops.sample_filtered(l, u, top_p=torch.ones(3, device=DEV))
    assert ops.sample_filtered(l[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_infinities_and_signalling_nans(dtype):
    """Several +inf logits with every filter (each mass 1, in index order); NaNs of either kind beside the largest."""
    rng = np.random.default_rng(31)
    V, B = 5003, 9
    l = rng.normal(0, 2, (B, V)).astype(np.float32)
    l[:, rng.random(V) < 0.01] = np.inf
    l[2, 17:] = np.nan
    l[3] = np.inf
    l[6:] = rng.normal(0, 2, (3, V))
    d = torch.from_numpy(l).to(dtype)
    bits = d.view(torch.int16 if dtype == torch.float16 else torch.int32)
    quiet = {torch.float16: 0x7C01, torch.float32: 0x7F800001}[dtype]                    # signalling: quiet bit clear
    bits[6:, rng.random(V) < 0.3] = quiet
    bits[7, 1::2] = quiet
    for T, k, tp, mp in [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (0.7, 0, 0.5, 0.0), (1.3, 30, 0.4, 1.0),
                         (0.9, 0, 0.0, 0.0), (0.9, 0, 1.0, 1.5), (float("inf"), 4000, 0.9, 0.0)]:
        run_check(d, rng.random(B).astype(np.float32), T, k, tp, mp)


@pytest.mark.parametrize("spread", [1e-38, 1e-6, 1.0, 1e4, 1e30])
def test_spreads(spread):
    """Logits closer together and further apart than any model's, around 0 and around a large value."""
    rng = np.random.default_rng(37)
    l = (rng.normal(0, 1, (8, 6007)) * spread).astype(np.float32)
    l[4:] += np.float32(1000.0 * spread)
    u = rng.random(8).astype(np.float32)
    for T in (0.8 * spread, 1.0):
        run_check(torch.from_numpy(l), u, T, np.array([0, 30, 0, 5000] * 2), np.array([0.9, 0.9, 1.0, 0.99] * 2),
                  np.array([0.0, 0.0, 0.05, 0.0] * 2))


@pytest.mark.parametrize("T", [1e-37, 1e-38, 1e-44])
def test_bins_out_of_reach(T):
    """So small a temperature that a bin of the logits further down begins beyond fp32: top_k cuts there."""
    rng = np.random.default_rng(43)
    l = torch.from_numpy(rng.normal(0, 4, (5, 7001)).astype(np.float32))
    l[1] = l[1].round()
    l[3:, ::2] = l[3:].amax()
    run_check(l, rng.random(5).astype(np.float32), T, np.array([2100, 5000, 0, 2047, 3600]), np.array([0.9, 1.0, 0.5, 1.0, 0.3]),
              np.array([0.0, 0.0, 0.0, 0.5, 0.0]))


def test_rows_past_32_bits():
    """Rows further apart than 2^31 elements."""
    V, ld = 9001, (1 << 31) + 24
    wide = torch.empty(ld + V, dtype=torch.float16, device=DEV)
    l = wide.as_strided((2, V), (ld, 1))
    l.copy_(torch.from_numpy(np.random.default_rng(47).normal(0, 2, (2, V)).astype(np.float32)))
    u = torch.tensor([0.3, 0.8], device=DEV)
    for kw in (dict(top_k=40), dict(top_p=0.9)):
        got = ops.sample_filtered(l, u, temperature=0.9, want_logprob=True, **kw)
        want = ops.sample_filtered(l.contiguous(), u, temperature=0.9, want_logprob=True, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
