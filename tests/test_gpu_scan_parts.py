"""The chunked selective scan where its factors' splitting into 16-bit parts shows: terms that cancel, and beside fp16 rows values of
very different size in one column.

Tolerances: see each test. Decays are switched off (A_log -200: e^-200 is zero in fp32), so that nothing else rounds."""
import pytest
import torch

import layer_math as lm
from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# Two values 2^-22 apart. Of 1 + 2^-9 + 2^-17 -+ 2^-23 two parts of 8 bits hold 1 + 2^-9 and 1 + 2^-9 + 2^-16, 2^-16 apart.
NEAR, FAR = 1 + 2.0 ** -9 + 2.0 ** -17 - 2.0 ** -23, 1 + 2.0 ** -9 + 2.0 ** -17 + 2.0 ** -23


def call(x, dt, B, C, state, lens, softplus=False, D=None):
    state = state.to(DEV)
    A_log = torch.full((x.shape[1],), -200.0, device=DEV)
    out = ops.selective_scan_prefill(x.to(DEV), dt.to(DEV), A_log, B.to(DEV), C.to(DEV), state, D=D, cu_seqlens=lm.offsets(lens, DEV),
                                     softplus=softplus)
    return out.cpu().double(), state.cpu().double()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,N", [(64, 128), (48, 64)])
@pytest.mark.parametrize("n", [0, 17, 62])
def test_a_state_whose_terms_cancel(n, P, N, dtype):
    """y = h_n - h_{n+1}, no time passes. The sums of two terms of size 1 in a few parts each take less than 16 roundings of 2^-24
    of 1: 2^-20. (Two bf16 parts are off by 2^-16.) Parts of halves are off by 2^-23 each."""
    T = 100
    x, B, C = torch.ones(T, 2, P).to(dtype), torch.ones(T, 1, N).to(dtype), torch.zeros(T, 1, N).to(dtype)
    C[:, 0, n], C[:, 0, n + 1] = 1, -1
    state = torch.zeros(1, 2, P, N)
    state[..., n], state[..., n + 1] = NEAR, FAR
    out, after = call(x, torch.zeros(T, 2), B, C, state, [T])
    assert (out - (NEAR - FAR)).abs().max() <= 2.0 ** -20 and torch.equal(after, state.double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("P,N", [(64, 128), (48, 64)])
@pytest.mark.parametrize("j", [0, 15, 17, 31, 40, 62])
def test_scores_that_cancel(j, P, N, dtype):
    """y_i = d_j x_j + d_{j+1} x_{j+1} with x = 1, -1, scores of 1: as above, in the matrix of scores and decays."""
    T = 64
    x, B, C = torch.zeros(T, 2, P).to(dtype), torch.zeros(T, 1, N).to(dtype), torch.zeros(T, 1, N).to(dtype)
    x[j], x[j + 1] = 1, -1
    B[:, 0, 3] = C[:, 0, 3] = 1
    dt = torch.zeros(T, 2)
    dt[j], dt[j + 1] = NEAR, FAR
    out, _ = call(x, dt, B, C, torch.zeros(1, 2, P, N), [T])
    assert not out[:j].any() and (out[j] - NEAR).abs().max() <= lm.half_step(dtype)[0] * NEAR
    assert (out[j + 1:] - (NEAR - FAR)).abs().max() <= 2.0 ** -20


def ordinary(lens, H, P, N, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    T = sum(lens)
    return r(T, H, P).half(), 0.1 + 0.1 * torch.rand(T, H, generator=gen), r(T, 1, N).half(), r(T, 1, N).half(), 0.01 * r(len(lens), H, P, N)


@pytest.mark.parametrize("large", [1e6, 1e8, 1e20])
@pytest.mark.parametrize("lens", [[100], [900, 70]])
def test_small_states_beside_a_large_one(lens, large):
    """fp16 rows: a state value far above the others of its column takes no bits from them: within 2^-18 of their own terms."""
    H, P, N = 2, 32, 64
    x, dt, B, C, state = ordinary(lens, H, P, N)
    state[..., 7] = large
    _, _, s, smag = lm.scan(x, dt, torch.full((H,), -200.0), B, C, state, None, None, lens, softplus=False)
    _, after = call(x, dt, B, C, state, lens)
    bad = (after - s).abs() > 2.0 ** -18 * smag
    assert not bad.any(), f"{int(bad.sum())} off, worst {float(((after - s).abs() / smag).max()):.3g}"


@pytest.mark.parametrize("x0,d0", [(20000.0, 10.0), (60000.0, 1e30), (1.0, 0.5)])
def test_nothing_after_large_values(x0, d0):
    """Tokens whose B is zero leave no state, however large their d x; what follows is zero, not NaN."""
    T, H, P, N = 256, 2, 32, 64
    x, B = torch.zeros(T, H, P).half(), torch.zeros(T, 1, N).half()
    x[:64] = x0
    out, after = call(x, torch.full((T, H), d0), B, torch.ones(T, 1, N).half(), torch.zeros(1, H, P, N), [T])
    assert not out.any() and not after.any()
    x[200:], B[200:] = 1.0, 0.5                                                 # and what comes then is there in full
    _, after = call(x, torch.full((T, H), min(d0, 1.0)), B, torch.ones(T, 1, N).half(), torch.zeros(1, H, P, N), [T])
    ref = 56 * 0.5 * min(d0, 1.0)
    assert ((after - ref).abs() <= 2.0 ** -18 * ref).all()


def off(got, ref, tol, what):
    bad = (got - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float(((got - ref).abs() / tol).max()):.3g} of the bound"


@pytest.mark.parametrize("lens", [[100], [900, 70]])
def test_small_values_beside_a_large_one_that_a_sum_leaves_out(lens):
    """fp16 rows: a factor may be off by 2^-39 of the largest of its kind, also where that one is multiplied by zero."""
    H, P, N = 2, 32, 64
    x, dt, B, C, state = ordinary(lens, H, P, N)
    A_log, rel, tiny = torch.full((H,), -200.0), *lm.half_step(torch.float16)
    total = lambda t: torch.stack([t[a:b].double().abs().sum(0) for a, b in lm.slices(lens)])          # over each sequence

    # d x of a token, its B zero in half the columns: those states
    X, dT, b = x.clone(), dt.clone(), B.clone()
    X[5], dT[5], b[5, :, :32] = 30000.0, 200.0, 0
    _, _, s, smag = lm.scan(X, dT, A_log, b, C, state, None, None, lens, softplus=False)
    _, after = call(X, dT, b, C, state, lens)
    off(after, s, 2.0 ** -18 * smag + 2.0 ** -39 * 6e6 * total(b)[:, :, None], "state")

    # a state that C leaves out
    S, c = state.clone(), C.clone()
    S[..., 7], c[..., 7] = 1e8, 0
    y, mag, _, _ = lm.scan(x, dt, A_log, B, c, S, None, None, lens, softplus=False)
    out, _ = call(x, dt, B, c, S, lens)
    off(out, y, rel * (1 + 2.0 ** -7) * y.abs() + 2.0 ** -16 * mag + tiny + 2.0 ** -39 * 1e8 * c.double().abs().sum(-1)[..., None], "state's out")

    # a score whose x is zero
    X, dT = x.clone(), dt.clone()
    X[3], dT[3] = 0, 1e5
    y, mag, _, _ = lm.scan(X, dT, A_log, B, C, state, None, None, lens, softplus=False)
    out, _ = call(X, dT, B, C, state, lens)
    score = 1e5 * (C.double() @ B[3, 0].double()).abs().amax()
    off(out, y, rel * (1 + 2.0 ** -7) * y.abs() + 2.0 ** -16 * mag + tiny + 2.0 ** -39 * score * total(x)[:1], "scores' out")


@pytest.mark.parametrize("large", [1e30, 1e35])
def test_outputs_that_leave_a_very_large_state_out(large):
    """fp16 rows: C is zero, so out is x's share alone (zero without D), however large the state and small the scores."""
    T, H, P, N = 100, 2, 32, 64
    gen = torch.Generator().manual_seed(0)
    x, B = torch.randn(T, H, P, generator=gen).half(), torch.randn(T, 1, N, generator=gen).half()
    state = torch.full((1, H, P, N), large)
    for D in (None, torch.tensor([2.0 ** -30, 1.0], device=DEV)):
        out, after = call(x, torch.zeros(T, H), B, torch.zeros(T, 1, N).half(), state, [T], D=D)
        ref = torch.zeros(T, H, P) if D is None else D.cpu().double()[:, None] * x.double()
        assert ((out - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -25).all() and torch.equal(after, state.double())


def test_a_very_large_state_that_decays():
    """e^-80 of 1e35, within a chunk and in the next: 1.8 C. (An exponent of 80 in fp32 is off by 80 2^-21 at most: 4e-5.)"""
    T, H, P, N = 100, 1, 32, 64
    x, B, C = torch.zeros(T, H, P).half(), torch.zeros(T, 1, N).half(), torch.zeros(T, 1, N).half()
    C[20:, 0, 3] = 1
    dt = torch.zeros(T, H)
    dt[10:20] = 8.0
    state = torch.full((1, H, P, N), 1e35, device=DEV)
    out = ops.selective_scan_prefill(x.to(DEV), dt.to(DEV), torch.zeros(H, device=DEV), B.to(DEV), C.to(DEV), state,
                                     cu_seqlens=lm.offsets([T], DEV), softplus=False).cpu().double()
    ref = float(torch.tensor(1e35, dtype=torch.float32)) * torch.exp(torch.tensor(-80.0, dtype=torch.float64))
    assert not out[:20].any() and ((out[20:] - ref).abs() <= (2.0 ** -11 + 4.1e-5) * ref).all()
    assert ((state.cpu().double() - ref).abs() <= 4.1e-5 * ref).all()
