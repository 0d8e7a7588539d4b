"""Tokens that are alike: rows that are one row expanded over all tokens (a stride of zero), and keys that all are the same,
with beta up to 2 (each token then undoes the one before it), where a chunk's triangle is as dense as it gets. Against the
recurrence in 64 bits (tolerances: test_gpu_delta.py)."""
import pytest
import torch

from test_gpu_delta import ATOL, check, gpu, make, prefill, recurrence

from dfssm import ops

pytestmark = pytest.mark.gpu
# With beta |k|^2 = 2 and one key a token takes the state along it times -1, so no rounding dies out. In a chunk's equations
# u_i = beta (v_i - ..) - sum_j<i A_ij u_j, |A_ij| <= 2, every A_ij has an error of its own: two exponentials within 1 ulp and
# three products, of a standard deviation of 2^-23 sqrt(2 / 3 + 3 / 12) = 2^-23. Each adds to the state, with a sign of its
# own: sqrt(64 63 / 2) 2 2^-23 |u| a chunk, and |u| <= 2 |S'k| + 2 |v| is at most 3 of the state's largest value: 2^-14.9 of it.
# Five standard deviations over three chunks: 2^-14.9 5 sqrt(3) = 2^-11.8, taken as 2^-11.5. (A chunk's form in fp32
# throughout is off by 2^-14.7 in this test's state; token by token by 2^-21.)
UNDAMPED = 2.0 ** -11.5
SHAPES = [([150, 20, 0, 64], 1, 2, 128, 64), ([70, 1, 40], 16, 64, 64, 64), ([70, 20, 64, 1, 9], 16, 64, 128, 64), ([5], 1, 2, 64, 32)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=["16", "32", "64", "tokens"])
@pytest.mark.parametrize("names", ["q", "k", "v", "g beta", "q k v g beta"])
def test_expanded(names, shape, dtype):
    lens, Hk, Hv, Dk, Dv = shape
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=13)
    d = gpu(x)
    for n in names.split():
        x[n] = x[n][:1].expand(x[n].shape)
        d[n] = d[n][:1].expand(d[n].shape)
        assert d[n].stride(0) == 0
    ref, ref_state = recurrence(gpu(x), lens, True)
    check(prefill(d, lens, l2norm=True), ref, "out")
    check(d["state"], ref_state.cpu(), "state")


def near(got, want, what, extra):
    """check() with `extra` more of the head's largest value."""
    got, half = got.cpu(), torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    dims = (-1, -2) if got.dtype == torch.float32 else (0, 2)
    top = want.abs().amax(dims, keepdim=True)
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    bad = err > half * want.abs() * (1 + 2.0 ** -7) + (ATOL + extra) * top + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {float((err / top).max()):.3g} of the largest"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES[:3], ids=["16", "32", "64"])
@pytest.mark.parametrize("beta", [1.0, 1.5, 2.0])
def test_one_key(beta, shape, dtype):
    """Beside what holds for any key, with beta = 2 an error of the key's norm does not die out. The norm's factor r = rsq(sum k^2 + 1e-6) is off by at most 2^-23 (1 ulp) and half of
    the sum's error, 12 additions of 2^-24 each: 2^-23 (1 + 3) = 2^-21. |k|^2 = sum k^2 r^2 is off by twice that, 2 |k|^2 by four
    times, 2^-19 a token; so after n tokens n 2^-19 of the largest value, on top of the usual. (Products and sums in
    fp32 with a root and a quotient for the norm are off by up to 2.4e-5 here after 150.)"""
    lens, Hk, Hv, Dk, Dv = shape
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=17)
    x["k"] = x["k"][:1].expand(x["k"].shape).clone()
    x["beta"].fill_(beta)
    x["g"] = x["g"] * 0.01
    ref, ref_state = recurrence(gpu(x), lens, True)
    d = gpu(x)
    extra = max(lens) * 2.0 ** -19 + UNDAMPED if beta == 2.0 else 0.0
    near(prefill(d, lens, l2norm=True), ref, "out", extra)
    near(d["state"], ref_state.cpu(), "state", extra)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES[:3], ids=["16", "32", "64"])
@pytest.mark.parametrize("beta", [1.0, 1.5, 2.0])
def test_one_unit_key(beta, shape, dtype):
    """The same with a key whose norm is 1 to the bit."""
    lens, Hk, Hv, Dk, Dv = shape
    x = make(lens, Hk, Hv, Dk, Dv, dtype, seed=23, l2norm=False)
    x["k"].zero_()
    x["k"][..., 5] = 1.0
    x["beta"].fill_(beta)
    x["g"] = x["g"] * 0.01
    ref, ref_state = recurrence(gpu(x), lens, False)
    d = gpu(x)
    extra = UNDAMPED if beta == 2.0 else 0.0
    near(prefill(d, lens), ref, "out", extra)
    near(d["state"], ref_state.cpu(), "state", extra)


def test_step_expanded():
    x = make([1] * 6, 1, 2, 64, 32, torch.float16, seed=19)
    d = gpu(x)
    for n in ("q", "k", "v", "g", "beta"):
        x[n], d[n] = x[n][:1].expand(x[n].shape), d[n][:1].expand(d[n].shape)
    ref, ref_state = recurrence(x, [1] * 6, True)
    out = ops.gated_delta_step(d["q"], d["k"], d["v"], d["g"], d["beta"], d["state"], l2norm=True)
    check(out, ref, "out")
    check(d["state"], ref_state, "state")
