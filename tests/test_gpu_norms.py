"""ops.gated_norm and ops.residual_norm against their formulas in 64 bits.

Tolerance: the mean of squares is a sum in fp32 of at most 16384 terms, in partial sums of 16 per lane and a tree, off by
at most 32 roundings of 2^-24; SiLU by (2 + |z|) 2^-22 of itself; the factors by a few roundings each. So an output of a norm
is off by (64 + 8 max|z|) 2^-24 of itself, and by half a step of its type; a residual by 64 2^-24 of its terms'
magnitudes, and half a step of its type. The second norm's input has the first one's error."""
import pytest
import torch

import layer_math as lm
from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
COLS = [1, 3, 8, 64, 100, 512, 520, 2048, 2051, 4096, 5120, 8200, 16384, 16383]


def check(got, ref, rel32, what, mag=None):
    got = got.cpu()
    assert torch.isfinite(got.double()).all(), what
    rel, tiny = lm.half_step(got.dtype) if got.dtype is not torch.float32 else (2.0 ** -24, 2.0 ** -149)
    bad = (got.double() - ref).abs() > rel * (1 + 2.0 ** -7) * ref.abs() + rel32 * (ref.abs() if mag is None else mag) + tiny
    assert not bad.any(), f"{what}: {int(bad.sum())} values off"


def rnd(gen, *shape):
    return torch.randn(*shape, generator=gen)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", COLS)
def test_gated(cols, dtype):
    gen = torch.Generator().manual_seed(cols)
    x, z, w = rnd(gen, 5, cols).to(dtype), (3 * rnd(gen, 5, cols)).to(dtype), 1 + 0.2 * rnd(gen, cols)
    rel = (64 + 8 * float(z.abs().max())) * 2.0 ** -24
    for first in (True, False):
        out = ops.gated_norm(x.to(DEV), z.to(DEV), w.to(DEV), gate_first=first)
        check(out, lm.gated(x, z, w, 1, first), rel, f"first {first}")
    check(ops.gated_norm(x.to(DEV), None, w.to(DEV)), lm.gated(x, None, w), rel, "no gate")


@pytest.mark.parametrize("cols,groups", [(64, 8), (40, 5), (5120, 8), (36, 4), (32768, 2), (7, 7)])
def test_groups(cols, groups):
    gen = torch.Generator().manual_seed(cols)
    x, z, w = rnd(gen, 9, cols).half(), rnd(gen, 9, cols).half(), 1 + 0.2 * rnd(gen, cols)
    x[:, :cols // groups] *= 100
    for first in (True, False):
        out = ops.gated_norm(x.to(DEV), z.to(DEV), w.to(DEV), groups=groups, gate_first=first, eps=1e-3)
        check(out, lm.gated(x, z, w, groups, first, 1e-3), 128 * 2.0 ** -24, "out")


@pytest.mark.parametrize("dtype,res", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                       (torch.float16, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("cols", COLS)
def test_residual(cols, dtype, res):
    gen = torch.Generator().manual_seed(cols)
    x, r = rnd(gen, 5, cols).to(dtype), (3 * rnd(gen, 5, cols)).to(res)
    w, post, sc = 1 + 0.2 * rnd(gen, cols), 0.5 + 0.1 * rnd(gen, cols), 0.3 + 0.1 * rnd(gen, cols)
    for p, s in ((post, sc), (None, 0.22), (post, -1.5), (None, sc)):
        ref, new, mag = lm.residual(x, r, w, p, s)
        out, ro = ops.residual_norm(x.to(DEV), r.to(DEV), w.to(DEV), post_weight=None if p is None else p.to(DEV),
                                    scale=s.to(DEV) if isinstance(s, torch.Tensor) else s)
        check(ro, new, 64 * 2.0 ** -24, "residual", mag)
        # out_c is off by what r_c is off by, times w_c / rms(r), besides its own roundings
        f = (w.double().abs() / (new.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt())
        check(out, ref, 2.0 ** -17, "out", ref.abs() / 2 + mag * f / 2)


def test_rows_of_any_layout():
    gen = torch.Generator().manual_seed(3)
    for cols in (24, 37, 600):
        wide = rnd(gen, 3, 7, cols + 9).half()
        x, z = wide[..., 3:3 + cols], rnd(gen, 3, 7, cols).half()
        w = 1 + 0.2 * rnd(gen, cols)
        ref = lm.gated(x, z, w)
        gx = wide.to(DEV)
        out = ops.gated_norm(gx[..., 3:3 + cols], z.to(DEV), w.to(DEV))
        assert out.shape == x.shape
        check(out, ref, 128 * 2.0 ** -24, "out")
        inplace = gx[0]
        same = ops.gated_norm(inplace[:, 3:3 + cols], z.to(DEV)[0], w.to(DEV), out=inplace[:, 3:3 + cols])
        assert torch.equal(same, out[0]) and torch.equal(inplace[:, :3].cpu(), wide[0, :, :3])
        assert torch.equal(inplace[:, 3 + cols:].cpu(), wide[0, :, 3 + cols:])


def test_in_place():
    gen = torch.Generator().manual_seed(4)
    for cols in (64, 700, 5120):
        x, r, w = rnd(gen, 6, cols).half().to(DEV), rnd(gen, 6, cols).to(DEV), (1 + 0.2 * rnd(gen, cols)).to(DEV)
        out, ro = ops.residual_norm(x, r, w, post_weight=w, scale=0.5)
        a, b = x.clone(), r.clone()
        o2, r2 = ops.residual_norm(a, b, w, post_weight=w, scale=0.5, out=a, residual_out=b)
        assert o2 is a and r2 is b and torch.equal(a, out) and torch.equal(b, ro)
        z = rnd(gen, 6, cols).half().to(DEV)
        out = ops.gated_norm(x, z, w)
        assert torch.equal(ops.gated_norm(x, z, w, out=z), out)


def test_rows_none_zero_and_not_finite():
    w = torch.ones(40, device=DEV)
    x = torch.zeros(4, 40, dtype=torch.float16, device=DEV)
    assert ops.gated_norm(x[:0], x[:0], w).shape == (0, 40) and ops.residual_norm(x[:0], x[:0], w)[0].shape == (0, 40)
    assert (ops.gated_norm(x, x, w) == 0).all() and (ops.residual_norm(x, x, w)[0] == 0).all()
    x = torch.randn(4, 40, device=DEV).half()
    x[1, 7] = float("nan")
    out, r = ops.residual_norm(x, x, w, post_weight=w)
    assert out[1].isnan().all() and out[[0, 2, 3]].isfinite().all() and r[[0, 2, 3]].isfinite().all()
    assert ops.gated_norm(x, x, w)[1].isnan().all()


def test_rows_past_32_bits_and_many_in_turn():
    """2.2 * 10^9 values; and more rows than are resident at once, in several turns, in place."""
    cols, rows = 8192, (1 << 18) + 100
    gen = torch.Generator().manual_seed(5)
    w = 1 + 0.2 * rnd(gen, cols)
    x = torch.zeros(rows, cols, dtype=torch.float16, device=DEV)
    tail = rnd(gen, 3, cols).half()
    x[-3:] = tail.to(DEV)
    check(ops.gated_norm(x, x, w.to(DEV), out=x)[-3:], lm.gated(tail, tail, w), 128 * 2.0 ** -24, "gated")
    x[-3:] = tail.to(DEV)
    out, r = ops.residual_norm(x, x, w.to(DEV), scale=0.5, out=x)
    ref, new, mag = lm.residual(tail, tail, w, None, 0.5)
    check(out[-3:], ref, 2.0 ** -17, "out")
    check(r[-3:], new, 64 * 2.0 ** -24, "residual", mag)
    for n in (64, 65, 1000):
        x, z = rnd(gen, 20000, n).half(), rnd(gen, 20000, n).half()
        wn = 1 + 0.2 * rnd(gen, n)
        check(ops.gated_norm(x.to(DEV), z.to(DEV), wn.to(DEV)), lm.gated(x, z, wn), 128 * 2.0 ** -24, f"{n}")
        out, r = ops.residual_norm(x.to(DEV), z.to(DEV), wn.to(DEV), post_weight=wn.to(DEV))
        check(r, lm.residual(x, z, wn, wn)[1], 64 * 2.0 ** -24, f"{n}", lm.residual(x, z, wn, wn)[2])


@pytest.mark.parametrize("cols", [2, 7, 9, 15, 63, 65, 127, 129, 511, 513, 1023, 1025, 2047, 2049, 4095, 4097, 8191, 8193, 16381])
def test_widths_that_end_inside_a_lane(cols):
    """The last lane's columns overlap its neighbour's: what lies beside the rows stays, in place too."""
    gen = torch.Generator().manual_seed(cols)
    wide = rnd(gen, 70, cols + 10).half()
    x, z, w = wide[:, 5:5 + cols], rnd(gen, 70, cols).half(), 1 + 0.2 * rnd(gen, cols)
    g = wide.to(DEV)
    out = ops.gated_norm(g[:, 5:5 + cols], z.to(DEV), w.to(DEV), out=g[:, 5:5 + cols])
    check(out, lm.gated(x, z, w), 128 * 2.0 ** -24, "gated")
    assert torch.equal(g[:, :5].cpu(), wide[:, :5]) and torch.equal(g[:, 5 + cols:].cpu(), wide[:, 5 + cols:])
    for res in (torch.float16, torch.float32):
        r = rnd(gen, 70, cols + 10).to(res)
        ref, new, mag = lm.residual(x, r[:, 3:3 + cols], w, w, 0.5)
        g, gr = wide.to(DEV), r.to(DEV)
        out, ro = ops.residual_norm(g[:, 5:5 + cols], gr[:, 3:3 + cols], w.to(DEV), post_weight=w.to(DEV), scale=0.5,
                                    out=g[:, 5:5 + cols], residual_out=gr[:, 3:3 + cols])
        check(ro, new, 64 * 2.0 ** -24, "residual", mag)
        f = (w.double().abs() / (new.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt())
        check(out, ref, 2.0 ** -17, "out", ref.abs() / 2 + mag * f / 2)
        assert torch.equal(gr[:, :3].cpu(), r[:, :3]) and torch.equal(gr[:, 3 + cols:].cpu(), r[:, 3 + cols:])
        assert torch.equal(g[:, :5].cpu(), wide[:, :5]) and torch.equal(g[:, 5 + cols:].cpu(), wide[:, 5 + cols:])


@pytest.mark.parametrize("n,groups", [(8, 8), (9, 5), (13, 40), (64, 3), (100, 7), (3, 11)])
def test_small_groups(n, groups):
    gen = torch.Generator().manual_seed(n)
    x, z, w = rnd(gen, 300, n * groups).bfloat16(), rnd(gen, 300, n * groups).bfloat16(), 1 + 0.2 * rnd(gen, n * groups)
    for first in (True, False):
        check(ops.gated_norm(x.to(DEV), z.to(DEV), w.to(DEV), groups=groups, gate_first=first), lm.gated(x, z, w, groups, first),
              128 * 2.0 ** -24, "out")
