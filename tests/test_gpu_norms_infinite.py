"""Infinite values in the norms' rows: by the formulas the mean of squares is infinite, so the row's other outputs are zero and the
infinite column's is NaN (inf * 0), wherever in the row it lies."""
import pytest
import torch

from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# widths whose lanes all have columns, whose last lanes have none, and whose last columns overlap a neighbour's
WIDTHS = [3, 8, 12, 40, 64, 100, 128, 520, 640, 1000, 1024, 1500, 2048, 2051, 3000, 5119, 5120, 8200, 16381, 16384]


def columns(n):
    return sorted({0, min(5, n - 1), n // 2, max(n - 10, 0), max(n - 3, 0), n - 1})


def ones(rows, cols, at, dtype):
    x = torch.ones(rows, cols, dtype=dtype)
    for r, c in enumerate(at):
        x[r, c] = float("inf") if r % 2 == 0 else float("-inf")
    return x.to(DEV)


def only_there(out, at):
    """NaN in row r's column at[r], zero in the others."""
    out = out.cpu().float()
    for r, c in enumerate(at):
        rest = torch.cat([out[r, :c], out[r, c + 1:]])
        assert out[r, c].isnan() and (rest == 0).all(), f"column {c}: {int(rest.isnan().sum())} others are NaN"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", WIDTHS)
def test_gated(n, dtype):
    at = columns(n)
    x, w = ones(len(at), n, at, dtype), torch.ones(n, device=DEV)
    z = torch.ones_like(x)
    for first in (True, False):
        only_there(ops.gated_norm(x, z, w, gate_first=first), at)
    only_there(ops.gated_norm(x, None, w), at)


@pytest.mark.parametrize("n", [5, 8, 20, 80, 100, 640, 1000])
def test_groups(n):
    """A group's infinity stays in its group."""
    at = columns(n)
    x = torch.cat([torch.ones(len(at), n, dtype=torch.float16, device=DEV), ones(len(at), n, at, torch.float16)], 1)
    out = ops.gated_norm(x, torch.ones_like(x), torch.ones(2 * n, device=DEV), groups=2)
    assert out[:, :n].isfinite().all()
    only_there(out[:, n:], at)


@pytest.mark.parametrize("res", [torch.float16, torch.float32])
@pytest.mark.parametrize("n", WIDTHS)
def test_residual(n, res):
    at = columns(n)
    w, one = torch.ones(n, device=DEV), torch.ones(len(at), n, device=DEV)
    x = ones(len(at), n, at, torch.float16)
    out, r = ops.residual_norm(x, one.to(res), w)
    only_there(out, at)
    assert (r.cpu().isinf().sum(1) == 1).all() and not r.isnan().any()
    out, r = ops.residual_norm(one.half(), ones(len(at), n, at, res), w, scale=0.5)
    only_there(out, at)
    _, r = ops.residual_norm(x, torch.zeros_like(one).to(res), w, post_weight=w)      # (x's norm: zeros and a NaN)
    only_there(r, at)


@pytest.mark.parametrize("n", [40, 1000, 5120])
def test_squares_past_fp32(n):
    """bf16 rows of finite values whose squares are infinite in fp32 come out as zeros, those of 2^50 as ones."""
    x, w = torch.full((3, n), 2.0 ** 70, dtype=torch.bfloat16, device=DEV), torch.ones(n, device=DEV)
    x[1] = 2.0 ** 50
    zero, one = torch.zeros(n, device=DEV), torch.ones(n, device=DEV)
    for out in (ops.gated_norm(x, None, w), ops.residual_norm(x, torch.zeros_like(x), w)[0]):
        assert torch.equal(out[0].float(), zero) and torch.equal(out[1].float(), one) and torch.equal(out[2].float(), zero)
