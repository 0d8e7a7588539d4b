"""Settings that are NaN: temperature takes the most probable token, top_p limits nothing, min_p leaves the most probable
token. As numbers and per row, in rows whose list is short, whose masses matter, and that have infinities. (Against the
draw on the sorted row in 64 bits, see test_gpu_draw.py.)"""
import itertools

import pytest
import torch

from test_gpu_draw import run_check

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.mark.parametrize("as_tensors", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("infinite", [False, True])
def test_nan_settings(infinite, dtype, as_tensors):
    gen = torch.Generator().manual_seed(3)
    logits = (2 * torch.randn(5, 6001, generator=gen)).to(dtype)
    if infinite:
        logits[:, 17::999] = float("inf")
    u = [0.0, 0.2, 0.5, 0.9, 0.999]
    for T, k, tp, mp in itertools.product([0.8, NAN], [0, 20], [0.9, 1.0, NAN], [0.0, 0.05, NAN]):
        if T != T or tp != tp or mp != mp:
            run_check(logits, u, T, k, tp, mp, as_tensors)
