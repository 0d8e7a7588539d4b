"""out of gated_delta_prefill without offsets: v's shape, and what is refused."""
import pytest
import torch

from dfssm import ops
from test_gpu_delta import DEV, gpu, make

pytestmark = pytest.mark.gpu


def test_out_of_a_batch():
    B, T = 2, 20
    x = make([T] * B, 1, 2, 64, 16, torch.float16)
    d = {n: t if n == "state" else t.view(B, T, *t.shape[1:]) for n, t in gpu(x).items()}
    before = d["state"].clone()
    want = ops.gated_delta_prefill(**d, l2norm=True)
    d["state"].copy_(before)
    out = torch.empty_like(want)
    assert ops.gated_delta_prefill(**d, l2norm=True, out=out) is out and torch.equal(out, want)
    for bad in (out.view(T, B, 2, 16), out.view(B, T, 1, 32), out[:, ::2], out.flatten(0, 1)):
        with pytest.raises(ValueError):
            ops.gated_delta_prefill(**d, out=bad)
    with pytest.raises(TypeError):
        ops.gated_delta_prefill(**d, out=out.bfloat16())
    assert torch.zeros(1, device=DEV).item() == 0
