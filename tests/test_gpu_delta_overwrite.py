"""Keys whose value is overwritten: a state of large values, beta 1 and no decay, each query the key of its own token. Of the
output, scale S q, the old value cancels and v is left, to the bit here: keys are unit vectors, v whole numbers of 7 bits
and the state whole numbers of 20, so nothing is rounded by arithmetic that keeps 22 bits or more of its factors. (Old
values are odd multiples of 1 beside 2^10 and 2^19: two parts of 8 bits would lose the 1.)
"""
import numpy as np
import pytest
import torch

from test_gpu_delta import DEV, gpu, prefill

pytestmark = pytest.mark.gpu

# sequences' lengths, heads and dimensions: 16, 32 and 64 value columns to a workgroup
SHAPES = [([70, 3, 64], 1, 2, 128, 64), ([40], 2, 2, 64, 48), ([70, 20, 64], 16, 64, 128, 64), ([130, 7, 33], 8, 64, 64, 48),
          ([70, 20, 64, 100, 13], 16, 64, 128, 64), ([33] * 5, 64, 64, 64, 80)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_overwritten_keys(shape, dtype):
    lens, Hk, Hv, Dk, Dv = shape
    T, rng = sum(lens), np.random.default_rng(sum(lens) + Dv)
    keys = torch.from_numpy(rng.integers(0, Dk, (T, Hk)))
    k = torch.nn.functional.one_hot(keys, Dk).to(dtype)
    v = torch.from_numpy(rng.integers(-100, 101, (T, Hv, Dv))).to(dtype)
    sign = lambda: torch.from_numpy(rng.choice([-1.0, 1.0], (len(lens), Hv, Dv, Dk)))
    state = (2.0 ** 19 * sign() + 2.0 ** 10 * sign() + sign()).float()
    x = {"q": k, "k": k, "v": v, "g": torch.zeros(T, Hv), "beta": torch.ones(T, Hv), "state": state}
    want, t = state.clone(), 0
    head = keys.repeat_interleave(Hv // Hk, 1)
    for b, n in enumerate(lens):
        for _ in range(n):
            want[b, torch.arange(Hv), :, head[t]] = v[t].float()
            t += 1
    d = gpu(x)
    out = prefill(d, lens, scale=1.0)
    assert torch.equal(out.cpu(), v)
    assert torch.equal(d["state"].cpu(), want)
