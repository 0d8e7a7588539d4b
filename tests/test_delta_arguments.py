"""What the gated delta rule's entry points make of arguments that are no tensors, or have too few dimensions: the errors
that every other argument's check gives. No GPU needed."""
import pytest
import torch

from dfssm import ops

ROW = torch.zeros(1, 1, 128, dtype=torch.float16)
ARGS = {"q": ROW, "k": ROW, "v": ROW[..., :64], "g": torch.zeros(1, 1), "beta": torch.zeros(1, 1),
        "state": torch.zeros(1, 1, 64, 128)}
CU = torch.tensor([0, 1], dtype=torch.int32)
BAD = [None, 1.0, [[0.0]], torch.zeros(()), "q"]


@pytest.mark.parametrize("bad", BAD, ids=["none", "number", "list", "scalar", "text"])
@pytest.mark.parametrize("name", list(ARGS))
def test_no_tensor(name, bad):
    args = {**ARGS, name: bad}
    batch = {n: t.unsqueeze(0) if n != "state" and isinstance(t, torch.Tensor) else t for n, t in args.items()}
    with pytest.raises((TypeError, ValueError)):
        ops.gated_delta_step(**args)
    with pytest.raises((TypeError, ValueError)):
        ops.gated_delta_prefill(**args)
    with pytest.raises((TypeError, ValueError)):
        ops.gated_delta_prefill(**batch)
    for cu in (CU, None, 3):
        with pytest.raises((TypeError, ValueError)):
            ops.gated_delta_prefill(**args, cu_seqlens=cu)


def test_no_tensor_out():
    batch = {n: t.unsqueeze(0) if n != "state" else t for n, t in ARGS.items()}
    with pytest.raises(TypeError):
        ops.gated_delta_prefill(**batch, out=3)
    with pytest.raises(TypeError):
        ops.gated_delta_prefill(**batch, out=torch.zeros(1, 1, 1, 64, dtype=torch.float16))   # on the host


@pytest.mark.parametrize("bad", BAD[:3] + BAD[4:], ids=["none", "number", "list", "text"])
def test_no_tensor_draw(bad):
    with pytest.raises(TypeError):
        ops.sample_filtered(bad, torch.zeros(1))
    with pytest.raises(TypeError):
        ops.sample_filtered(torch.zeros(1, 8), bad)
