"""gated_delta_prefill over more chunks than one pass holds, with empty sequences between, before and behind those with
tokens: an empty one's chunk numbers may lie behind the pass that passes its state on. Against the recurrence in
64 bits (tolerances: test_gpu_delta.py).
"""
import pytest
import torch

from dfssm import _C
from test_gpu_delta import DEV, check, prefill, recurrence

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_empty_sequences_in_several_passes(dtype):
    lens, Hk, Hv, Dk, Dv = [0, 7001, 0, 5000, 0, 0], 2, 512, 128, 64
    T, n = sum(lens), len(lens)
    bytes_of = lambda tokens: _C.lib().dfssm_gated_delta_workspace_bytes(_C.Delta(
        n_tokens=tokens, n_seq=n, n_slots=n, k_heads=Hk, v_heads=Hv, k_dim=Dk, v_dim=Dv,
        type=0 if dtype is torch.float16 else 1))
    assert bytes_of(T) == bytes_of(2 * T)                              # the workspace holds a part of the chunks
    gen = torch.Generator(DEV).manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    x = {"q": rand(T, Hk, Dk).to(dtype), "k": rand(T, Hk, Dk).to(dtype), "v": rand(T, Hv, Dv).to(dtype),
         "g": -torch.nn.functional.softplus(2 * rand(T, Hv) - 3), "beta": torch.sigmoid(rand(T, Hv)),
         "state": 0.3 * rand(n, Hv, Dv, Dk)}
    before, so = x["state"].clone(), torch.full_like(x["state"], 7.0)
    out = prefill(x, lens, l2norm=True, state_out=so)
    assert torch.equal(x["state"], before)
    assert torch.equal(prefill(x, lens, l2norm=True), out) and torch.equal(x["state"], so)
    empty = [b for b in range(n) if not lens[b]]
    assert torch.equal(so[empty], before[empty])
    heads = [0, Hv - 1]                                                # one of each key head
    sub = {"q": x["q"], "k": x["k"], "state": before[:, heads], **{m: x[m][:, heads] for m in ("v", "g", "beta")}}
    ref, ref_state = recurrence({m: t.cpu() for m, t in sub.items()}, lens, True)
    check(out[:, heads], ref, "out")
    check(so[:, heads], ref_state, "state")
