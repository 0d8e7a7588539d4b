"""What the gated delta rule's and the filtered draw's entry points refuse before any launch. No GPU needed."""
import ctypes

import pytest
import torch

from dfssm import _C, ops


def _delta(**kw):
    base = dict(q=16, k=16, v=16, g=16, beta=16, state=16, state_out=16, slots=0, cu_seqlens=0, out=16,
                ld_q=128, ld_k=128, ld_v=64, ld_g=1, ld_beta=1, ld_out=64, n_tokens=2, n_seq=2, n_slots=2,
                k_heads=1, v_heads=1, k_dim=128, v_dim=64, type=0, l2norm=0, scale=1.0)
    base.update(kw)
    return _C.Delta(*[base[f] for f, _ in _C.Delta._fields_])


BAD = [({"q": 0}, -1), ({"state": 0}, -1), ({"out": 0}, -1), ({"beta": 0}, -1), ({"k_dim": 96}, -2), ({"v_dim": 24}, -2),
       ({"v_dim": 272}, -2), ({"v_dim": 0}, -2), ({"k_heads": 0}, -2), ({"k_heads": 2}, -2), ({"type": 2}, -2),
       ({"q": 8}, -4), ({"state_out": 8}, -4), ({"ld_v": 68}, -4), ({"n_seq": -1}, -5), ({"n_slots": -1}, -5)]


@pytest.mark.parametrize("kw,rc", BAD)
def test_delta(kw, rc):
    L = _C.lib()
    assert L.dfssm_gated_delta_step(_delta(**kw), None) == rc
    assert L.dfssm_gated_delta_prefill(_delta(**kw), None, None) == rc


def test_delta_counts():
    L = _C.lib()
    assert L.dfssm_gated_delta_step(None, None) == -1
    assert L.dfssm_gated_delta_step(_delta(n_tokens=3), None) == -5          # one token per sequence
    assert L.dfssm_gated_delta_step(_delta(cu_seqlens=16), None) == -5
    assert L.dfssm_gated_delta_prefill(_delta(n_tokens=3), None, None) == -5       # 3 tokens of 2 equal sequences
    assert L.dfssm_gated_delta_step(_delta(n_seq=0, n_tokens=0), None) == 0  # nothing to do
    assert L.dfssm_gated_delta_prefill(_delta(n_seq=0), None, None) == 0
    many = _delta(n_tokens=200)
    assert L.dfssm_gated_delta_workspace_bytes(many) > 0 and L.dfssm_gated_delta_workspace_bytes(_delta()) == 0
    assert L.dfssm_gated_delta_prefill(many, None, None) == -1 and L.dfssm_gated_delta_prefill(many, 8, None) == -4


def test_draw():
    L = _C.lib()
    f = _C.Filter(0, 0, 0, 0, 1.0, 0, 1.0, 0.0)
    call = lambda logits=16, type=0, ld=8, batch=2, vocab=8, u=16, flt=f, nxt=16: L.dfssm_sample_filtered(
        logits, type, ld, batch, vocab, u, flt, nxt, None, None)
    assert call(logits=None) == -1 and call(u=None) == -1 and call(nxt=None) == -1 and call(flt=None) == -1
    assert call(type=3) == -2 and call(vocab=0) == -2 and call(vocab=262145, ld=262145) == -2 and call(ld=7) == -2
    assert call(batch=-1) == -3 and call(batch=0) == 0


def test_host_tensors():
    x = torch.zeros(1, 1, 128, dtype=torch.float16)
    f = torch.zeros(1, 1)
    with pytest.raises(TypeError):
        ops.gated_delta_step(x, x, x[..., :64], f, f, torch.zeros(1, 1, 64, 128))
    with pytest.raises(TypeError):
        ops.gated_delta_prefill(x, x, x[..., :64], f, f, torch.zeros(1, 1, 64, 128),
                                cu_seqlens=torch.tensor([0, 1], dtype=torch.int32))
    with pytest.raises(TypeError):
        ops.sample_filtered(torch.zeros(1, 8), torch.zeros(1))


def test_overlapping_rows_of_out():
    L = _C.lib()
    assert L.dfssm_gated_delta_step(_delta(ld_out=56), None) == -2
    assert L.dfssm_gated_delta_prefill(_delta(ld_out=56, n_tokens=64), None, None) == -2


def test_numbers_of_settings():
    """A top_k past 32 bits means all, not what is left of it there; a fraction is refused."""
    value = lambda x: ops._per_row(x, torch.int32, "top_k", 2, None, [])
    assert value(7) == (7, 0) and value(2**32 + 5) == (2**31 - 1, 0) and value(-2**40) == (-1, 0)
    with pytest.raises(TypeError):
        value(2.5)
