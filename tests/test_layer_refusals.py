"""What the entry points of the operators between a layer's projections refuse before any launch. No GPU needed."""
import ctypes

import pytest
import torch

from dfssm import _C, ops


def fill(cls, base, kw):
    return cls(*[dict(base, **kw)[f] for f, _ in cls._fields_])


CONV = dict(x=16, weight=16, bias=0, state=16, state_out=16, slots=0, cu_seqlens=0, out=32, ld_x=8, ld_out=8, n_tokens=2,
            n_seq=2, n_slots=2, channels=8, width=4, type=0, silu=1)
SCAN = dict(x=16, dt=16, B=16, C=16, A_log=16, D=0, dt_bias=0, state=16, state_out=16, slots=0, cu_seqlens=0, out=32, ld_x=64,
            ld_dt=1, ld_B=128, ld_C=128, ld_out=64, n_tokens=2, n_seq=2, n_slots=2, heads=1, groups=1, dim=64, cols=128,
            type=0, dt_type=0, softplus=1)
GATED = dict(x=16, gate=0, weight=16, out=16, ld_x=8, ld_gate=8, ld_out=8, rows=2, cols=8, groups=1, type=0, gate_first=1,
             eps=1e-5)
RESIDUAL = dict(x=16, residual=16, post_weight=0, scales=0, weight=16, out=16, residual_out=16, ld_x=8, ld_residual=8, ld_out=8,
                ld_residual_out=8, rows=2, cols=8, type=0, residual_type=0, scale=1.0, eps=1e-5)
NAN = float("nan")


@pytest.mark.parametrize("kw,rc", [({"x": 0}, -1), ({"weight": 0}, -1), ({"state": 0}, -1), ({"out": 0}, -1), ({"width": 5}, -2),
                                   ({"width": 1}, -2), ({"channels": 0}, -2), ({"type": 2}, -2), ({"ld_out": 7}, -2),
                                   ({"x": 17}, -4), ({"state": 17}, -4), ({"ld_x": -1}, -5), ({"n_seq": -1}, -5),
                                   ({"n_slots": -1}, -5), ({"n_tokens": -2}, -5)])
def test_conv(kw, rc):
    L = _C.lib()
    assert L.dfssm_causal_conv_step(fill(_C.Conv, CONV, kw), None) == rc
    assert L.dfssm_causal_conv_prefill(fill(_C.Conv, CONV, kw), None) == rc


@pytest.mark.parametrize("kw,rc", [({"x": 0}, -1), ({"dt": 0}, -1), ({"B": 0}, -1), ({"C": 0}, -1), ({"A_log": 0}, -1),
                                   ({"state_out": 0}, -1), ({"cols": 96}, -2), ({"cols": 256}, -2), ({"dim": 24}, -2),
                                   ({"dim": 0}, -2), ({"dim": 272}, -2), ({"groups": 2}, -2), ({"groups": 0}, -2), ({"type": 2}, -2),
                                   ({"dt_type": 1}, -2), ({"ld_out": 56}, -2), ({"x": 8}, -4), ({"state": 8}, -4), ({"ld_B": 132}, -4),
                                   ({"dt_type": 2, "dt": 18}, -4), ({"ld_x": 1 << 24}, -5), ({"ld_dt": -1}, -5), ({"n_seq": -1}, -5)])
def test_scan(kw, rc):
    L = _C.lib()
    assert L.dfssm_selective_scan_step(fill(_C.Scan, SCAN, kw), None) == rc
    assert L.dfssm_selective_scan_prefill(fill(_C.Scan, SCAN, kw), None, None) == rc


def test_counts():
    L = _C.lib()
    scan = lambda args, stream: L.dfssm_selective_scan_prefill(args, None, stream)
    for cls, base, step, whole in ((_C.Conv, CONV, L.dfssm_causal_conv_step, L.dfssm_causal_conv_prefill),
                                   (_C.Scan, SCAN, L.dfssm_selective_scan_step, scan)):
        assert step(None, None) == -1 and whole(None, None) == -1
        assert step(fill(cls, base, {"n_tokens": 3}), None) == -5 and step(fill(cls, base, {"cu_seqlens": 16}), None) == -5
        assert whole(fill(cls, base, {"n_tokens": 3}), None) == -5
        assert step(fill(cls, base, {"n_tokens": 0, "n_seq": 0}), None) == 0 and whole(fill(cls, base, {"n_seq": 0}), None) == 0
    assert L.dfssm_causal_conv_prefill(fill(_C.Conv, CONV, {"out": 16}), None) == -5      # out is x
    bytes_ = L.dfssm_selective_scan_workspace_bytes
    long = fill(_C.Scan, SCAN, {"n_tokens": 40000, "n_seq": 1})
    assert bytes_(long) > 0 and bytes_(fill(_C.Scan, SCAN, {})) == 0 and bytes_(None) == 0
    assert bytes_(fill(_C.Scan, SCAN, {"n_tokens": 40000, "n_seq": 1, "cols": 96})) == 0
    assert L.dfssm_selective_scan_prefill(long, None, None) == -1 and L.dfssm_selective_scan_prefill(long, 8, None) == -4


@pytest.mark.parametrize("kw,rc", [({"x": 0}, -1), ({"weight": 0}, -1), ({"out": 0}, -1), ({"cols": 0}, -2), ({"groups": 3}, -2),
                                   ({"cols": 16385}, -2), ({"type": 2}, -2), ({"ld_out": 7}, -2), ({"gate": 17}, -4),
                                   ({"weight": 18}, -4), ({"rows": -1}, -5), ({"ld_gate": -1}, -5), ({"eps": 0.0}, -5), ({"eps": NAN}, -5)])
def test_gated(kw, rc):
    assert _C.lib().dfssm_gated_norm(fill(_C.Gated, GATED, kw), None) == rc


@pytest.mark.parametrize("kw,rc", [({"residual": 0}, -1), ({"residual_out": 0}, -1), ({"cols": 16385}, -2), ({"residual_type": 1}, -2),
                                   ({"ld_residual_out": 7}, -2), ({"residual_type": 2, "residual": 18}, -4), ({"scales": 18}, -4),
                                   ({"rows": -1}, -5), ({"eps": -1.0}, -5)])
def test_residual(kw, rc):
    L = _C.lib()
    assert L.dfssm_residual_norm(fill(_C.Residual, RESIDUAL, kw), None) == rc
    assert L.dfssm_residual_norm(None, None) == -1 and L.dfssm_gated_norm(None, None) == -1
    assert L.dfssm_residual_norm(fill(_C.Residual, RESIDUAL, {"rows": 0}), None) == 0


def test_host_tensors():
    x, f = torch.zeros(2, 8, dtype=torch.float16), torch.zeros(8)
    with pytest.raises(TypeError):
        ops.causal_conv_step(x, x, None, x)
    with pytest.raises(TypeError):
        ops.causal_conv_prefill(x, x, None, x, cu_seqlens=torch.tensor([0, 2], dtype=torch.int32))
    with pytest.raises(TypeError):
        ops.selective_scan_step(x[None], x, f, x[None], x[None], x)
    with pytest.raises(TypeError):
        ops.selective_scan_prefill(x[None], x, f, x[None], x[None], x)
    with pytest.raises(TypeError):
        ops.gated_norm(x, x, f)
    with pytest.raises(TypeError):
        ops.residual_norm(x, x, f)
    with pytest.raises(TypeError):
        ops.gated_norm(x.float(), x, f)


def test_what_overlaps():
    """Rows beside each other in one tensor do not overlap; shifted ones do."""
    t = torch.zeros(10, 32)
    assert ops._apart(t[:, :8], t[:, 8:16]) and ops._apart(t[:, 8:16], t[:, :8]) and ops._apart(t[:3], t[3:])
    assert not ops._apart(t[:, :9], t[:, 8:16]) and not ops._apart(t[:5], t[4:]) and not ops._apart(t, t)
    assert not ops._apart(t[:, 28:], t[:, :30]) and ops._apart(t[:, 24:], t[1:, :8]) and ops._apart(t[:0], t)
    assert not ops._apart(t.view(-1)[4:36].view(4, 8), t[:, :8])
    h = t.view(10, 4, 8)
    assert ops._apart(h[:, :2], h[:, 2:]) and not ops._apart(h[:, :2], h[:, 1:])
