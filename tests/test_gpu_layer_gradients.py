"""The operators between a layer's projections have no backward pass: they refuse a tensor whose gradient would be lost, and take
it where gradients are off."""
import pytest
import torch

from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def calls():
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    conv = dict(x=r(5, 24).half(), weight=r(24, 4).half(), bias=r(24).half(), state=r(5, 24, 3).half())
    scan = dict(x=r(5, 2, 16).half(), dt=r(5, 2), A_log=r(2), B=r(5, 1, 64).half(), C=r(5, 1, 64).half(), state=r(5, 2, 16, 64), D=r(2),
                dt_bias=r(2))
    gated = dict(x=r(5, 24).half(), gate=r(5, 24).half(), weight=r(24))
    residual = dict(x=r(5, 24).half(), residual=r(5, 24), weight=r(24), post_weight=r(24), scale=r(24))
    return [(ops.causal_conv_step, conv, {}), (ops.causal_conv_prefill, conv, {"cu_seqlens": cu}), (ops.selective_scan_step, scan, {}),
            (ops.selective_scan_prefill, scan, {"cu_seqlens": cu}), (ops.gated_norm, gated, {}), (ops.residual_norm, residual, {})]


@pytest.mark.parametrize("i", range(6))
def test_each_argument(i):
    op, tensors, more = calls()[i]
    flat = lambda y: y if isinstance(y, tuple) else (y,)
    plain = {k: t.clone() for k, t in tensors.items()}
    want = flat(op(**plain, **more))
    assert not any(t.requires_grad for t in want)
    for name in tensors:
        leaf = {k: t.clone() for k, t in tensors.items()}
        leaf[name].requires_grad_()
        before = {k: t.detach().clone() for k, t in leaf.items()}
        with pytest.raises(ValueError, match="gradient"):
            op(**leaf, **more)
        assert all(torch.equal(leaf[k], before[k]) for k in leaf)               # no state has moved on
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(flat(op(**leaf, **more)), want))
        leaf = {k: t.clone() for k, t in tensors.items()}
        leaf[name] = leaf[name].requires_grad_().detach()
        assert all(torch.equal(a, b) for a, b in zip(flat(op(**leaf, **more)), want))
