"""A state space layer between its projections, its operators in a row: prompts and tokens, eager and captured, on other
streams; and what the wrappers refuse on a GPU."""
import pytest
import torch

import layer_math as lm
from dfssm import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, P, G, N, D = 8, 64, 2, 64, 256
DI, C = H * P, H * P + 2 * G * N


def weights(seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    w = {"conv_w": (0.5 * r(C, 4)).half(), "conv_b": (0.2 * r(C)).half(), "A_log": torch.log(1 + 15 * torch.rand(H, generator=gen)),
         "D": 1 + 0.2 * r(H), "dt_bias": 4 * torch.rand(H, generator=gen) - 5, "norm": 1 + 0.2 * r(DI), "out": (r(DI, D) / DI ** 0.5).half(),
         "post": 0.5 + 0.1 * r(D), "next": 1 + 0.1 * r(D)}
    return {k: v.to(DEV) for k, v in w.items()}


def layer(w, xbc, dt, z, residual, conv, ssm, step, cu=None, slots=None):
    """Prompts (rows of all sequences) or one token each; the states are updated in place."""
    if step:
        x = ops.causal_conv_step(xbc, w["conv_w"], w["conv_b"], conv, slots=slots)
    else:
        x = ops.causal_conv_prefill(xbc, w["conv_w"], w["conv_b"], conv, cu_seqlens=cu, slots=slots)
    args = (x[:, :DI].unflatten(1, (H, P)), dt, w["A_log"], x[:, DI:DI + G * N].unflatten(1, (G, N)),
            x[:, DI + G * N:].unflatten(1, (G, N)), ssm)
    if step:
        y = ops.selective_scan_step(*args, D=w["D"], dt_bias=w["dt_bias"], slots=slots)
    else:
        y = ops.selective_scan_prefill(*args, D=w["D"], dt_bias=w["dt_bias"], cu_seqlens=cu, slots=slots)
    y = ops.gated_norm(y.flatten(1), z, w["norm"], groups=2)
    return ops.residual_norm(y @ w["out"], residual, w["next"], post_weight=w["post"], scale=0.5)


def inputs(T, seed=1):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    return [r(T, C).half().to(DEV), r(T, H).half().to(DEV), r(T, DI).half().to(DEV), r(T, D).to(DEV)]


def states(n, seed=2):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(n, C, 3, generator=gen).half().to(DEV), (0.3 * torch.randn(n, H, P, N, generator=gen)).to(DEV)


def exact(w, xbc, dt, z, residual, conv, ssm, lens):
    w = {k: v.cpu() for k, v in w.items()}
    xbc, dt, z, residual, conv, ssm = (t.cpu() for t in (xbc, dt, z, residual, conv, ssm))
    x, _, conv = lm.conv(xbc, w["conv_w"], w["conv_b"], conv, lens)
    x = x.half()
    y, _, ssm, _ = lm.scan(x[:, :DI].unflatten(1, (H, P)), dt, w["A_log"], x[:, DI:DI + G * N].unflatten(1, (G, N)),
                           x[:, DI + G * N:].unflatten(1, (G, N)), ssm, w["D"], w["dt_bias"], lens)
    y = lm.gated(y.flatten(1), z, w["norm"], 2)
    out, res, _ = lm.residual(y @ w["out"].double(), residual, w["next"], w["post"], 0.5)
    return out, res, conv, ssm


def close(got, ref, rounds):
    """Of values of size 1, `rounds` roundings of a half (2^-11 of each) of the largest."""
    err = (got.cpu().double() - ref).abs().max() / ref.abs().max()
    assert err < rounds * 2.0 ** -11, float(err)


def test_prompts_then_tokens():
    """The layer over packed prompts, then three tokens of each sequence, against the formulas in 64 bits. Each of its four
    operators rounds to halves once and the projection once more; the norms pass an error on with a factor near 1."""
    lens = [70, 1, 130, 40]
    T, n = sum(lens), len(lens)
    w = weights()
    xbc, dt, z, res = inputs(T + 3 * n)
    conv, ssm = states(n)
    off = lm.offsets(lens).tolist()
    order, at = [], T                                                          # rows of each sequence: its prompt, its tokens
    for b in range(n):
        order += list(range(off[b], off[b + 1])) + [T + 3 * b + i for i in range(3)]
    ref = exact(w, xbc[order], dt[order], z[order], res[order], conv, ssm, [x + 3 for x in lens])
    got = [torch.empty(T + 3 * n, D, dtype=torch.float16, device=DEV), torch.empty(T + 3 * n, D, device=DEV)]
    o, r = layer(w, xbc[:T], dt[:T], z[:T], res[:T], conv, ssm, False, cu=lm.offsets(lens, DEV))
    got[0][:T], got[1][:T] = o, r
    for i in range(3):
        rows = [T + 3 * b + i for b in range(n)]
        o, r = layer(w, xbc[rows], dt[rows], z[rows], res[rows], conv, ssm, True)
        got[0][rows], got[1][rows] = o, r
    close(got[0][order], ref[0], 8)
    close(got[1][order], ref[1], 8)
    assert torch.equal(conv.cpu(), ref[2])
    close(ssm, ref[3], 4)


@pytest.mark.parametrize("step", [False, True])
def test_captured(step):
    """A captured layer, replayed with other inputs and the program's own work in between, gives what the eager one gives."""
    lens = [1] * 5 if step else [1500, 3, 200]                                 # (the scan in segments: with a workspace)
    T, n = sum(lens), len(lens)
    w = weights()
    cu = None if step else lm.offsets(lens, DEV)
    data = inputs(T)
    conv, ssm = states(n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(w, *data, conv, ssm, step, cu)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                                         # two graphs, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = layer(w, *data, conv, ssm, step, cu)
        graphs.append((g, got))
    for i in range(6):
        for t, new in zip(data, inputs(T, 10 + i)):
            t.copy_(new)
        for t, new in zip((conv, ssm), states(n, 20 + i)):
            t.copy_(new)
        want_conv, want_ssm = conv.clone(), ssm.clone()
        want = layer(w, *data, want_conv, want_ssm, step, cu)
        torch.cuda.synchronize()
        g, got = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(conv, want_conv) and torch.equal(ssm, want_ssm)
        torch.randn(1 << 20, device=DEV).sum().item()


def test_streams_beside_each_other():
    lens = [700, 64, 3]
    w, cu = weights(), lm.offsets(lens, DEV)
    data = inputs(sum(lens))
    conv, ssm = states(3)
    want_state = (conv.clone(), ssm.clone())
    want = layer(w, *data, *want_state, False, cu)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            st = (conv.clone(), ssm.clone())
            got.append((*layer(w, *data, *st, False, cu), *st))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, (*want, *want_state)))


def test_refusals():
    w = weights()
    xbc, dt, z, res = inputs(10)
    conv, ssm = states(10)
    x, B = xbc[:, :DI].unflatten(1, (H, P)), xbc[:, DI:DI + G * N].unflatten(1, (G, N))
    cu = torch.tensor([0, 10], dtype=torch.int32, device=DEV)
    bad = [lambda: ops.causal_conv_step(xbc, w["conv_w"][:-1], None, conv), lambda: ops.causal_conv_step(xbc, w["conv_w"], w["conv_b"], conv[:9]),
           lambda: ops.causal_conv_step(xbc, w["conv_w"], w["conv_b"], conv[..., :2]),
           lambda: ops.causal_conv_step(xbc, w["conv_w"], w["conv_b"], conv, slots=torch.zeros(9, dtype=torch.int32, device=DEV)),
           lambda: ops.causal_conv_step(xbc, w["conv_w"], w["conv_b"], conv, out=xbc.flip(0)[:, :-1]),
           lambda: ops.causal_conv_prefill(xbc, w["conv_w"], w["conv_b"], conv, cu_seqlens=cu, out=xbc),
           lambda: ops.causal_conv_prefill(xbc, w["conv_w"], w["conv_b"], conv, cu_seqlens=cu[None]),
           lambda: ops.causal_conv_prefill(xbc, w["conv_w"], w["conv_b"], conv),
           lambda: ops.causal_conv_step(xbc, w["conv_w"], None, conv, state_out=conv[:9]),
           lambda: ops.selective_scan_step(x, dt[:9], w["A_log"], B, B, ssm), lambda: ops.selective_scan_step(x, dt, w["A_log"][:7], B, B, ssm),
           lambda: ops.selective_scan_step(x, dt, w["A_log"], B, B[:, :1], ssm), lambda: ops.selective_scan_step(x, dt, w["A_log"], B, B, ssm.transpose(2, 3)),
           lambda: ops.selective_scan_step(x, dt, w["A_log"], B, B, ssm, out=x), lambda: ops.selective_scan_prefill(x, dt, w["A_log"], B, B, ssm),
           lambda: ops.selective_scan_prefill(x[..., :8], dt, w["A_log"], B, B, ssm, cu_seqlens=cu),
           lambda: ops.gated_norm(z, z[:9], w["norm"]), lambda: ops.gated_norm(z, z, w["norm"][:9]), lambda: ops.gated_norm(z, z, w["norm"], groups=3),
           lambda: ops.gated_norm(z, None, w["norm"], eps=0.0), lambda: ops.gated_norm(z[1:], None, w["norm"], out=z[:-1]),
           lambda: ops.residual_norm(res.half(), res[:9], w["next"]), lambda: ops.residual_norm(res.half(), res, w["next"], scale=w["norm"]),
           lambda: ops.residual_norm(res.half(), res, w["next"], residual_out=res.t().contiguous().t())]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted:", i)
    wrong = [lambda: ops.causal_conv_step(xbc, w["conv_w"].float(), None, conv), lambda: ops.causal_conv_step(xbc.float(), w["conv_w"], None, conv),
             lambda: ops.causal_conv_prefill(xbc, w["conv_w"], None, conv, cu_seqlens=cu.long()),
             lambda: ops.selective_scan_step(x, dt.bfloat16(), w["A_log"], B, B, ssm), lambda: ops.selective_scan_step(x, dt, w["A_log"], B, B, ssm.half()),
             lambda: ops.gated_norm(z, z.bfloat16(), w["norm"]), lambda: ops.gated_norm(z, z, w["norm"].half()),
             lambda: ops.residual_norm(res.half(), res.bfloat16(), w["next"]), lambda: ops.causal_conv_step(xbc, w["conv_w"], None, conv.cpu())]
    for call in wrong:
        with pytest.raises(TypeError):
            call()
