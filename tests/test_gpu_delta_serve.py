"""Serving with the three operators together: ragged prompts through gated_delta_prefill, then a step, logits and a
filtered draw per token, the drawn token's row of the tables being the next step's input; a padding row in the
batch and sequences in slots of a larger pool. The recurrence in 64 bits over the prompt and the drawn tokens
must give every output and the states, and the draw in 64 bits on the logits every token. Then the same steps
captured once and replayed: the same bits.
"""
import numpy as np
import pytest
import torch

from dfssm import ops
from test_gpu_delta import check, recurrence
from test_gpu_draw import reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HK, HV, DK, DV, VOCAB = 2, 4, 128, 64, 1000
LENS, STEPS, POOL = [70, 1, 33, 130], 9, 7
SLOTS = [5, 0, 3, 6]                                      # of the pool; the batch has one padding row behind them


def tables(dtype):
    gen = torch.Generator().manual_seed(17)
    rand = lambda *s: torch.randn(*s, generator=gen)
    return {"q": rand(VOCAB, HK, DK).to(dtype), "k": rand(VOCAB, HK, DK).to(dtype), "v": rand(VOCAB, HV, DV).to(dtype),
            "g": -torch.nn.functional.softplus(2 * rand(VOCAB, HV) - 3), "beta": torch.sigmoid(rand(VOCAB, HV)),
            "head": 0.5 * rand(HV * DV, VOCAB), "state": 0.3 * rand(POOL, HV, DV, DK),
            "prompt": torch.randint(VOCAB, (sum(LENS),), generator=gen), "u": torch.rand(STEPS, len(LENS) + 1, generator=gen)}


FILTERS = dict(temperature=0.9, top_k=50, top_p=0.95, min_p=0.01)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serve(dtype):
    t = tables(dtype)
    d = {n: x.to(DEV) for n, x in t.items()}
    n = len(LENS)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(LENS)]), dtype=torch.int32, device=DEV)
    slots = torch.tensor(SLOTS, dtype=torch.int32, device=DEV)
    padded = torch.tensor(SLOTS + [-1], dtype=torch.int32, device=DEV)
    rows = lambda tok: [d[name][tok] for name in ("q", "k", "v", "g", "beta")]

    def prefill(state):
        out = ops.gated_delta_prefill(*rows(d["prompt"]), state, cu_seqlens=cu, slots=slots, l2norm=True)
        last = torch.zeros(n + 1, HV, DV, dtype=dtype, device=DEV)
        last[:n] = out[cu[1:].long() - 1]
        return out, last

    def draw(o, u):
        logits = (o.float().flatten(1) @ d["head"]).to(dtype)
        return logits, ops.sample_filtered(logits, u, **FILTERS)

    state = d["state"].clone()
    prompt_out, last = prefill(state)
    outs, logits, toks = [], [], []
    lg, tok = draw(last, d["u"][0])
    for s in range(1, STEPS):
        logits.append(lg)
        toks.append(tok)
        o = ops.gated_delta_step(*rows(tok), state, slots=padded, l2norm=True)
        outs.append(o)
        lg, tok = draw(o, d["u"][s])
    logits.append(lg)
    toks.append(tok)
    assert all(not o[n].any() for o in outs)                              # the padding row
    drawn = torch.stack(toks).cpu()

    f = {k: (v if k == "top_k" else np.float64(np.float32(v))) for k, v in FILTERS.items()}
    for s in range(STEPS):
        host = logits[s].float().cpu().numpy()
        for b in range(n + 1):
            want = reference(host[b], float(t["u"][s, b]), f["temperature"], f["top_k"], f["top_p"], f["min_p"])[0]
            assert drawn[s, b] == want, (s, b)

    every = torch.cat([torch.cat([p, drawn[:-1, b]]) for b, p in enumerate(t["prompt"].split(LENS))])
    lens = [l + STEPS - 1 for l in LENS]
    x = {name: t[name][every] for name in ("q", "k", "v", "g", "beta")}
    ref, ref_state = recurrence({**x, "state": t["state"]}, lens, True, slots=SLOTS)
    ref = ref.split(lens)
    got = [torch.cat([p, torch.stack([o[b] for o in outs])]) for b, p in enumerate(prompt_out.split(LENS))]
    check(torch.cat(got), torch.cat(ref), "out")
    check(state, ref_state, "state")

    # captured: one graph of a step and its draw, whose token is the next replay's input
    state2 = d["state"].clone()
    _, last = prefill(state2)
    tok, u = draw(last, d["u"][0])[1], d["u"][1].clone()

    def step():
        o = ops.gated_delta_step(*rows(tok), state2, slots=padded, l2norm=True)
        lg, new = draw(o, u)
        tok.copy_(new)
        return o, lg
    keep = state2.clone(), tok.clone()
    step()                                                                # once outside a capture
    state2.copy_(keep[0])
    tok.copy_(keep[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lg = step()
    for s in range(1, STEPS):
        u.copy_(d["u"][s])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, outs[s - 1]) and torch.equal(lg, logits[s]) and torch.equal(tok, toks[s]), s
    assert torch.equal(state2, state)
