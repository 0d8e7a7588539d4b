"""generate() with top_k / min_p: the tokens of the model's own logits, drawn by the formula in 64 bits with the
random numbers that the documentation names; through graphs, eager steps and repeated calls."""
import numpy as np
import pytest
import torch

from df_ssm_inference import DFSSMModel
from dfssm.synth import config_tiny, make_prompts, make_weights
from test_gpu_draw import reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def expected(model, prompts, n, T, k, tp, mp, seed):
    """Eager forward() steps, each followed by the draw on the host."""
    model.reset_state()
    B = prompts.shape[0]
    u = torch.rand(n, B, generator=torch.Generator().manual_seed(seed)).numpy().astype(np.float64)
    f = lambda x: np.float64(np.float32(x))
    for t in range(prompts.shape[1] - 1):
        model.forward(prompts[:, t].to(DEV))
    tok, out = prompts[:, -1], []
    for t in range(n):
        lg = model.forward(tok.to(DEV)).float().cpu().numpy()
        tok = torch.tensor([reference(lg[b], u[t, b], f(T), k, f(tp), f(mp))[0] for b in range(B)])
        out.append(tok)
    return torch.stack(out, 1)


@pytest.mark.parametrize("B,T,k,tp,mp", [(1, 0.8, 40, 0.95, 0.0), (3, 1.2, 0, 1.0, 0.05), (6, 0.7, 200, 0.9, 0.01)])
def test_generate_filtered(B, T, k, tp, mp):
    w = make_weights(config_tiny(n_layer=2), seed=21)
    prompts = torch.from_numpy(make_prompts(B, w.cfg.vocab_size, 5))
    m = DFSSMModel.from_weights(w, device=DEV, batch_size=B)
    kw = dict(prompt=prompts, return_tokens=True, verbose=False, temperature=T)
    greedy = m.generate(n_tokens=6, prompt=prompts, return_tokens=True, verbose=False)
    plain = m.generate(n_tokens=11, top_p=tp, seed=5, **kw)
    ref = expected(m, prompts, 11, T, k, tp, mp, 77)
    got = m.generate(n_tokens=11, top_k=k, top_p=tp, min_p=mp, seed=77, **kw)
    assert torch.equal(got.cpu(), ref)
    # the state goes on from the last token: two greedy tokens after it, as after the same tokens as a prompt
    cont = m.decode(2)
    m.reset_state()
    m.ingest(torch.cat([prompts, got.cpu()], 1), step_by_step=True)
    first = m._next.clone()
    assert torch.equal(cont, torch.cat([first[:, None], m.decode(1)], 1))
    # graphs shared by every setting: another setting, then the first one again; top_k = 1 is greedy
    assert torch.equal(m.generate(n_tokens=6, top_k=1, seed=3, **kw), greedy)
    assert torch.equal(m.generate(n_tokens=11, top_k=k, top_p=tp, min_p=mp, seed=77, **kw), got)
    # a shorter run is the beginning of a longer one; other paths keep their results
    assert torch.equal(m.generate(n_tokens=4, top_k=k, top_p=tp, min_p=mp, seed=77, **kw), got[:, :4])
    assert torch.equal(m.generate(n_tokens=11, top_p=tp, seed=5, **kw), plain)
    assert torch.equal(m.generate(n_tokens=6, prompt=prompts, return_tokens=True, verbose=False), greedy)
    assert m.error_flag() == 0


def test_refused_before_the_state_changes():
    w = make_weights(config_tiny(n_layer=2), seed=21)
    m = DFSSMModel.from_weights(w, device=DEV, batch_size=1)
    m.forward(torch.tensor([3]))
    before = m.h_state.clone(), m.x.clone()
    with pytest.raises(ValueError):
        m.generate(n_tokens=2, verbose=False, temperature=0.8, top_k=4, repetition_penalty=1.2)
    with pytest.raises(ValueError):
        m.generate(n_tokens=2, verbose=False, top_k=4)
    assert torch.equal(m.h_state, before[0]) and torch.equal(m.x, before[1])
