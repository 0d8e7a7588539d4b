"""The operators between a state space layer's projections in 64 bits, for the tests: plain loops over tokens, and
beside each result the same formula over magnitudes, which bounds what rounding can do."""
import torch


def slices(lens):
    t = 0
    for n in lens:
        yield t, t + n
        t += n


def offsets(lens, device=None):
    return torch.tensor([0] + [b for _, b in slices(lens)], dtype=torch.int32, device=device)


def silu(x):
    return x * torch.sigmoid(x)


def conv(x, w, bias, state, lens, slots=None, act=True):
    """out, the sums' magnitudes (T, C) and the states afterwards."""
    W = w.shape[1]
    out = torch.zeros(x.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    state = state.clone()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if bias is None else bias.double()
    for i, (t0, t1) in enumerate(slices(lens)):
        s = i if slots is None else slots[i]
        rows = torch.cat([state[s].t(), x[t0:t1]])
        state[s] = rows[t1 - t0:].t()
        for t in range(t1 - t0):
            terms = rows[t:t + W].double() * w.t().double()
            out[t0 + t] = terms.sum(0) + b
            mag[t0 + t] = terms.abs().sum(0) + b.abs()
    return (silu(out) if act else out), mag, state


def time_step(dt, dt_bias, softplus=True):
    z = dt.double() + (0.0 if dt_bias is None else dt_bias.double())
    return torch.nn.functional.softplus(z, threshold=1e9) if softplus else z.clamp(min=0.0)


def scan(x, dt, A_log, B, C, state, D, dt_bias, lens, slots=None, softplus=True):
    """out and its magnitudes (T, H, P); the states afterwards and theirs."""
    T, H, P = x.shape
    G = B.shape[1]
    x, B, C = x.double(), B.double().repeat_interleave(H // G, 1), C.double().repeat_interleave(H // G, 1)
    d = time_step(dt, dt_bias, softplus)
    a = torch.exp(-d * torch.exp(A_log.double()))
    skip = torch.zeros(H, dtype=torch.float64) if D is None else D.double()
    state, smag = state.double().clone(), state.double().abs()
    out = torch.zeros(x.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for i, (t0, t1) in enumerate(slices(lens)):
        s = i if slots is None else slots[i]
        h, m = state[s], smag[s]
        for t in range(t0, t1):
            u = (d[t][:, None] * x[t])[..., None] * B[t][:, None]
            h.mul_(a[t][:, None, None]).add_(u)
            m.mul_(a[t][:, None, None]).add_(u.abs())
            out[t] = (h * C[t][:, None]).sum(-1) + skip[:, None] * x[t]
            mag[t] = (m * C[t][:, None].abs()).sum(-1) + (skip[:, None] * x[t]).abs()
    return out, mag, state, smag


def rms(x, w, eps=1e-5):
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w


def gated(x, z, w, groups=1, first=True, eps=1e-5):
    g = torch.ones(x.shape, dtype=torch.float64) if z is None else silu(z.double())
    shape = (*x.shape[:-1], groups, -1)
    x, g, w = x.double().reshape(shape), g.reshape(shape), w.double().reshape(groups, -1)
    return (rms(x * g, w, eps) if first else rms(x, w, eps) * g).flatten(-2)


def residual(x, r, w, post=None, scale=1.0, eps=1e-5):
    x = x.double() if post is None else rms(x.double(), post.double(), eps)
    scale = scale.double() if isinstance(scale, torch.Tensor) else float(torch.tensor(scale, dtype=torch.float32))
    new = r.double() + scale * x
    return rms(new, w.double(), eps), new, r.double().abs() + (scale * x).abs()


def half_step(dtype):
    """Of a rounding, relative; and absolute, of a subnormal."""
    return (torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -134)
