"""Single-operator wrappers over the C ABI, taking torch tensors on the GPU.

These are the operator-level entry points (scaffold GEMM, RMSNorm+quantize, conv step, SSM step,
bit/embedding tiling). Every call launches on torch's current stream and raises on any error;
there is no CPU fallback. Arguments that are not contiguous are copied; all copies of a call stay bound
to names until its launch, so that the allocator cannot give one's memory to the next.
"""
from __future__ import annotations

import threading

import torch

from . import _C


def _need(t: torch.Tensor, dtype, name: str):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is dtype:
        return
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise TypeError(f"{name} must be a CUDA (HIP) tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def tile_bits(packed: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """(rows, k/32) int32 sign-bit words -> tiled copy for the scaffold kernels."""
    _need(packed, torch.int32, "packed")
    if not packed.is_contiguous() or packed.numel() != rows * (k // 32):
        raise ValueError("packed must be a contiguous (rows, k/32) int32 tensor")
    out = torch.empty(_C.lib().dfssm_tiled_bits_bytes(rows, k) // 4, dtype=torch.int32, device=packed.device)
    _C.check(_C.lib().dfssm_tile_bits(packed.data_ptr(), out.data_ptr(), rows, k, _C.stream()), "tile_bits")
    return out


def scaffold_gemm(tiled_bits: torch.Tensor, q: torch.Tensor, N: int, xscale=None, wscale=None, want_y=False):
    """int32 acc (M, N) = q (M, K) int8 x sign-bit matrix^T; optionally y fp16 (M, N)."""
    _need(q, torch.int8, "q")
    M, K = q.shape
    acc = torch.empty(M, N, dtype=torch.int32, device=q.device)
    y = torch.empty(M, N, dtype=torch.float16, device=q.device) if want_y else None
    q = q.contiguous()
    _C.check(_C.lib().dfssm_scaffold_gemm(
        tiled_bits.data_ptr(), q.data_ptr(), _C.ptr(xscale), _C.ptr(wscale), M, N, K,
        acc.data_ptr(), _C.ptr(y), _C.stream()), "scaffold_gemm")
    return (acc, y) if want_y else acc


SCAFFOLD_WORKSPACE_BYTES = 64 << 10   # DFSSM_SCAFFOLD_WORKSPACE_BYTES
SCAFFOLD_ERROR_OFFSET = 1024          # DFSSM_SCAFFOLD_ERROR_OFFSET
SCAFFOLD_WORKSPACE_STREAMS = 64       # streams whose workspaces are kept
_scaffold_ws = {}
_scaffold_ws_lock = threading.Lock()


def _new_scaffold_workspace(device) -> torch.Tensor:
    return torch.zeros(SCAFFOLD_WORKSPACE_BYTES // 4, dtype=torch.int32, device=device)


def scaffold_workspace(device) -> torch.Tensor:
    """The exchange workspace of dfssm_scaffold_lora_gemm for calls on torch's current stream of `device`,
    zeroed on that stream at allocation. Calls that share one must not overlap, so every stream has its
    own; those of the last SCAFFOLD_WORKSPACE_STREAMS streams are kept. A stream that is being captured
    gets a new one at each call, owned by its graph and zeroed at every replay: a kept one would tie
    the graph's replays to whatever runs on the capture's stream then."""
    return _stream_workspace(device, _C.stream())


def _stream_workspace(device, stream: int) -> torch.Tensor:
    dev = device if isinstance(device, torch.device) else torch.device(device)
    if stream and torch.cuda.is_current_stream_capturing():  # (the null stream cannot be captured)
        return _new_scaffold_workspace(dev)
    if dev.index is None:
        dev = torch.device(dev.type, torch.cuda.current_device())
    key = (dev, stream)
    ws = _scaffold_ws.get(key)
    if ws is None:
        with _scaffold_ws_lock:
            ws = _scaffold_ws.get(key)
            if ws is None:
                while len(_scaffold_ws) >= SCAFFOLD_WORKSPACE_STREAMS:  # (freed in its stream's order)
                    del _scaffold_ws[next(iter(_scaffold_ws))]
                ws = _scaffold_ws[key] = _new_scaffold_workspace(dev)
    return ws


def scaffold_error(workspace: torch.Tensor) -> int:
    """The workspace's error word (synchronizes): non-zero after a call whose wait timed out."""
    return int(workspace[SCAFFOLD_ERROR_OFFSET // 4].item())


def scaffold_lora_gemm(tiled_bits: torch.Tensor, wscale: torch.Tensor, q: torch.Tensor, xscale: torch.Tensor,
                       xn: torch.Tensor, lA: torch.Tensor, lA_s: torch.Tensor, lBq: torch.Tensor, N: int,
                       workspace="auto"):
    """One projection with its LoRA (dfssm_scaffold_lora_gemm): returns (acc int32 (M, N),
    y fp16 (M, N), lora_h fp16 (M, 16)). q (M, K) int8 with fp16 scales xscale (M,), xn (M, K) fp16,
    lA (N, 16) int8, lA_s (N,) fp16, lBq (16, K) fp16, wscale (N,) fp16. workspace: "auto" (the
    current stream's exchange workspace: one launch at M <= 4; in a capture one more, which clears it),
    None (no workspace) or an int32 tensor of SCAFFOLD_WORKSPACE_BYTES, zeroed before its first use and
    used by calls that do not overlap."""
    _need(q, torch.int8, "q")
    _need(xn, torch.float16, "xn")
    _need(lBq, torch.float16, "lBq")
    _need(lA, torch.int8, "lA")
    M, K = q.shape
    if xn.shape != (M, K) or lBq.shape != (16, K) or lA.shape != (N, 16):
        raise ValueError("shape mismatch: q/xn (M, K), lBq (16, K), lA (N, 16)")
    acc = torch.empty(M, N, dtype=torch.int32, device=q.device)
    y = torch.empty(M, N, dtype=torch.float16, device=q.device)
    h = torch.empty(M, 16, dtype=torch.float16, device=q.device)
    stream = _C.stream()
    if isinstance(workspace, str):
        if workspace != "auto":
            raise ValueError('workspace must be "auto", None or a tensor')
        workspace = _stream_workspace(q.device, stream) if M <= 4 else None  # (unused by more rows)
    elif workspace is not None:
        _need(workspace, torch.int32, "workspace")
        if workspace.numel() * 4 < SCAFFOLD_WORKSPACE_BYTES:
            raise ValueError(f"workspace must hold {SCAFFOLD_WORKSPACE_BYTES} bytes")
    wscale, q, xscale, xn = wscale.contiguous(), q.contiguous(), xscale.contiguous(), xn.contiguous()
    lA, lA_s, lBq = lA.contiguous(), lA_s.contiguous(), lBq.contiguous()
    _C.check(_C.lib().dfssm_scaffold_lora_gemm(
        tiled_bits.data_ptr(), wscale.data_ptr(), q.data_ptr(), xscale.data_ptr(), xn.data_ptr(), lA.data_ptr(),
        lA_s.data_ptr(), lBq.data_ptr(), M, N, K, h.data_ptr(), acc.data_ptr(), y.data_ptr(), _C.ptr(workspace), stream), "scaffold_lora_gemm")
    return acc, y, h


def rmsnorm_quantize(x: torch.Tensor, w: torch.Tensor):
    """x (M, K) fp16, w (K) fp32 -> (xn fp16 (M, K), q int8 (M, K), scale fp16 (M,))."""
    _need(x, torch.float16, "x")
    _need(w, torch.float32, "w")
    M, K = x.shape
    xn = torch.empty(M, K, dtype=torch.float16, device=x.device)
    q = torch.empty(M, K, dtype=torch.int8, device=x.device)
    s = torch.empty(M, dtype=torch.float16, device=x.device)
    x, w = x.contiguous(), w.contiguous()
    _C.check(_C.lib().dfssm_rmsnorm_quantize(x.data_ptr(), w.data_ptr(), M, K,
                                             xn.data_ptr(), q.data_ptr(), s.data_ptr(), _C.stream()),
             "rmsnorm_quantize")
    return xn, q, s


def conv_step(conv_state: torch.Tensor, xbc: torch.Tensor, conv_w: torch.Tensor, conv_b: torch.Tensor) -> None:
    """In place: conv_state (B, C, 3) fp16 and xbc (B, C) fp16 (row stride honoured)."""
    for t, n in ((conv_state, "conv_state"), (xbc, "xBC"), (conv_w, "conv_weight"), (conv_b, "conv_bias")):
        _need(t, torch.float16, n)
    B, C = xbc.shape
    if conv_state.shape != (B, C, 3) or not conv_state.is_contiguous():
        raise ValueError(f"conv_state must be contiguous ({B}, {C}, 3)")
    if xbc.stride(1) != 1:
        raise ValueError("xBC rows must be contiguous")
    conv_w, conv_b = conv_w.contiguous(), conv_b.contiguous()
    _C.check(_C.lib().dfssm_conv_step(conv_state.data_ptr(), xbc.data_ptr(), xbc.stride(0), conv_w.data_ptr(),
                                      conv_b.data_ptr(), B, C, _C.stream()), "conv_step")


def ssm_step(h: torch.Tensor, xbc: torch.Tensor, dt: torch.Tensor, dt_bias, A_log, D, y_out: torch.Tensor) -> None:
    """h (B, H, P, N) fp32 in place; xbc rows x|B|C fp16; dt (B, H) fp16; y_out (B, H*P) fp16."""
    _need(h, torch.float32, "h_state")
    _need(xbc, torch.float16, "xBC")
    _need(dt, torch.float16, "dt")
    _need(y_out, torch.float16, "y_out")
    for t, n in ((dt_bias, "dt_bias"), (A_log, "A_log"), (D, "D")):
        _need(t, torch.float32, n)
    B, H, P, N = h.shape
    if not h.is_contiguous() or xbc.stride(1) != 1 or dt.stride(1) != 1 or y_out.stride(1) != 1:
        raise ValueError("h_state must be contiguous and xBC / dt / y_out rows contiguous")
    dt_bias, A_log, D = dt_bias.contiguous(), A_log.contiguous(), D.contiguous()
    _C.check(_C.lib().dfssm_ssm_step(h.data_ptr(), xbc.data_ptr(), xbc.stride(0), dt.data_ptr(), dt.stride(0),
                                     dt_bias.data_ptr(), A_log.data_ptr(), D.data_ptr(), y_out.data_ptr(),
                                     y_out.stride(0), B, H, P, N, _C.stream()), "ssm_step")


# ---------------------------------------------------------------------------------------------
# gated delta rule
# ---------------------------------------------------------------------------------------------
_TYPE16 = {torch.float16: 0, torch.bfloat16: 1}   # DFSSM_TYPE_F16, DFSSM_TYPE_BF16


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """(tokens, heads, dim) with heads contiguous and 16-byte aligned tokens: t itself or a copy."""
    s = t.stride()
    if s[2] == 1 and s[1] == t.shape[2] and s[0] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _on_device(t: torch.Tensor, name: str, dev) -> None:
    if t is not None and t.device != dev:
        raise ValueError(f"{name} is on {t.device}, not on {dev}")


def _delta_call(step: bool, q, k, v, g, beta, state, cu_seqlens, slots, scale, l2norm, out, state_out, n_seq):
    """Checks (tokens, heads, dim) arguments, launches and returns out."""
    dev = q.device if isinstance(q, torch.Tensor) else None
    kind = _TYPE16.get(q.dtype) if isinstance(q, torch.Tensor) else None
    if kind is None:
        raise TypeError("q must be a float16 or bfloat16 tensor")
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, q.dtype, n)
        if t.dim() != 3:
            raise ValueError(f"{n} must have 3 dimensions, got {tuple(t.shape)}")
    for t, n in ((g, "g"), (beta, "beta"), (state, "state")):
        _need(t, torch.float32, n)
    T, Hk, Dk = q.shape
    Hv, Dv = v.shape[1:]
    if k.shape != q.shape or v.shape[0] != T or g.shape != (T, Hv) or beta.shape != (T, Hv):
        raise ValueError("shape mismatch: q, k (tokens, key heads, k_dim), v (tokens, value heads, v_dim), "
                         f"g, beta (tokens, value heads); got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}, "
                         f"{tuple(g.shape)}, {tuple(beta.shape)}")
    if Dk not in (64, 128) or Dv % 16 or not 16 <= Dv <= 256 or Hk < 1 or Hv < 1 or Hv % Hk:
        raise ValueError("k_dim must be 64 or 128, v_dim a multiple of 16 up to 256, and the value heads a multiple "
                         f"of the key heads; got k_dim {Dk}, v_dim {Dv}, {Hv} and {Hk} heads")
    if state.dim() != 4 or state.shape[1:] != (Hv, Dv, Dk) or not state.is_contiguous():
        raise ValueError(f"state must be contiguous (slots, {Hv}, {Dv}, {Dk})")
    if state_out is None:
        state_out = state
    elif state_out is not state:
        _need(state_out, torch.float32, "state_out")
        if state_out.shape != state.shape or not state_out.is_contiguous():
            raise ValueError("state_out must be contiguous and of state's shape")
        lo, n = state.data_ptr(), state.numel() * 4
        if lo != state_out.data_ptr() and abs(state_out.data_ptr() - lo) < n:
            raise ValueError("state_out must be state or not overlap it")
    if slots is not None:
        _need(slots, torch.int32, "slots")
        if slots.shape != (n_seq,):
            raise ValueError(f"slots must be ({n_seq},)")
        slots = slots.contiguous()
    elif state.shape[0] < n_seq:
        raise ValueError(f"state has {state.shape[0]} slots for {n_seq} sequences")
    if state.data_ptr() % 16 or state_out.data_ptr() % 16:
        raise ValueError("state must be 16-byte aligned")
    if out is None:
        out = torch.empty(T, Hv, Dv, dtype=q.dtype, device=dev)
    else:
        _need(out, q.dtype, "out")
        if out.shape != v.shape or (T and _rows16(out) is not out):
            raise ValueError("out must have v's shape, contiguous heads and 16-byte aligned tokens")
    for t, n in ((k, "k"), (v, "v"), (g, "g"), (beta, "beta"), (state, "state"), (state_out, "state_out"),
                 (slots, "slots"), (cu_seqlens, "cu_seqlens"), (out, "out")):
        _on_device(t, n, dev)
    if n_seq == 0:
        return out
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    g = g if g.stride(1) == 1 else g.contiguous()
    beta = beta if beta.stride(1) == 1 else beta.contiguous()
    args = _C.Delta(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), state.data_ptr(),
                    state_out.data_ptr(), _C.ptr(slots), _C.ptr(cu_seqlens), out.data_ptr(),
                    q.stride(0), k.stride(0), v.stride(0), g.stride(0), beta.stride(0), out.stride(0), T,
                    n_seq, state.shape[0], Hk, Hv, Dk, Dv, kind, 1 if l2norm else 0,
                    Dk ** -0.5 if scale is None else scale)
    with torch.cuda.device(dev):
        if step:
            _C.check(_C.lib().dfssm_gated_delta_step(args, _C.stream()), "gated_delta_step")
        else:
            need = _C.lib().dfssm_gated_delta_workspace_bytes(args)
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            _C.check(_C.lib().dfssm_gated_delta_prefill(args, _C.ptr(ws), _C.stream()), "gated_delta_prefill")
    return out


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, slots=None, scale=None, l2norm=False, out=None, state_out=None) -> torch.Tensor:
    """One token per sequence of the gated delta rule (dfssm_gated_delta_step): per value head, with
    a = exp(g), S' = a S, u = beta (v - S' k), S = S' + u k^T, and returns scale S q.

    q, k (B, Hk, Dk) and v (B, Hv, Dv) fp16 or bf16, Hv a multiple of Hk (value head h reads key head
    h // (Hv // Hk)), Dk 64 or 128, Dv a multiple of 16 up to 256; g (log decay, at most 0) and beta (B, Hv)
    fp32; state (slots, Hv, Dv, Dk) fp32, contiguous, updated in place, or written to state_out (of the same
    shape; slots that no sequence has are left as they are there). Rows of B may be strided. slots (B,) int32:
    the slot of each sequence (default 0..B-1); a negative one marks padding (zeros returned), one past the
    state or taken by an earlier row gives NaN, and neither touches a state. scale defaults to Dk^-0.5;
    l2norm divides q and k by sqrt(sum x^2 + 1e-6) first."""
    return _delta_call(True, q, k, v, g, beta, state, None, slots, scale, l2norm, out, state_out,
                       q.shape[0])


def gated_delta_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                        state: torch.Tensor, cu_seqlens=None, slots=None, scale=None, l2norm=False, out=None,
                        state_out=None) -> torch.Tensor:
    """The gated delta rule over whole prompts (dfssm_gated_delta_prefill), from the states the sequences
    have to those they leave: what gated_delta_step gives token by token, up to rounding in fp32.

    Either packed, q, k (T, Hk, Dk), v (T, Hv, Dv), g, beta (T, Hv) with cu_seqlens (n + 1,) int32 on the
    device (sequence b has tokens cu_seqlens[b] .. cu_seqlens[b + 1]; any length, zero included; rows of no
    sequence are left as they are in out), or one dimension more in front and no cu_seqlens: (B, T, ...).
    The other arguments are those of gated_delta_step."""
    if cu_seqlens is not None:
        _need(cu_seqlens, torch.int32, "cu_seqlens")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError("cu_seqlens must be (sequences + 1,)")
        return _delta_call(False, q, k, v, g, beta, state, cu_seqlens.contiguous(), slots, scale, l2norm,
                           out, state_out, cu_seqlens.numel() - 1)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or g.dim() != 3 or beta.dim() != 3:
        raise ValueError("without cu_seqlens: q, k, v (batch, tokens, heads, dim), g, beta (batch, tokens, heads)")
    B, T = q.shape[:2]
    if any(t.shape[:2] != (B, T) for t in (k, v, g, beta)):
        raise ValueError("q, k, v, g and beta must agree in batch and tokens")
    if out is not None and not out.is_contiguous():
        raise ValueError("out must be contiguous")
    o = _delta_call(False, q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), g.flatten(0, 1),
                    beta.flatten(0, 1), state, None, slots, scale, l2norm,
                    None if out is None else out.flatten(0, 1), state_out, B)
    return o.view(B, T, *v.shape[2:]) if out is None else out


# ---------------------------------------------------------------------------------------------
# token draw
# ---------------------------------------------------------------------------------------------
_LOGIT_TYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}   # DFSSM_TYPE_*


def sample_filtered(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                    want_logprob=False):
    """Tokens (B,) int64 drawn from logits (B, V) fp16, bf16 or fp32 with the random numbers u (B,) fp32 in
    [0, 1) (dfssm_sample_filtered): temperature, then the top_k most probable, of those the ones with at most
    top_p of the mass ranked above them, of those the ones at least min_p times as probable as the most
    probable, which is always kept; then the inverse of the cumulative mass in rank order at u. Equal logits
    rank by index.

    temperature, top_p, min_p: numbers, or (B,) fp32 on the device; top_k: a number, or (B,) int32. temperature
    <= 0 takes the most probable token; top_k <= 0, top_p >= 1, min_p <= 0 filter nothing. A row whose logits
    are all -inf gives -1. V at most 262144; rows may be strided. With want_logprob also the logarithm of each
    token's share of what was kept, (B,) fp32."""
    kind = _LOGIT_TYPE.get(logits.dtype) if isinstance(logits, torch.Tensor) else None
    if kind is None:
        raise TypeError("logits must be a float16, bfloat16 or float32 tensor")
    _need(logits, logits.dtype, "logits")
    _need(u, torch.float32, "u")
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= 262144:
        raise ValueError(f"logits must be (B, V) with 1 <= V <= 262144, got {tuple(logits.shape)}")
    dev = logits.device
    B, V = logits.shape
    if u.shape != (B,):
        raise ValueError(f"u must be ({B},)")
    _on_device(u, "u", dev)
    ptrs, values, held = [], [], [u.contiguous()]
    for x, n, dt in ((temperature, "temperature", torch.float32), (top_k, "top_k", torch.int32),
                     (top_p, "top_p", torch.float32), (min_p, "min_p", torch.float32)):
        if isinstance(x, torch.Tensor):
            _need(x, dt, n)
            if x.shape != (B,):
                raise ValueError(f"{n} must be a number or ({B},)")
            _on_device(x, n, dev)
            x = x.contiguous()
            held.append(x)
            ptrs.append(x.data_ptr())
            values.append(0)
        else:
            ptrs.append(0)
            values.append(int(x) if dt is torch.int32 else float(x))
    if logits.stride(1) != 1 or (B > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    tokens = torch.empty(B, dtype=torch.int64, device=dev)
    logprob = torch.empty(B, dtype=torch.float32, device=dev) if want_logprob else None
    with torch.cuda.device(dev):
        _C.check(_C.lib().dfssm_sample_filtered(logits.data_ptr(), kind, logits.stride(0), B, V, held[0].data_ptr(),
                                                _C.Filter(*ptrs, *values), tokens.data_ptr(), _C.ptr(logprob),
                                                _C.stream()), "sample_filtered")
    return (tokens, logprob) if want_logprob else tokens
