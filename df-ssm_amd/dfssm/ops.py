"""Single-operator wrappers over the C ABI, taking torch tensors on the GPU.

These are the operator-level entry points (scaffold GEMM, RMSNorm+quantize, conv step, SSM step,
bit/embedding tiling). Every call launches on torch's current stream and raises on any error;
there is no CPU fallback. Arguments that are not contiguous are copied; all copies of a call stay bound
to names until its launch, so that the allocator cannot give one's memory to the next.
"""
from __future__ import annotations

import operator
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


_MAX_LD = 1 << 23   # elements from token to token: the kernels' offsets within a chunk are 32-bit


def _rows16(t: torch.Tensor, width: int):
    """t (tokens, heads, dim) with heads contiguous and 16-byte aligned tokens, itself or a copy, the
    distance of its tokens in elements and its address; width = heads * dim."""
    p = t.data_ptr()
    if not p & 15:
        if t.is_contiguous():
            return t, width, p
        ld, h, d = t.stride()
        if t.shape[0] <= 1:
            ld = width
        if d == 1 and h == t.shape[2] and ld % 8 == 0 and ld <= _MAX_LD:
            return t, ld, p
    t = t.clone(memory_format=torch.contiguous_format)
    return t, width, t.data_ptr()


def _rows32(t: torch.Tensor, width: int):
    """The same of (tokens, width) fp32."""
    if not t.is_contiguous():
        ld, h = t.stride()
        if t.shape[0] <= 1:
            ld = width
        if (h == 1 or width == 1) and ld <= _MAX_LD:
            return t, ld, t.data_ptr()
        t = t.clone(memory_format=torch.contiguous_format)
    return t, width, t.data_ptr()


def _delta_call(step: bool, q, k, v, g, beta, state, cu_seqlens, slots, scale, l2norm, out, state_out, n_seq):
    """Checks (tokens, heads, dim) arguments, launches and returns out. n_seq None: a sequence per token."""
    T_, f32 = torch.Tensor, torch.float32
    dt = q.dtype if isinstance(q, T_) else None
    kind = _TYPE16.get(dt)
    if kind is None:
        raise TypeError("q must be a float16 or bfloat16 tensor")
    dev = q.get_device()
    # (in one expression: these checks are a tenth of a small call's time)
    if not (dev >= 0 and isinstance(k, T_) and isinstance(v, T_) and isinstance(g, T_) and isinstance(beta, T_)
            and isinstance(state, T_) and k.dtype is dt and v.dtype is dt and g.dtype is f32 and beta.dtype is f32
            and state.dtype is f32 and k.get_device() == dev and v.get_device() == dev and g.get_device() == dev
            and beta.get_device() == dev and state.get_device() == dev):
        for t, d, n in ((q, dt, "q"), (k, dt, "k"), (v, dt, "v"), (g, f32, "g"), (beta, f32, "beta"), (state, f32, "state")):
            _need(t, d, n)
        raise ValueError("all tensors must be on one device")
    qs, vs, gs = q.shape, v.shape, g.shape
    if len(qs) != 3 or len(vs) != 3 or k.shape != qs or vs[0] != qs[0] or gs != vs[:2] or beta.shape != gs:
        raise ValueError("shape mismatch: q, k (tokens, key heads, k_dim), v (tokens, value heads, v_dim), "
                         f"g, beta (tokens, value heads); got {tuple(qs)}, {tuple(k.shape)}, {tuple(vs)}, "
                         f"{tuple(gs)}, {tuple(beta.shape)}")
    T, Hk, Dk = qs
    _, Hv, Dv = vs
    if n_seq is None:
        n_seq = T
    if Dk not in (64, 128) or Dv % 16 or not 16 <= Dv <= 256 or Hk < 1 or Hv < 1 or Hv % Hk:
        raise ValueError("k_dim must be 64 or 128, v_dim a multiple of 16 up to 256, and the value heads a multiple "
                         f"of the key heads; got k_dim {Dk}, v_dim {Dv}, {Hv} and {Hk} heads")
    ss = state.shape
    if len(ss) != 4 or ss[1] != Hv or ss[2] != Dv or ss[3] != Dk or not state.is_contiguous():
        raise ValueError(f"state must be contiguous (slots, {Hv}, {Dv}, {Dk})")
    sp = state.data_ptr()
    if state_out is None or state_out is state:
        state_out, so = state, sp
    else:
        _need(state_out, torch.float32, "state_out")
        if state_out.shape != ss or not state_out.is_contiguous() or state_out.get_device() != dev:
            raise ValueError("state_out must be contiguous, of state's shape and on its device")
        so = state_out.data_ptr()
        if sp != so and abs(so - sp) < state.numel() * 4:
            raise ValueError("state_out must be state or not overlap it")
    if sp % 16 or so % 16:
        raise ValueError("state must be 16-byte aligned")
    if slots is not None:
        _need(slots, torch.int32, "slots")
        if slots.shape != (n_seq,):
            raise ValueError(f"slots must be ({n_seq},)")
        if slots.get_device() != dev:
            raise ValueError("slots is on another device than q")
        slots = slots.contiguous()
    elif ss[0] < n_seq:
        raise ValueError(f"state has {ss[0]} slots for {n_seq} sequences")
    if cu_seqlens is not None and cu_seqlens.get_device() != dev:
        raise ValueError("cu_seqlens is on another device than q")
    width = Hv * Dv
    if out is None:
        out, ld_out = v.new_empty(vs), width
    else:
        _need(out, dt, "out")
        if out.shape != vs or out.get_device() != dev:
            raise ValueError("out must have v's shape and be on q's device")
        row, ld_out, _ = _rows16(out, width)
        if row is not out or ld_out < width:
            raise ValueError("out must have contiguous heads and 16-byte aligned tokens that do not overlap")
    if n_seq == 0:
        return out
    # (copies live until the launch)
    q, ld_q, qp = _rows16(q, Hk * Dk)
    k, ld_k, kp = _rows16(k, Hk * Dk)
    v, ld_v, vp = _rows16(v, width)
    g, ld_g, gp = _rows32(g, Hv)
    beta, ld_beta, bp = _rows32(beta, Hv)
    args = _C.Delta(qp, kp, vp, gp, bp, sp, so, _C.ptr(slots), _C.ptr(cu_seqlens), out.data_ptr(), ld_q, ld_k, ld_v, ld_g,
                    ld_beta, ld_out, T, n_seq, ss[0], Hk, Hv, Dk, Dv, kind, 1 if l2norm else 0,
                    Dk ** -0.5 if scale is None else scale)
    if dev != _C.current_device():
        with torch.cuda.device(dev):
            _delta_launch(step, args, q.device)
    else:
        _delta_launch(step, args, q.device)
    return out


def _delta_launch(step: bool, args, device) -> None:
    if step:
        rc = _C.lib().dfssm_gated_delta_step(args, _C.stream())
        if rc:
            _C.check(rc, "gated_delta_step")
        return
    need = _C.lib().dfssm_gated_delta_workspace_bytes(args)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _C.check(_C.lib().dfssm_gated_delta_prefill(args, _C.ptr(ws), _C.stream()), "gated_delta_prefill")


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
    l2norm divides q and k by sqrt(sum x^2 + 1e-6) first. out, if given, overlaps none of the others."""
    return _delta_call(True, q, k, v, g, beta, state, None, slots, scale, l2norm, out, state_out, None)


def gated_delta_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                        state: torch.Tensor, cu_seqlens=None, slots=None, scale=None, l2norm=False, out=None,
                        state_out=None) -> torch.Tensor:
    """The gated delta rule over whole prompts (dfssm_gated_delta_prefill), from the states the sequences
    have to those they leave: what gated_delta_step gives token by token, up to rounding in fp32 (relative to
    the largest v - S' k of the value column in 64 tokens: beside one more than 2^17 times as large, a token's
    own is off by up to 2^-39 of that one; and where 64 tokens have one key and beta |k|^2 close to 2, rounding
    grows to about 2^-15 of the state).

    Either packed, q, k (T, Hk, Dk), v (T, Hv, Dv), g, beta (T, Hv) with cu_seqlens (n + 1,) int32 on the
    device (sequence b has tokens cu_seqlens[b] .. cu_seqlens[b + 1], which must not fall; any length, zero
    included; rows of no sequence are left as they are in out), or one dimension more in front and no
    cu_seqlens: (B, T, ...). The other arguments are those of gated_delta_step. A value that is not finite may also make up to 63 tokens
    before it not finite."""
    if cu_seqlens is not None:
        _need(cu_seqlens, torch.int32, "cu_seqlens")
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
            raise ValueError("cu_seqlens must be (sequences + 1,)")
        return _delta_call(False, q, k, v, g, beta, state, cu_seqlens.contiguous(), slots, scale, l2norm,
                           out, state_out, cu_seqlens.numel() - 1)
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (g, "g"), (beta, "beta")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{n} must be a tensor")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4 or g.dim() != 3 or beta.dim() != 3:
        raise ValueError("without cu_seqlens: q, k, v (batch, tokens, heads, dim), g, beta (batch, tokens, heads)")
    B, T = q.shape[:2]
    if any(t.shape[:2] != (B, T) for t in (k, v, g, beta)):
        raise ValueError("q, k, v, g and beta must agree in batch and tokens")
    if out is not None:
        _need(out, q.dtype, "out")
        if out.shape != v.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous and have v's shape")
    o = _delta_call(False, q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), g.flatten(0, 1),
                    beta.flatten(0, 1), state, None, slots, scale, l2norm,
                    None if out is None else out.flatten(0, 1), state_out, B)
    return o.view(B, T, *v.shape[2:]) if out is None else out


# ---------------------------------------------------------------------------------------------
# token draw
# ---------------------------------------------------------------------------------------------
MAX_DRAW_VOCAB = 262144   # tokens of a row of sample_filtered
LOGIT_TYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}   # DFSSM_TYPE_*


def _on_device(t: torch.Tensor, name: str, dev) -> None:
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, not on {dev}")


def _per_row(x, dtype, name: str, B: int, dev, held: list):
    """A parameter as (number, device pointer): one of them counts."""
    if not isinstance(x, torch.Tensor):
        return (max(-1, min(operator.index(x), 2**31 - 1)) if dtype is torch.int32 else float(x)), 0
    if x.dtype is dtype and x.device == dev and x.shape == (B,) and x.is_contiguous():
        return 0, x.data_ptr()
    _need(x, dtype, name)
    if x.shape != (B,):
        raise ValueError(f"{name} must be a number or ({B},)")
    _on_device(x, name, dev)
    x = x.contiguous()
    held.append(x)
    return 0, x.data_ptr()


def sample_filtered(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                    want_logprob=False):
    """Tokens (B,) int64 drawn from logits (B, V) fp16, bf16 or fp32 with the random numbers u (B,) fp32 in
    [0, 1) (dfssm_sample_filtered): temperature, then the top_k most probable, of those the ones with at most
    top_p of the mass ranked above them, of those the ones at least min_p times as probable as the most
    probable, which is always kept; then the inverse of the cumulative mass in rank order at u. Equal logits
    rank by index.

    temperature, top_p, min_p: numbers, or (B,) fp32 on the device; top_k: a number, or (B,) int32. temperature
    <= 0 or NaN takes the most probable token; top_k <= 0, top_p >= 1 or NaN, min_p <= 0 filter nothing, min_p > 1
    or NaN leaves the most probable one. A NaN logit counts as -inf; a row whose logits are all -inf gives -1. V at
    most 262144; rows may be strided. With want_logprob also the logarithm of each token's share of what was kept,
    (B,) fp32."""
    kind = LOGIT_TYPE.get(logits.dtype) if isinstance(logits, torch.Tensor) else None
    if kind is None:
        raise TypeError("logits must be a float16, bfloat16 or float32 tensor")
    _need(logits, logits.dtype, "logits")
    _need(u, torch.float32, "u")
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= MAX_DRAW_VOCAB:
        raise ValueError(f"logits must be (B, V) with 1 <= V <= {MAX_DRAW_VOCAB}, got {tuple(logits.shape)}")
    dev = logits.device
    B, V = logits.shape
    if u.shape != (B,):
        raise ValueError(f"u must be ({B},)")
    _on_device(u, "u", dev)
    u = u.contiguous()
    held = []   # copies of parameters live until the launch
    temperature, tp = _per_row(temperature, torch.float32, "temperature", B, dev, held)
    top_k, kp = _per_row(top_k, torch.int32, "top_k", B, dev, held)
    top_p, pp = _per_row(top_p, torch.float32, "top_p", B, dev, held)
    min_p, mp = _per_row(min_p, torch.float32, "min_p", B, dev, held)
    ld, one = logits.stride()
    if (one != 1 and V > 1) or (B > 1 and ld < V):
        logits, ld = logits.clone(memory_format=torch.contiguous_format), V
    tokens = u.new_empty(B, dtype=torch.int64)
    logprob = u.new_empty(B) if want_logprob else None
    flt = _C.Filter(tp, kp, pp, mp, temperature, top_k, top_p, min_p)

    def launch():
        rc = _C.lib().dfssm_sample_filtered(logits.data_ptr(), kind, ld, B, V, u.data_ptr(), flt, tokens.data_ptr(),
                                            _C.ptr(logprob), _C.stream())
        if rc:
            _C.check(rc, "sample_filtered")
    if dev.index != _C.current_device():
        with torch.cuda.device(dev):
            launch()
    else:
        launch()
    return (tokens, logprob) if want_logprob else tokens
