"""Temporal operators: a mixer over the windows of many streams, and the norms, gate and residual around it.

`decay_attention` (linear attention with one constant decay per head) stands beside `ConvLSTM` and the LSTM of `LSTMNetVIT`:
each stream carries a state of fixed size from call to call, a whole recording is one call on the matrix cores, a single window is
one pass over the state (`decay_attention_step`). `block_norm` is a residual block's end and the next one's beginning in one
pass per token: y = res_scale * x + act(gate) * norm_post(f), h = norm_pre(y); evfly's own LayerNorm(x + f)
(learner/ViTsubmodules.py:143-146) is its plainest form. Both have gradients; the arithmetic runs in libevfly_hip.so
(`evfly_decay_attention_*`, `evfly_block_norm_*`, include/evfly_hip.h), on the current stream of the tensors' device.

Tokens are float32 or bfloat16 CUDA tensors; sums, statistics and states are float32 in both.
"""
import ctypes as C
import math

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib

_DTYPE = {torch.float32: 0, torch.bfloat16: 1}
MAX_HEAD_DIM = 128
MAX_CHANNELS = 8192
STEP_TOKENS = 16                    # up to here a forward needs no workspace (EVFLY_DECAY_STEP_TOKENS)
_NORM = {None: 0, "layer": 1, "rms": 2}
_GATE_ACT = {a: _lib.ACT_CODES[a] for a in ("none", "sigmoid", "tanh")}


_getDevice, _rawStream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream      # (a tick's call is a few microseconds: no Stream object for it)
_tracingState, _dispatchModes = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack


def _ptr(t):
    return None if t is None else t.data_ptr()


def _dense(t):
    return None if t is None else t.contiguous()


def _workspace(nbytes, like):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes > 0 else None


def _watched():
    """Something other than autograd may follow the call (`_refuse_unseen`)."""
    return _forward_ad._current_level >= 0 or _dispatchModes() > 0 or _tracingState() is not None


def _refuse_unseen(who, tensors, recorded):
    """The library's work is no torch operation: forward-mode differentiation takes its results for constants, a tracer for memory that nothing writes. (recorded: the
    call is an autograd function's, which torch.jit.trace keeps as a whole.)"""
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{who} has no forward-mode derivatives")
    if not recorded and _tracingState() is not None:
        raise RuntimeError(f"{who}: torch.jit.trace does not see its work")
    if _dispatchModes() > 0:
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        if get_proxy_mode() is not None:
            raise RuntimeError(f"{who}: make_fx does not see its work")


def _check_tokens(who, named, like):
    for name, t in named:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{who}: {name} must be a CUDA tensor")
        if t.dtype != like.dtype or t.dtype not in _DTYPE:
            raise ValueError(f"{who}: {name} is {t.dtype}; the token tensors are all float32 or all bfloat16")
        if t.device != like.device:
            raise ValueError(f"{who}: {name} is on {t.device}, not on {like.device}")


def _check_f32(who, name, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != tuple(shape) or t.device != device:
        raise ValueError(f"{who}: {name} must be a float32 tensor {tuple(shape)} on {device}" +
                         (f", not {t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else f", not {type(t).__name__}"))


# ---------------------------------------------------------------------------------------- decay attention
def _decay_fits(q, k, v, log_decay, state, lengths, lead):
    """Everything `_refuse_decay` asks for, in one look."""
    try:
        dt, dev, qs, ks, vs = q.dtype, q.device, q.shape, k.shape, v.shape
        H, KV, dk, dv = qs[-2], ks[-2], qs[-1], vs[-1]
        return (len(qs) == len(ks) == len(vs) == lead + 2 and dt in _DTYPE and k.dtype is dt and v.dtype is dt and dev.type == "cuda" and k.device == dev and v.device == dev and
                ks[:lead] == qs[:lead] and vs[:lead] == qs[:lead] and ks[-1] == dk and vs[-2] == KV and KV > 0 and H > 0 and H % KV == 0 and
                0 < dk <= MAX_HEAD_DIM and 0 < dv <= MAX_HEAD_DIM and
                log_decay.dtype is torch.float32 and log_decay.shape == (H,) and log_decay.device == dev and not log_decay.requires_grad and
                (state is None or (state.dtype is torch.float32 and state.shape == (qs[0], H, dk, dv) and state.device == dev)) and
                (lengths is None or (lengths.dtype is torch.int32 and lengths.shape == qs[:1] and lengths.device == dev)))
    except (AttributeError, IndexError):
        return False


def _refuse_decay(who, q, k, v, log_decay, state, lengths, lead):
    sizes = "(streams, tokens, heads, head size)" if lead == 2 else "(streams, heads, head size)"
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != lead + 2:
            raise ValueError(f"{who}: {name} must be a tensor {sizes}")
    _check_tokens(who, (("q", q), ("k", k), ("v", v)), q)
    H, KV, dk, dv = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    if k.shape[:lead] != q.shape[:lead] or v.shape[:lead] != q.shape[:lead] or k.shape[-1] != dk or v.shape[-2] != KV:
        raise ValueError(f"{who}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if KV == 0 or H == 0 or H % KV:
        raise ValueError(f"{who}: {H} heads do not share {KV} key / value heads evenly")
    if not (1 <= dk <= MAX_HEAD_DIM and 1 <= dv <= MAX_HEAD_DIM):
        raise ValueError(f"{who}: head sizes {dk}, {dv} are not in 1 .. {MAX_HEAD_DIM}")
    _check_f32(who, "log_decay", log_decay, (H,), q.device)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: log_decay is a constant of the head and has no gradient (detach it)")
    if state is not None:
        _check_f32(who, "state", state, (q.shape[0], H, dk, dv), q.device)
    if lengths is not None and (not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or tuple(lengths.shape) != (q.shape[0],)
                                or lengths.device != q.device):
        raise ValueError(f"{who}: lengths must be an int32 tensor ({q.shape[0]},) on {q.device}")


def _check_decay(who, q, k, v, log_decay, state, lengths, scale, lead):
    _lib.lib()                                                   # (no GPU / no library: that error first)
    if not _decay_fits(q, k, v, log_decay, state, lengths, lead):
        _refuse_decay(who, q, k, v, log_decay, state, lengths, lead)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{who}: scale is not finite")
    return scale


def _rows(t):
    """Rows of a token tensor as the kernels read them: any strides, the last dimension dense."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(q, k, v):
    if q.dim() == 3:                                             # one token: its stride is never taken
        return (C.c_int64 * 9)(*(s for t in (q, k, v) for s in (t.stride(0), 0, t.stride(1))))
    return (C.c_int64 * 9)(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])


def _decay_forward(q, k, v, log_decay, state, lengths, scale, new_state):
    idx = q.get_device()
    if idx != _getDevice():
        with torch.cuda.device(idx):
            return _decay_forward(q, k, v, log_decay, state, lengths, scale, new_state)
    qs, ks, dtype = q.shape, k.shape, q.dtype
    n, H, dk, KV, dv = qs[0], qs[-2], qs[-1], ks[-2], v.shape[-1]
    T = qs[1] if len(qs) == 4 else 1
    strides = None
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        q, k, v = _rows(q), _rows(k), _rows(v)
        strides = _strides(q, k, v)
    log_decay = log_decay.contiguous()
    if state is not None:
        state = state.contiguous()
    if lengths is not None:
        lengths = lengths.contiguous()
    dt = _DTYPE[dtype]
    L = _lib.load_library()
    out = torch.empty(qs[:-1] + (dv,), dtype=dtype, device=q.device)
    nb, ws = 0, None
    if T > STEP_TOKENS:
        nb = _lib.check(L.evfly_decay_attention_workspace_bytes(n, T, H, KV, dk, dv, dt, 0))
        ws = _workspace(nb, q)
    _lib.check(L.evfly_decay_attention_forward(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, log_decay.data_ptr(), state.data_ptr() if state is not None else None,
        lengths.data_ptr() if lengths is not None else None, n, T, H, KV, dk, dv, scale, dt, out.data_ptr(), new_state.data_ptr(),
        ws.data_ptr() if ws is not None else None, nb, _rawStream(idx)))
    return out


def _decay_backward(q, k, v, log_decay, state, lengths, scale, d_out, d_state, want_state):
    if q.get_device() != _getDevice():
        with torch.cuda.device(q.device):
            return _decay_backward(q, k, v, log_decay, state, lengths, scale, d_out, d_state, want_state)
    n, T, H, dk = q.shape
    KV, dv = v.shape[2], v.shape[3]
    dt = _DTYPE[q.dtype]
    L = _lib.load_library()
    d_out = torch.zeros((n, T, H, dv), dtype=q.dtype, device=q.device) if d_out is None else d_out.contiguous()
    dq, dk_, dv_ = (torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
    strides = None
    if not (q.is_contiguous() and k.is_contiguous() and v.is_contiguous()):
        q, k, v = _rows(q), _rows(k), _rows(v)
        strides = _strides(q, k, v)
    log_decay, state, lengths, d_state = log_decay.contiguous(), _dense(state), _dense(lengths), _dense(d_state)
    ds = torch.empty_like(state) if want_state else None
    nb = _lib.check(L.evfly_decay_attention_workspace_bytes(n, T, H, KV, dk, dv, dt, 1))
    ws = _workspace(nb, q)
    _lib.check(L.evfly_decay_attention_backward(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, log_decay.data_ptr(), _ptr(state), _ptr(lengths), d_out.data_ptr(), _ptr(d_state),
        n, T, H, KV, dk, dv, scale, dt, dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr(), _ptr(ds), _ptr(ws), nb, _rawStream(q.get_device())))
    return dq, dk_, dv_, ds


def _new_state(q, v):
    return torch.empty((q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1]), dtype=torch.float32, device=q.device)


def _no_second_order(who):
    if torch.is_grad_enabled():
        raise RuntimeError(f"{who}: its gradients have no gradients (create_graph=True)")


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale):
        ctx.set_materialize_grads(False)
        new_state = _new_state(q, v)
        out = _decay_forward(q, k, v, log_decay, state, lengths, scale, new_state)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        return out, new_state

    @staticmethod
    def backward(ctx, d_out, d_state):
        _no_second_order("decay_attention")
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        dq, dk, dv, ds = _decay_backward(q, k, v, log_decay, state, lengths, ctx.scale, d_out, d_state, ctx.needs_input_grad[4])
        return dq, dk, dv, None, ds, None, None


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None):
    """Linear attention with a constant decay per head over the tokens (windows) of every stream:
    S_t = exp(log_decay) * S_{t-1} + k_t v_t^T, out_t = scale * q_t S_t.

    q (streams, tokens, heads, dk), k (streams, tokens, kv_heads, dk), v (streams, tokens, kv_heads, dv), any strides; query head h
    reads key / value head h // (heads // kv_heads). log_decay (heads,) float32: log of the factor per token (0 keeps everything,
    -inf nothing); a constant, without a gradient. state (streams, heads, dk, dv) float32 from the call before, None = zeros.
    lengths (streams,) int32: tokens of each stream that are there, None = all; the others are not read, `out` is zero there.
    scale: dk ** -0.5 if None. Returns (out (streams, tokens, heads, dv), new state). Gradients to q, k, v and state."""
    scale = _check_decay("decay_attention", q, k, v, log_decay, state, lengths, scale, 2)
    recorded = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad))
    if _watched():
        _refuse_unseen("decay_attention", (q, k, v, log_decay, state), recorded)
    if recorded:
        return _DecayAttention.apply(q, k, v, log_decay, state, lengths, scale)
    new_state = _new_state(q, v)
    return _decay_forward(q, k, v, log_decay, state, lengths, scale, new_state), new_state


def decay_attention_step(q, k, v, log_decay, state, lengths=None, scale=None, new_state=None):
    """One token (window) per stream, the serving form: q (streams, heads, dk), k (streams, kv_heads, dk), v (streams, kv_heads, dv)
    against `state` (streams, heads, dk, dv) float32, contiguous, which is updated in place -- or left as it is, with the new state
    written to `new_state` (a pair of buffers used in turn). lengths (streams,) int32: 0 = no token for this stream in this call (its state
    stays, its row of the result is zero). Returns out (streams, heads, dv). No gradients: use `decay_attention` for them."""
    who = "decay_attention_step"
    scale = _check_decay(who, q, k, v, log_decay, state, lengths, scale, 1)
    if state is None or not state.is_contiguous():
        raise ValueError(f"{who}: state must be a contiguous tensor")
    dst = state
    if new_state is not None:
        _check_f32(who, "new_state", new_state, state.shape, q.device)
        if not new_state.is_contiguous():
            raise ValueError(f"{who}: new_state must be a contiguous tensor")
        apart = new_state.data_ptr() - state.data_ptr()
        if apart and abs(apart) < 4 * state.numel():
            raise ValueError(f"{who}: state and new_state overlap in part")
        dst = new_state
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad or dst.requires_grad):
        raise ValueError(f"{who} has no gradients: call decay_attention, or wrap the call in torch.no_grad()")
    if _watched():
        _refuse_unseen(who, (q, k, v, log_decay, state, new_state), False)
    out = _decay_forward(q, k, v, log_decay, state, lengths, scale, dst)
    if not dst.is_inference():                                   # (an inference tensor has no version)
        torch.autograd.graph.increment_version(dst)              # written behind autograd's back
    return out


# ---------------------------------------------------------------------------------------- block norm
def _gate_rows(f, gate):
    """Token rows per gate row: the gate's leading sizes are those of f up to some dimension and 1 behind it (or the gate is one row)."""
    if gate.dim() == 1 and gate.shape[0] == f.shape[-1]:
        return f.numel() // f.shape[-1]
    if gate.dim() == f.dim() and gate.shape[-1] == f.shape[-1]:
        i = 0
        while i < f.dim() - 1 and gate.shape[i] == f.shape[i]:
            i += 1
        if all(s == 1 for s in gate.shape[i:-1]):
            return math.prod(f.shape[i:-1])
    raise ValueError(f"block_norm: a gate {tuple(gate.shape)} for tokens {tuple(f.shape)} (a row (channels,), or f's leading sizes up to some "
                     f"dimension and 1 from there on)")


def _block_forward(f, x, gate, res_scale, w1, b1, w2, b2, opt):
    idx = f.get_device()
    if idx != _getDevice():
        with torch.cuda.device(idx):
            return _block_forward(f, x, gate, res_scale, w1, b1, w2, b2, opt)
    rows_per_gate, gate_f32, act, post, pre, eps = opt
    f = f.contiguous()
    ins = [t if t is None or t.is_contiguous() else t.contiguous() for t in (x, gate, res_scale, w1, b1, w2, b2)]
    px, pg, pa, p1, q1, p2, q2 = [None if t is None else t.data_ptr() for t in ins]
    Cn = f.shape[-1]
    y = torch.empty_like(f)
    h = torch.empty_like(f) if pre else None
    _lib.check(_lib.load_library().evfly_block_norm_forward(
        f.data_ptr(), px, pg, rows_per_gate, gate_f32, act, pa, post, p1, q1, pre, p2, q2, eps, f.numel() // Cn, Cn, _DTYPE[f.dtype], y.data_ptr(),
        h.data_ptr() if pre else None, _rawStream(idx)))
    return y, h


def _block_backward(f, x, gate, res_scale, w1, b1, w2, b2, opt, dy, dh, need):
    if f.get_device() != _getDevice():
        with torch.cuda.device(f.device):
            return _block_backward(f, x, gate, res_scale, w1, b1, w2, b2, opt, dy, dh, need)
    rows_per_gate, gate_f32, act, post, pre, eps = opt
    f, x, gate, res_scale, w1, b1, w2, b2, dy, dh = (f.contiguous(), _dense(x), _dense(gate), _dense(res_scale), _dense(w1), _dense(b1), _dense(w2), _dense(b2),
                                                     _dense(dy), _dense(dh))
    Cn = f.shape[-1]
    rows, dt = f.numel() // Cn, _DTYPE[f.dtype]
    L = _lib.load_library()
    # f's gradient is always formed; of the others what is asked for, the vectors as rows of one tensor
    df = torch.empty_like(f)
    dx = torch.empty_like(x) if x is not None and need[1] else None
    dg = torch.empty_like(gate) if gate is not None and need[2] else None
    if dg is not None and rows == 0:
        dg.zero_()
    vec = [None] * 5
    ask = [i for i, t in enumerate((res_scale, w1, b1, w2, b2)) if t is not None and need[3 + i]]
    if ask:
        for i, t in zip(ask, torch.empty((len(ask), Cn), dtype=torch.float32, device=f.device).unbind(0)):
            vec[i] = t
    nb = _lib.check(L.evfly_block_norm_workspace_bytes(rows, Cn, rows_per_gate, dt))
    ws = _workspace(nb, f)
    _lib.check(L.evfly_block_norm_backward(
        f.data_ptr(), _ptr(x), _ptr(gate), rows_per_gate, gate_f32, act, _ptr(res_scale), post, _ptr(w1), _ptr(b1), pre, _ptr(w2), _ptr(b2), eps, _ptr(dy),
        _ptr(dh), rows, Cn, dt, df.data_ptr(), _ptr(dx), _ptr(dg), *map(_ptr, vec), _ptr(ws), nb, _rawStream(f.get_device())))
    return (df if need[0] else None, dx, dg, *vec, None)


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, x, gate, res_scale, w1, b1, w2, b2, opt):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(f, x, gate, res_scale, w1, b1, w2, b2)
        ctx.opt = opt
        y, h = _block_forward(f, x, gate, res_scale, w1, b1, w2, b2, opt)
        return (y, h) if h is not None else y

    @staticmethod
    def backward(ctx, dy, dh=None):
        _no_second_order("block_norm")
        return _block_backward(*ctx.saved_tensors, ctx.opt, dy, dh, ctx.needs_input_grad)


def _block_fits(f, x, gate, gate_act, res_scale, post, w1, b1, pre, w2, b2):
    """Everything `_refuse_block` asks for, in one look."""
    try:
        dt, dev, shape = f.dtype, f.device, f.shape
        vec = shape[-1:]
        if not (0 < vec[0] <= MAX_CHANNELS and dt in _DTYPE and dev.type == "cuda" and post in _NORM and pre in _NORM and gate_act in _GATE_ACT and
                (x is None or (x.dtype is dt and x.device == dev and x.shape == shape)) and (x is not None or res_scale is None) and
                (post is not None or (w1 is None and b1 is None)) and (pre is not None or (w2 is None and b2 is None)) and
                (gate is None or ((gate.dtype is dt or gate.dtype is torch.float32) and gate.device == dev))):
            return False
        for t in (res_scale, w1, b1, w2, b2):
            if t is not None and (t.dtype is not torch.float32 or t.shape != vec or t.device != dev):
                return False
        return True
    except (AttributeError, IndexError, TypeError):
        return False


def _refuse_block(f, x, gate, gate_act, res_scale, post, w1, b1, pre, w2, b2):
    who = "block_norm"
    if not isinstance(f, torch.Tensor) or f.dim() < 1 or not 1 <= f.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"{who}: f must be a tensor (..., channels) of 1 .. {MAX_CHANNELS} channels")
    _check_tokens(who, (("f", f),) if x is None else (("f", f), ("x", x)), f)
    if x is not None and x.shape != f.shape:
        raise ValueError(f"{who}: x {tuple(x.shape)} is not shaped like f {tuple(f.shape)}")
    if not all(n is None or isinstance(n, str) for n in (post, pre)) or post not in _NORM or pre not in _NORM:
        raise ValueError(f"{who}: norms {post!r}, {pre!r} (\"layer\", \"rms\" or None)")
    if res_scale is not None and x is None:
        raise ValueError(f"{who}: res_scale without a residual x")
    for kind, name, t in ((True, "res_scale", res_scale), (post, "post_weight", w1), (post, "post_bias", b1), (pre, "pre_weight", w2), (pre, "pre_bias", b2)):
        if t is not None:
            if not kind:
                raise ValueError(f"{who}: {name} without a norm")
            _check_f32(who, name, t, f.shape[-1:], f.device)
    if not isinstance(gate_act, str) or gate_act not in _GATE_ACT:
        raise ValueError(f"{who}: gate_act {gate_act!r} (\"none\", \"sigmoid\" or \"tanh\")")
    if gate is not None and (not isinstance(gate, torch.Tensor) or gate.dtype not in (f.dtype, torch.float32) or gate.device != f.device):
        raise ValueError(f"{who}: gate must be a {f.dtype} or float32 tensor on {f.device}")


def block_norm(f, x=None, gate=None, gate_act="none", res_scale=None, post=None, post_weight=None, post_bias=None,
               pre=None, pre_weight=None, pre_bias=None, eps=1e-5):
    """y = res_scale * x + act(gate) * norm_post(f) and h = norm_pre(y) in one pass per token; returns (y, h), h None without `pre`.

    f (..., channels): the sub-layer's output; x: the residual, like f, or None. gate: (channels,), or f's leading sizes up to some
    dimension and 1 behind it ((streams, 1, channels) = one per stream, f's own shape = one per token), in f's type or float32; gate_act
    "none", "sigmoid" or "tanh" of it. res_scale (channels,) float32 times x. post, pre: "layer", "rms" or None = no norm, with
    weight and bias (channels,) float32 or None. h is formed from y before y is rounded to the tokens' type. Gradients to every tensor.
    post=None, pre="layer" without a gate is evfly's LayerNorm(x + f)."""
    _lib.lib()
    if not _block_fits(f, x, gate, gate_act, res_scale, post, post_weight, post_bias, pre, pre_weight, pre_bias):
        _refuse_block(f, x, gate, gate_act, res_scale, post, post_weight, post_bias, pre, pre_weight, pre_bias)
    eps = float(eps)
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError("block_norm: eps is negative or not finite")
    rows_per_gate, gate_f32 = 1, 0
    if gate is not None:
        rows_per_gate, gate_f32 = max(1, _gate_rows(f, gate)), int(gate.dtype is torch.float32)
    opt = (rows_per_gate, gate_f32, _GATE_ACT[gate_act], _NORM[post], _NORM[pre], eps)
    ins = (f, x, gate, res_scale, post_weight, post_bias, pre_weight, pre_bias)
    recorded = False
    if torch.is_grad_enabled():
        for t in ins:
            if t is not None and t.requires_grad:
                recorded = True
                break
    if _watched():
        _refuse_unseen("block_norm", ins, recorded)
    if recorded:
        got = _BlockNorm.apply(*ins, opt)
        return got if isinstance(got, tuple) else (got, None)
    return _block_forward(*ins, opt)
