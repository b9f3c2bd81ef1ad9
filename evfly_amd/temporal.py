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
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPE = {torch.float32: 0, torch.bfloat16: 1}
MAX_HEAD_DIM = 128
MAX_CHANNELS = 8192
STEP_TOKENS = 16                    # up to here a forward needs no workspace (EVFLY_DECAY_STEP_TOKENS)
_NORM = {None: 0, "layer": 1, "rms": 2}


class _on:
    """`with torch.cuda.device(t.device)` that costs nothing where the device is the current one (the usual case)."""

    def __init__(self, t):
        self.prev = torch.cuda.current_device()
        self.dev = t.device.index

    def __enter__(self):
        if self.dev != self.prev:
            torch.cuda.set_device(self.dev)

    def __exit__(self, *exc):
        if self.dev != self.prev:
            torch.cuda.set_device(self.prev)


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


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
def _check_decay(who, q, k, v, log_decay, state, lengths, scale):
    _lib.lib()                                                   # (no GPU / no library: that error first)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{who}: {name} must be a tensor (streams, tokens, heads, head size)")
    _check_tokens(who, (("q", q), ("k", k), ("v", v)), q)
    n, T, H, dk = q.shape
    KV, dv = v.shape[2], v.shape[3]
    if tuple(k.shape) != (n, T, KV, dk) or tuple(v.shape[:2]) != (n, T):
        raise ValueError(f"{who}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if KV == 0 or H == 0 or H % KV:
        raise ValueError(f"{who}: {H} heads do not share {KV} key / value heads evenly")
    if not (1 <= dk <= MAX_HEAD_DIM and 1 <= dv <= MAX_HEAD_DIM):
        raise ValueError(f"{who}: head sizes {dk}, {dv} are not in 1 .. {MAX_HEAD_DIM}")
    _check_f32(who, "log_decay", log_decay, (H,), q.device)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{who}: log_decay is a constant of the head and has no gradient (detach it)")
    if state is not None:
        _check_f32(who, "state", state, (n, H, dk, dv), q.device)
    if lengths is not None and (not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or tuple(lengths.shape) != (n,)
                                or lengths.device != q.device):
        raise ValueError(f"{who}: lengths must be an int32 tensor ({n},) on {q.device}")
    scale = dk ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{who}: scale is not finite")
    return scale


def _rows(t):
    """Rows of a token tensor as the kernels read them: any strides, the last dimension dense."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _strides(q, k, v):
    if q.is_contiguous() and k.is_contiguous() and v.is_contiguous():
        return None
    return (C.c_int64 * 9)(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])


def _decay_forward(q, k, v, log_decay, state, lengths, scale, new_state):
    n, T, H, dk = q.shape
    KV, dv = v.shape[2], v.shape[3]
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    lengths = lengths.contiguous() if lengths is not None else None
    dt = _DTYPE[q.dtype]
    L = _lib.load_library()
    with _on(q):
        out = torch.empty((n, T, H, dv), dtype=q.dtype, device=q.device)
        nb = 0 if T <= STEP_TOKENS else _lib.check(L.evfly_decay_attention_workspace_bytes(n, T, H, KV, dk, dv, dt, 0))
        ws = _workspace(nb, q.device)
        _lib.check(L.evfly_decay_attention_forward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _strides(q, k, v), log_decay.data_ptr(), _lib.ptr(state), _lib.ptr(lengths),
            n, T, H, KV, dk, dv, scale, dt, out.data_ptr(), _lib.ptr(new_state), _lib.ptr(ws), nb, _lib.cur_stream()))
    return out


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale):
        ctx.set_materialize_grads(False)
        n, T, H, dk = q.shape
        new_state = torch.empty((n, H, dk, v.shape[3]), dtype=torch.float32, device=q.device)
        out = _decay_forward(q, k, v, log_decay, state.contiguous() if state is not None else None, lengths, scale, new_state)
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        return out, new_state

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_state):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        n, T, H, dk = q.shape
        KV, dv = v.shape[2], v.shape[3]
        dt = _DTYPE[q.dtype]
        L = _lib.load_library()
        with _on(q):
            d_out = torch.zeros((n, T, H, dv), dtype=q.dtype, device=q.device) if d_out is None else d_out.contiguous()
            d_state = d_state.contiguous() if d_state is not None else None
            qr, kr, vr, g = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
            s_in = state.contiguous() if state is not None else None
            ln = lengths.contiguous() if lengths is not None else None
            dq, dk_, dv_ = (torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
            ds = torch.empty((n, H, dk, dv), dtype=torch.float32, device=q.device) if state is not None and ctx.needs_input_grad[4] else None
            nb = _lib.check(L.evfly_decay_attention_workspace_bytes(n, T, H, KV, dk, dv, dt, 1))
            ws = _workspace(nb, q.device)
            _lib.check(L.evfly_decay_attention_backward(
                qr.data_ptr(), kr.data_ptr(), vr.data_ptr(), _strides(qr, kr, vr), g.data_ptr(), _lib.ptr(s_in), _lib.ptr(ln), d_out.data_ptr(),
                _lib.ptr(d_state), n, T, H, KV, dk, dv, ctx.scale, dt, dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr(), _lib.ptr(ds),
                _lib.ptr(ws), nb, _lib.cur_stream()))
        return dq, dk_, dv_, None, ds, None, None


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None):
    """Linear attention with a constant decay per head over the tokens (windows) of every stream:
    S_t = exp(log_decay) * S_{t-1} + k_t v_t^T, out_t = scale * q_t S_t.

    q (streams, tokens, heads, dk), k (streams, tokens, kv_heads, dk), v (streams, tokens, kv_heads, dv), any strides; query head h
    reads key / value head h // (heads // kv_heads). log_decay (heads,) float32: log of the factor per token (0 keeps everything,
    -inf nothing); a constant, without a gradient. state (streams, heads, dk, dv) float32 from the call before, None = zeros.
    lengths (streams,) int32: tokens of each stream that are there, None = all; the others are not read, `out` is zero there.
    scale: dk ** -0.5 if None. Returns (out (streams, tokens, heads, dv), new state). Gradients to q, k, v and state."""
    scale = _check_decay("decay_attention", q, k, v, log_decay, state, lengths, scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        return _DecayAttention.apply(q, k, v, log_decay, state, lengths, scale)
    n, T, H, dk = q.shape
    new_state = torch.empty((n, H, dk, v.shape[3]), dtype=torch.float32, device=q.device)
    return _decay_forward(q, k, v, log_decay, state.contiguous() if state is not None else None, lengths, scale, new_state), new_state


def decay_attention_step(q, k, v, log_decay, state, lengths=None, scale=None, new_state=None):
    """One token (window) per stream, the serving form: q (streams, heads, dk), k (streams, kv_heads, dk), v (streams, kv_heads, dv)
    against `state` (streams, heads, dk, dv) float32, contiguous, which is updated in place -- or left as it is, with the new state
    written to `new_state` (a pair of buffers used in turn). lengths (streams,) int32: 0 = no token for this stream in this call (its state
    stays, its row of the result is zero). Returns out (streams, heads, dv). No gradients: use `decay_attention` for them."""
    if not all(isinstance(t, torch.Tensor) and t.dim() == 3 for t in (q, k, v)):
        _lib.lib()
        raise ValueError("decay_attention_step: q, k and v must be tensors (streams, heads, head size)")
    q, k, v = q.unsqueeze(1), k.unsqueeze(1), v.unsqueeze(1)
    scale = _check_decay("decay_attention_step", q, k, v, log_decay, state, lengths, scale)
    if state is None or not state.is_contiguous():
        raise ValueError("decay_attention_step: state must be a contiguous tensor")
    dst = state
    if new_state is not None:
        _check_f32("decay_attention_step", "new_state", new_state, state.shape, q.device)
        if not new_state.is_contiguous():
            raise ValueError("decay_attention_step: new_state must be a contiguous tensor")
        dst = new_state
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state, dst)):
        raise ValueError("decay_attention_step has no gradients: call decay_attention, or wrap the call in torch.no_grad()")
    out = _decay_forward(q, k, v, log_decay, state, lengths, scale, dst)
    torch.autograd.graph.increment_version(dst)                  # written behind autograd's back
    return out[:, 0]


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


def _block_args(f, x, gate, res_scale, vecs, opt):
    gate_f32 = gate is not None and gate.dtype == torch.float32
    return (f.data_ptr(), _lib.ptr(x), _lib.ptr(gate), opt["rows_per_gate"], int(gate_f32), opt["act"], _lib.ptr(res_scale), opt["post"],
            _lib.ptr(vecs[0]), _lib.ptr(vecs[1]), opt["pre"], _lib.ptr(vecs[2]), _lib.ptr(vecs[3]), opt["eps"])


def _block_forward(f, x, gate, res_scale, vecs, opt):
    Cn = f.shape[-1]
    rows = f.numel() // Cn
    with _on(f):
        y = torch.empty(f.shape, dtype=f.dtype, device=f.device)
        h = torch.empty(f.shape, dtype=f.dtype, device=f.device) if opt["pre"] else None
        _lib.check(_lib.load_library().evfly_block_norm_forward(*_block_args(f, x, gate, res_scale, vecs, opt), rows, Cn, _DTYPE[f.dtype],
                                                                y.data_ptr(), _lib.ptr(h), _lib.cur_stream()))
    return y, h


def _dense(t):
    return t.contiguous() if t is not None else None


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, x, gate, res_scale, w1, b1, w2, b2, opt):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(f, x, gate, res_scale, w1, b1, w2, b2)
        ctx.opt = opt
        y, h = _block_forward(_dense(f), _dense(x), _dense(gate), _dense(res_scale), [_dense(t) for t in (w1, b1, w2, b2)], opt)
        return (y, h) if h is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        opt, need = ctx.opt, ctx.needs_input_grad
        ins = [_dense(t) for t in ctx.saved_tensors]
        f, x, gate = ins[:3]
        Cn = f.shape[-1]
        rows = f.numel() // Cn
        L = _lib.load_library()
        with _on(f):
            dy, dh = _dense(dy), _dense(dh)
            # f's gradient is always formed; of the others what was asked for. (no rows: the kernels write the vectors' zeros, a gate's come from here)
            g = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and (i == 0 or need[i]) else None
                 for i, t in enumerate(ins)]
            if rows == 0 and g[2] is not None:
                g[2].zero_()
            nb = _lib.check(L.evfly_block_norm_workspace_bytes(rows, Cn, opt["rows_per_gate"], _DTYPE[f.dtype]))
            ws = _workspace(nb, f.device)
            _lib.check(L.evfly_block_norm_backward(*_block_args(f, x, gate, ins[3], ins[4:], opt), _lib.ptr(dy), _lib.ptr(dh), rows, Cn, _DTYPE[f.dtype],
                                                   g[0].data_ptr(), _lib.ptr(g[1]), _lib.ptr(g[2]), _lib.ptr(g[3]), _lib.ptr(g[4]), _lib.ptr(g[5]),
                                                   _lib.ptr(g[6]), _lib.ptr(g[7]), _lib.ptr(ws), nb, _lib.cur_stream()))
        return (*[t if need[i] else None for i, t in enumerate(g)], None)


def block_norm(f, x=None, gate=None, gate_act="none", res_scale=None, post=None, post_weight=None, post_bias=None,
               pre=None, pre_weight=None, pre_bias=None, eps=1e-5):
    """y = res_scale * x + act(gate) * norm_post(f) and h = norm_pre(y) in one pass per token; returns (y, h), h None without `pre`.

    f (..., channels): the sub-layer's output; x: the residual, like f, or None. gate: (channels,), or f's leading sizes up to some
    dimension and 1 behind it ((streams, 1, channels) = one per stream, f's own shape = one per token), in f's type or float32; gate_act
    "none", "sigmoid" or "tanh" of it. res_scale (channels,) float32 times x. post, pre: "layer", "rms" or None = no norm, with
    weight and bias (channels,) float32 or None. h is formed from y before y is rounded to the tokens' type. Gradients to every tensor.
    post=None, pre="layer" without a gate is evfly's LayerNorm(x + f)."""
    _lib.lib()
    if not isinstance(f, torch.Tensor) or f.dim() < 1 or not 1 <= f.shape[-1] <= MAX_CHANNELS:
        raise ValueError(f"block_norm: f must be a tensor (..., channels) of 1 .. {MAX_CHANNELS} channels")
    _check_tokens("block_norm", (("f", f),) if x is None else (("f", f), ("x", x)), f)
    Cn = f.shape[-1]
    if x is not None and x.shape != f.shape:
        raise ValueError(f"block_norm: x {tuple(x.shape)} is not shaped like f {tuple(f.shape)}")
    if post not in _NORM or pre not in _NORM:
        raise ValueError(f"block_norm: norms {post!r}, {pre!r} (\"layer\", \"rms\" or None)")
    if res_scale is not None and x is None:
        raise ValueError("block_norm: res_scale without a residual x")
    for kind, name, t in ((True, "res_scale", res_scale), (post, "post_weight", post_weight), (post, "post_bias", post_bias),
                          (pre, "pre_weight", pre_weight), (pre, "pre_bias", pre_bias)):
        if t is not None:
            if not kind:
                raise ValueError(f"block_norm: {name} without a norm")
            _check_f32("block_norm", name, t, (Cn,), f.device)
    if gate_act not in ("none", "sigmoid", "tanh"):
        raise ValueError(f"block_norm: gate_act {gate_act!r} (\"none\", \"sigmoid\" or \"tanh\")")
    eps = float(eps)
    if not (math.isfinite(eps) and eps >= 0.0):
        raise ValueError("block_norm: eps is negative or not finite")
    rows_per_gate = 1
    if gate is not None:
        if not isinstance(gate, torch.Tensor) or gate.dtype not in (f.dtype, torch.float32) or gate.device != f.device:
            raise ValueError(f"block_norm: gate must be a {f.dtype} or float32 tensor on {f.device}")
        rows_per_gate = max(1, _gate_rows(f, gate))
    opt = dict(rows_per_gate=rows_per_gate, act=_lib.ACT_CODES[gate_act], post=_NORM[post], pre=_NORM[pre], eps=eps)
    ins = (f, x, gate, res_scale, post_weight, post_bias, pre_weight, pre_bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ins):
        got = _BlockNorm.apply(*ins, opt)
        return got if isinstance(got, tuple) else (got, None)
    return _block_forward(*[_dense(t) for t in ins[:4]], [_dense(t) for t in ins[4:]], opt)
