"""Oracle of the temporal operators: their definitions token by token in 64 bits (torch on the CPU, differentiable)."""
import torch


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None):
    """S_t = exp(log_decay) S_{t-1} + k_t v_t^T, out_t = scale q_t S_t; (out, state behind each stream's last token)."""
    n, T, H, dk = q.shape
    KV, dv = v.shape[2], v.shape[3]
    head = torch.arange(H) // (H // KV)
    q, k, v = q.double(), k.double()[:, :, head], v.double()[:, :, head]
    scale = dk ** -0.5 if scale is None else scale
    keep = torch.exp(log_decay.double())[None, :, None, None]
    S = torch.zeros(n, H, dk, dv, dtype=torch.float64) if state is None else state.double()
    lens = torch.full((n,), T) if lengths is None else lengths.long()
    outs = []
    for t in range(T):
        live = (t < lens)[:, None, None]
        new = torch.where(keep > 0, keep * S, torch.zeros_like(S)) + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(live[..., None], new, S)
        outs.append(torch.where(live, scale * (q[:, t, :, :, None] * S).sum(-2), torch.zeros(())))
    out = torch.stack(outs, 1) if outs else torch.zeros(n, 0, H, dv, dtype=torch.float64)
    return out, S


def _norm(x, kind, weight, bias, eps):
    if kind is None:
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    x = x if weight is None else x * weight.double()
    return x if bias is None else x + bias.double()


def block_norm(f, x=None, gate=None, gate_act="none", res_scale=None, post=None, post_weight=None, post_bias=None, pre=None, pre_weight=None,
               pre_bias=None, eps=1e-5):
    """y = res_scale x + act(gate) norm_post(f), h = norm_pre(y) (None without a pre norm)."""
    y = _norm(f.double(), post, post_weight, post_bias, eps)
    if gate is not None:
        y = y * {"none": lambda z: z, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[gate_act](gate.double())
    if x is not None:
        y = y + (x.double() if res_scale is None else x.double() * res_scale.double())
    return y, _norm(y, pre, pre_weight, pre_bias, eps) if pre else None
