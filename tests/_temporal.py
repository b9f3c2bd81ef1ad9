"""Inputs and bounds shared by the tests of the temporal operators."""
import math

import torch

from oracle import temporal as ot

EPS32 = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # finfo(t).eps / 2


def decay_inputs(n, T, H, KV, dk, dv, dtype, seed=0, state=True, lengths=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    d = dict(q=r(n, T, H, dk).to(dtype), k=r(n, T, KV, dk).to(dtype), v=r(n, T, KV, dv).to(dtype))
    d["log_decay"] = torch.tensor([math.log1p(-2.0 ** -(1 + 8 * h / max(1, H - 1))) for h in range(H)])
    d["state"] = r(n, H, dk, dv) if state else None
    d["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    d["d_out"], d["d_state"] = r(n, T, H, dv).to(dtype), r(n, H, dk, dv)
    return d


def decay_exact(d, scale=None, grads=False, d_state=True, absolute=False):
    """The oracle's outputs (and gradients by its own autograd). absolute: the same sums with every term's magnitude, the scale of their rounding."""
    f = (lambda t: None if t is None else t.double().abs()) if absolute else (lambda t: None if t is None else t.double())
    lv = [None if t is None else f(t).clone().requires_grad_(grads) for t in (d["q"], d["k"], d["v"], d["state"])]
    out, S = ot.decay_attention(lv[0], lv[1], lv[2], d["log_decay"], lv[3], d["lengths"], abs(scale) if absolute and scale is not None else scale)
    got = dict(out=out.detach(), new_state=S.detach())
    if grads:
        up = [f(d["d_out"])] + ([f(d["d_state"])] if d_state else [])
        have = [t for t in lv if t is not None]
        gr = torch.autograd.grad([out, S][:len(up)], have, up, allow_unused=True)
        for name, g in zip([m for m, t in zip(("dq", "dk", "dv", "dstate"), lv) if t is not None], gr):
            got[name] = g
    return got


def decay_bound(d, absolute, dtype, is_state, want):
    """Rounding bound of one result, element by element: a chain of `steps` roundings of 2^-24 on the sum of magnitudes -- two inner products of up to 128
    terms, three sums over a chunk of 64, two roundings of the carried state per chunk and head, a weight whose exponent g (t - s) is rounded (a
    weight below e^-100 is nothing) -- and for bf16 tokens the two-part operands (2^-17 each of the pair product, of the state and of
    the final sum's weights) and the result's own rounding."""
    T, H, KV = d["q"].shape[1], d["q"].shape[2], d["k"].shape[2]
    steps = 2 * 128 + 3 * 64 + 2 * (T // 64 + 1) + H // KV + 100 + 16
    e = steps * EPS32 * absolute
    if dtype == torch.bfloat16 and not is_state:
        e = e + 3 * 2.0 ** -17 * absolute + HALF_STEP[dtype] * (want.abs() + 4 * 2.0 ** -17 * absolute)
    return e + 1e-37


def assert_decay(tag, got, want, absolute, d, dtype, is_state):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (tag, got.shape, want.shape)
    assert torch.isfinite(got).all(), tag
    err = (got - want).abs()
    lim = decay_bound(d, absolute, dtype, is_state, want)
    worst = (err / lim).max().item() if err.numel() else 0.0
    assert worst <= 1.0, (tag, worst, err.max().item())
