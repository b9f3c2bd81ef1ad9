"""Column sums of block norm's gradients: their terms row by row in 64 bits, and a bound on what rounding may do to each sum.

y = al x + a u, u = w1 fh + b1, fh = r1 (f - mean f), h = w2 yh + b2, yh = r2 (y - mean y); dh, dy come in. With g = w2 dh and means over the channels,
    dyt = dy + r2 (g - mean g - yh mean(g yh))                                  (the gradient of y from both outputs)
    d_pre_weight  sum dh yh       d_pre_bias  sum dh        d_res_scale  sum dyt x
    d_post_weight sum dyt a fh    d_post_bias sum dyt a     d_gate       sum dyt u act'(gate)
"""
import torch

from _temporal import EPS32

NAMES = ("d_res_scale", "d_post_weight", "d_post_bias", "d_pre_weight", "d_pre_bias", "d_gate")


def sum_terms(d, act="none", post="layer", pre="layer", eps=1e-5):
    """{name: (terms, magnitudes)}, both (rows, channels): `magnitudes` is the same expression with every product's and every sum's parts taken by size, the scale of the
    roundings of a term in fp32."""
    C = d["f"].shape[-1]
    rows = d["f"].numel() // C
    f, x, dy, dh = (d[m].double().reshape(rows, C) for m in ("f", "x", "dy", "dh"))
    al, w1, b1, w2 = (d[m].double() for m in ("res_scale", "post_weight", "post_bias", "pre_weight"))
    z = d["gate"].double().expand(d["f"].shape).reshape(rows, C)
    a = {"none": z, "sigmoid": torch.sigmoid(z), "tanh": torch.tanh(z)}[act]
    slope = {"none": torch.ones_like(z), "sigmoid": a * (1 - a), "tanh": 1 - a * a}[act]
    slope_size = torch.ones_like(z) if act == "none" else a.abs() if act == "sigmoid" else 1 + a * a
    mean = lambda t: t.mean(-1, keepdim=True)

    def norm(t, size, kind):
        c = t - mean(t) if kind == "layer" else t
        r = 1 / torch.sqrt(mean(c * c) + eps)
        return c * r, r * (size + mean(size) if kind == "layer" else size), r

    fh, Fh, r1 = norm(f, f.abs(), post)
    u, U = fh * w1 + b1, Fh * w1.abs() + b1.abs()
    y, Y = al * x + a * u, (al * x).abs() + a.abs() * U
    yh, Yh, r2 = norm(y, Y, pre)
    g = dh * w2
    layer = pre == "layer"
    dyt = dy + r2 * (g - (mean(g) if layer else 0) - yh * mean(g * yh))
    D = dy.abs() + r2 * (g.abs() + (mean(g.abs()) if layer else 0) + Yh * mean(g.abs() * Yh))
    return dict(d_res_scale=(dyt * x, D * x.abs()), d_post_weight=(dyt * a * fh, D * a.abs() * Fh), d_post_bias=(dyt * a, D * a.abs()), d_pre_weight=(dh * yh, dh.abs() * Yh),
                d_pre_bias=(dh, dh.abs()), d_gate=(dyt * u * slope, D * U * slope_size))


def per_gate(t, d, name):
    """Rows of one sum next to each other: (sums, rows of each, channels)."""
    C = t.shape[-1]
    return t.reshape(d["gate"].numel() // C if name == "d_gate" else 1, -1, C)


def sum_bound(name, magnitudes, rows, C, act):
    """Roundings (2^-24 each) times magnitudes. In a term: a mean or a sum over the channels is eight values of a lane, at most six lane exchanges and sixteen waves, then
    its factor; two norms lie in a row (the second one's mean square is of values that carry the first one's error), each with a mean, a mean square, a root and its
    products, and the backward of the second has two means more: six such sums, some sixty products and differences. tanh and exp some ulp. Adding the
    terms: a lane's rows, at most 4 rows / (lanes' groups x blocks) + 2, exchanges and groups of a block (8), a sixteenth of 512 blocks, sixteen runs."""
    G = 4
    while G * 8 < C:
        G *= 2
    channels = 8 + min(6, G.bit_length()) + max(0, G // 64)
    term = 0 if name == "d_pre_bias" else 3 * channels + 30 if name == "d_pre_weight" else 6 * channels + 60 + (8 if act != "none" else 0)
    adds = 4 * rows / (256 * max(1, 256 // G)) + 2 + 8 + 32 + 16
    return (term + adds) * EPS32 * magnitudes
