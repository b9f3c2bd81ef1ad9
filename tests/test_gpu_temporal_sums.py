"""Sums over rows in block norm's gradients, held to a bound that one missing row exceeds (tests/test_temporal_sums.py shows that it does)."""
import pytest
import torch

from _norm_sums import NAMES, per_gate, sum_bound, sum_terms
from test_gpu_temporal import F32, BF16, HALF_STEP, _norm_call, _norm_inputs

pytestmark = pytest.mark.gpu

# (streams, tokens, channels, gate): one gate row for all, per stream, per token; more rows than the blocks hold at once, fewer in a stream than in a block
CASES = [(s, t, c, g) for s, t, c in ((1, 5000, 64), (2, 3001, 128), (700, 3, 32), (600, 9, 64), (40, 100, 2048), (7, 401, 72), (3, 700, 1000), (1, 4000, 24), (1, 600, 8192))
         for g in ("channel", "stream")]


def inputs(streams, tokens, C, gate, dtype):
    act = "tanh" if gate == "stream" else "none"
    return _norm_inputs((streams, tokens), C, dtype, ((streams, 1), dtype) if gate == "stream" else ((), F32), 40), act


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_block_norm_sums_over_rows(gpu_device, case, dtype):
    from evfly_amd.temporal import block_norm
    d, act = inputs(*case, dtype)
    C = d["f"].shape[-1]
    got = _norm_call(block_norm, d, act, "layer", "layer", 1e-5, lambda t: t.cuda())
    terms = sum_terms(d, act)
    for name in NAMES:
        t, size = (per_gate(x, d, name) for x in terms[name])
        want = t.sum(1)
        lim = sum_bound(name, size.sum(1), t.shape[0] * t.shape[1], C, act)
        if got[name].dtype == BF16:
            lim = lim + HALF_STEP[BF16] * (want.abs() + lim)
        err = (got[name].double().cpu().reshape(want.shape) - want).abs()
        assert (err <= lim).all(), (name, (err / lim).max().item())
