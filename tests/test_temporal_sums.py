"""The bound that the sums over rows are held to on the GPU: one row that is missing, or there twice, is outside it, at every shape that is tested there."""
import pytest
import torch

from _norm_sums import NAMES, per_gate, sum_bound, sum_terms
from test_gpu_temporal_sums import CASES, inputs


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_a_row_more_or_less_is_outside_the_bound(case):
    d, act = inputs(*case, torch.float32)
    C = d["f"].shape[-1]
    terms = sum_terms(d, act)
    for name in NAMES:
        t, size = (per_gate(x, d, name) for x in terms[name])
        if t.shape[1] == 1:
            continue
        lim = sum_bound(name, size.sum(1), t.shape[0] * t.shape[1], C, act)
        # of the row's channels the one that shows it best
        seen = (t.abs() / lim[:, None]).amax(-1)
        assert seen.min() > 2, (name, seen.min().item())                 # (its term less what rounding may hide)
