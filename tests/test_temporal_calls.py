"""Calls of the temporal operators that must not reach the device, on the CPU: stand-ins carry shapes, types and devices, the library's entries are replaced."""
import itertools
import types

import pytest
import torch

from evfly_amd import temporal

DEV = torch.device("cuda", 0)


def _like(*shape, dtype=torch.float32):
    return types.SimpleNamespace(shape=torch.Size(shape), dtype=dtype, device=DEV, requires_grad=False)


def _ranks(t, lead):
    """The shape with a dimension too few or too many that agrees wherever leading and last sizes are compared."""
    first, last = t[:lead], t[lead:]
    yield t[1:]
    yield first + last[1:]
    yield first + last[:1]
    yield first + (2,) + last
    yield first + last[:1] + (2,) + last[1:]
    yield t + t[-1:]
    yield (1,) + t
    yield t[:1] + t[-1:]


@pytest.mark.parametrize("lead", [1, 2])
def test_k_and_v_of_another_rank_do_not_fit(lead):
    n, H, KV, dk, dv = 4, 8, 4, 32, 32
    lead_sizes = (n, 4)[:lead]
    q, k, v = lead_sizes + (H, dk), lead_sizes + (KV, dk), lead_sizes + (KV, dv)
    ld = _like(H)
    fits = lambda a, b, c: temporal._decay_fits(_like(*a), _like(*b), _like(*c), ld, None, None, lead)
    assert fits(q, k, v)
    for a, b, c in itertools.product([q, *_ranks(q, lead)], [k, *_ranks(k, lead)], [v, *_ranks(v, lead)]):
        if (a, b, c) != (q, k, v):
            assert not (fits(a, b, c) and not (len(a) == len(b) == len(c) == lead + 2)), (a, b, c)
    # the ones that agree in every size that is compared
    assert not fits((4, 8, 32), (4, 32), (4, 32)) if lead == 1 else not fits((2, 100, 8, 64), (2, 100, 2, 8, 64), (2, 100, 2, 8, 64))


def test_k_and_v_of_another_rank_are_refused():
    """The message's own path, on tensors without a device (the ranks are looked at first)."""
    z = torch.zeros
    for lead, bad in ((1, [(z(4, 8, 32), z(4, 32), z(4, 32)), (z(4, 8, 32), z(4, 8, 32), z(4, 2, 8, 32))]),
                      (2, [(z(2, 3, 8, 16), z(2, 3, 2, 8, 16), z(2, 3, 2, 8, 16)), (z(2, 4, 4, 16), z(2, 4, 16), z(2, 4, 4, 16))])):
        for q, k, v in bad:
            with pytest.raises(ValueError, match="must be a tensor"):
                temporal._refuse_decay("decay_attention", q, k, v, z(8), None, None, lead)
