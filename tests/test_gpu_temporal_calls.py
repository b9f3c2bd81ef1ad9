"""Calls of the temporal operators' public entries that are refused, and rarely made ones that are not."""
import pytest
import torch

from _temporal import decay_inputs

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _cuda(d):
    return {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in d.items()}


def test_k_and_v_of_another_rank_are_refused(gpu_device):
    from evfly_amd.temporal import decay_attention, decay_attention_step
    z = lambda *s: torch.zeros(*s, device="cuda")
    for q, k, v in ((z(4, 8, 32), z(4, 32), z(4, 32)), (z(4, 8, 32), z(4, 2, 8, 32), z(4, 2, 8, 32)), (z(4, 8, 32), z(4, 8, 32), z(4, 2, 8, 32))):
        with pytest.raises(ValueError):
            decay_attention_step(q, k, v, z(8), z(4, 8, 32, 32))
    for q, k, v in ((z(2, 100, 8, 64), z(2, 100, 2, 8, 64), z(2, 100, 2, 8, 64)), (z(2, 4, 4, 64), z(2, 4, 64), z(2, 4, 4, 64)), (z(2, 4, 4, 64), z(2, 4, 4, 64), z(2, 4, 64))):
        with pytest.raises(ValueError):
            decay_attention(q, k, v, z(q.shape[2]))


def test_states_that_overlap_in_part_are_refused(gpu_device):
    """Shifted views of one buffer are refused; neighbouring ones and the same one are not."""
    from evfly_amd.temporal import decay_attention_step
    d = _cuda(decay_inputs(4, 1, 2, 2, 32, 32, F32, seed=30))
    q, k, v = (d[m][:, 0] for m in "qkv")
    buf = torch.zeros(9, 2, 32, 32, device="cuda")
    buf[:4] = d["state"]
    for a, b in ((buf[:4], buf[1:5]), (buf[1:5], buf[:4])):
        with pytest.raises(ValueError, match="overlap"):
            decay_attention_step(q, k, v, d["log_decay"], a, new_state=b)
    out = decay_attention_step(q, k, v, d["log_decay"], buf[:4], new_state=buf[4:8])
    assert torch.equal(buf[:4], d["state"]) and not buf[8].any()
    assert torch.equal(decay_attention_step(q, k, v, d["log_decay"], d["state"]), out) and torch.equal(d["state"], buf[4:8])
