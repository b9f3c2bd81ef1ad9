"""Calls of the temporal operators' public entries that are refused, and rarely made ones that are not."""
import pytest
import torch

from _temporal import decay_inputs
from test_gpu_temporal import _compare, _cuda

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


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


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("state", [True, False], ids=["state", "no_state"])
@pytest.mark.parametrize("T", [1, 9, 100, 520])
def test_decay_gradients_at_extreme_decays(gpu_device, T, state, dtype):
    """No decay, none kept (-inf), one that underflows within a chunk, one that grows: every result and gradient against the oracle, the state's among them."""
    d = decay_inputs(2, T, 4, 2, 24, 32, dtype, seed=31, state=state)
    d["log_decay"] = torch.tensor([0.0, float("-inf"), -30.0, 0.01])
    got = _compare(d, dtype, grads=True)
    if state:
        assert not got["dstate"][:, 1].any()                                 # (nothing of it is kept, so nothing comes back)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(64, 64), (32, 33), (33, 32), (32, 32), (128, 100)], ids=lambda x: str(x))
@pytest.mark.parametrize("T", [10, 11, 12, 13, 15, 16, 17])
def test_decay_where_the_recurrence_ends(gpu_device, T, dk, dv, dtype):
    """Token counts on both sides of the change from the recurrence to chunks (11 / 12 for wide bf16 heads, 16 / 17 otherwise), padded streams among them."""
    _compare(decay_inputs(3, T, 4, 2, dk, dv, dtype, seed=32, lengths=[T, 0, T - 1]), dtype, grads=True)


def test_tensors_of_another_device_than_the_current_one(gpu_device, monkeypatch):
    """The current device is taken for another one on the first look: the call goes on under the tensors' own."""
    from evfly_amd import temporal
    d = _cuda(decay_inputs(2, 40, 4, 2, 32, 32, F32, seed=33))

    def run():
        lv = [d[m].detach().requires_grad_() for m in ("q", "k", "v", "state")]
        out, S = temporal.decay_attention(*lv[:3], d["log_decay"], state=lv[3])
        y, h = temporal.block_norm(out, lv[0], pre="layer")
        step = temporal.decay_attention_step(*(d[m][:, 0] for m in "qkv"), d["log_decay"], d["state"], new_state=torch.empty_like(d["state"]))
        return [out, S, y, h, step, *torch.autograd.grad([y, h, S], lv, [d["d_out"], d["d_out"], d["d_state"]])]

    want, seen, true = run(), [], temporal._getDevice

    def other():
        seen.append(None)
        return true() + len(seen) % 2

    monkeypatch.setattr(temporal, "_getDevice", other)
    got = run()
    assert len(seen) == 10 and all(torch.equal(a, b) for a, b in zip(got, want))      # (five calls of the library, each looked at twice)


def test_block_norm_of_strided_rows_with_weights(gpu_device):
    """Slices and transposed tensors, the weights as every second value of a vector: both results and every gradient are the dense tensors'."""
    from evfly_amd.temporal import block_norm
    g = torch.Generator().manual_seed(34)
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    a, x, gate, dy = r(8, 6, 40), r(6, 8, 40).transpose(0, 1), r(8, 64)[:, None, ::2], r(6, 8, 32).transpose(0, 1)
    vec = [(1 + 0.1 * r(64))[::2] for _ in range(5)]
    ins = [a[..., 1:33], x[..., 3:35], gate, *vec]

    def run(ins):
        lv = [t.detach().requires_grad_() for t in ins]
        f, x, gate, al, w1, b1, w2, b2 = lv
        y, h = block_norm(f, x, gate, "sigmoid", al, post="rms", post_weight=w1, post_bias=b1, pre="layer", pre_weight=w2, pre_bias=b2)
        return [y, h, *torch.autograd.grad([y, h], lv, [dy, dy])]

    assert not any(t.is_contiguous() for t in ins)
    assert all(torch.equal(p, q) for p, q in zip(run(ins), run([t.contiguous() for t in ins])))
