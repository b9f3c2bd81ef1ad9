"""Temporal operators on inputs whose sums are exact in fp32 in any order: the result is then the oracle's, to the last bit of its type."""
import pytest
import torch

from oracle import temporal as ot

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
TINY = 2.0 ** -22                   # of 1 + 2^-10 + 2^-22: in the last of its 24 bits, behind the 17 that two bf16 values hold
DIMS = [(32, 32), (64, 64), (128, 128), (128, 32), (40, 72), (33, 65)]


def _same_as_oracle(dtype, q, k, v, state, log_decay=None):
    """A call with gradients (of the last token's first value: sums of one term) and the oracle's: every result the same numbers."""
    from evfly_amd.temporal import decay_attention
    ld = torch.zeros(q.shape[2]) if log_decay is None else log_decay
    lc = [t.to(dtype).cuda().requires_grad_() for t in (q, k, v)] + [state.cuda().requires_grad_()]
    lo = [t.double().requires_grad_() for t in (q, k, v, state)]
    up = torch.zeros(*q.shape[:3], v.shape[-1])
    up[:, -1, :, 0] = 1.0
    out, new = decay_attention(*lc[:3], ld.cuda(), state=lc[3], scale=1.0)
    want, wnew = ot.decay_attention(*lo[:3], ld, lo[3], scale=1.0)
    got = [out, new, *torch.autograd.grad(out, lc, up.to(dtype).cuda())]
    ref = [want, wnew, *torch.autograd.grad(want, lo, up.double())]
    for name, a, b in zip(("out", "new_state", "dq", "dk", "dv", "dstate"), got, ref):
        like = F32 if "state" in name else dtype
        assert a.dtype == like
        assert torch.equal(a.detach().cpu(), b.detach().to(like)), name
    return out


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,dv", DIMS, ids=lambda d: str(d))
@pytest.mark.parametrize("T", [3, 20, 64, 100])
def test_state_enters_the_products_with_all_its_bits(gpu_device, T, dk, dv, dtype):
    """q_t (S[0] - S[1]) = 2^-22 where S[0] = 1 + 2^-10 + 2^-22 and S[1] = 1 + 2^-10: what is left of the state's last bits is the whole result."""
    q, k, v, S = torch.zeros(2, T, 2, dk), torch.zeros(2, T, 1, dk), torch.zeros(2, T, 1, dv), torch.zeros(2, 2, dk, dv)
    q[..., 0], q[..., 1] = 1.0, -1.0
    S[..., 0, :], S[..., 1, :] = 1 + 2.0 ** -10 + TINY, 1 + 2.0 ** -10
    out = _same_as_oracle(dtype, q, k, v, S)
    assert (out.float() == TINY).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,dv", DIMS, ids=lambda d: str(d))
@pytest.mark.parametrize("T", [3, 20, 64, 100])
def test_pair_products_enter_the_sum_with_all_their_bits(gpu_device, T, dk, dv, dtype):
    """Token 0 brings (1 + 2^-10 + 2^-22) v, token 1 -(1 + 2^-10) v: 2^-22 v is left from there on."""
    q, k, v, S = torch.zeros(2, T, 2, dk), torch.zeros(2, T, 1, dk), torch.zeros(2, T, 1, dv), torch.zeros(2, 2, dk, dv)
    q[..., 0], q[..., 1], q[..., 2] = 1.0, 2.0 ** -10, TINY
    k[:, 0, :, :3], k[:, 1, :, :2] = 1.0, 1.0
    v[:, 0], v[:, 1] = 1.0, -1.0
    out = _same_as_oracle(dtype, q, k, v, S)
    assert (out[:, 1:].float() == TINY).all()


@pytest.mark.parametrize("dk,dv", DIMS, ids=lambda d: str(d))
@pytest.mark.parametrize("T", [64, 128, 1024])
def test_a_chunk_is_added_to_the_state_whole(gpu_device, T, dk, dv):
    """fp32: every chunk of 64 tokens adds 64 / 16 = 4 to a state of 2^24, whose neighbours are 2 apart: 4 is there, a token's 1/16 alone would not be. The same
    backwards for the state's gradient."""
    from evfly_amd.temporal import decay_attention
    q, k, v = (torch.full((2, T, h, d), x, device="cuda", requires_grad=True) for h, d, x in ((2, dk, 0.0625), (1, dk, 0.0625), (1, dv, 1.0)))
    S = torch.full((2, 2, dk, dv), 2.0 ** 24, device="cuda", requires_grad=True)
    out, new = decay_attention(q, k, v, torch.zeros(2, device="cuda"), state=S, scale=1.0)
    assert (new == 2.0 ** 24 + T // 16).all()
    assert (torch.autograd.grad([out, new], S, [torch.ones_like(out), torch.full_like(new, 2.0 ** 24)])[0] == 2.0 ** 24 + T // 16).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("C", [32, 256, 2048])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -132])
def test_block_norm_of_rows_whose_mean_square_is_subnormal(gpu_device, eps, kind, C, dtype):
    """+-2^-66: squares 2^-132, which fp32 holds below its normal numbers, so does their mean. eps 0: +-1 back, within the reciprocal root's ulp, the output's
    product and its half step; eps = 2^-132: sqrt(1/2) of it."""
    from evfly_amd.temporal import block_norm
    f = torch.full((5, C), 2.0 ** -66)
    f[:, 1::2] *= -1
    f[3] = 2.0 ** -60 * f[3].sign()                                          # (and one that is not: 2^-120)
    f = f.to(dtype)
    want = f.double() / torch.sqrt(f.double().square().mean(-1, keepdim=True) + eps)
    lv = f.cuda().requires_grad_()
    tol = 4 * 2.0 ** -24 + torch.finfo(dtype).eps / 2
    for got in (block_norm(lv, pre=kind, eps=eps)[1], block_norm(lv, post=kind, eps=eps)[0]):
        assert ((got.detach().double().cpu() - want).abs() <= tol * want.abs()).all()
        assert torch.isfinite(torch.autograd.grad(got[:, 0].sum(), lv)[0]).all()
