"""GPU parity of the temporal operators against the 64-bit oracle: sizes where tiles, chunks and segments end, head layouts, strides, lengths, states, streams, graphs."""
import math

import pytest
import torch

from _temporal import EPS32, HALF_STEP, assert_decay, decay_exact, decay_inputs
from oracle import temporal as ot

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _cuda(d, grad=False):
    c = {k: t.cuda() if isinstance(t, torch.Tensor) else t for k, t in d.items()}
    if grad:
        for m in ("q", "k", "v", "state"):
            if c[m] is not None:
                c[m].requires_grad_()
    return c


def _run_decay(d, scale=None, grads=False, d_state=True):
    from evfly_amd.temporal import decay_attention
    c = _cuda(d, grads)
    out, S = decay_attention(c["q"], c["k"], c["v"], c["log_decay"], state=c["state"], lengths=c["lengths"], scale=scale)
    got = dict(out=out, new_state=S)
    if grads:
        have = [m for m in ("q", "k", "v", "state") if c[m] is not None]
        outs, ups = ([out, S], [c["d_out"], c["d_state"]]) if d_state else ([out], [c["d_out"]])
        for m, g in zip(have, torch.autograd.grad(outs, [c[m] for m in have], ups)):
            got["d" + m] = g
    return got


def _compare(d, dtype, scale=None, grads=False, d_state=True):
    want, mag = decay_exact(d, scale, grads, d_state), decay_exact(d, scale, grads, d_state, absolute=True)
    got = _run_decay(d, scale, grads, d_state)
    assert set(got) == set(want)
    for m in want:
        state = m in ("new_state", "dstate")
        assert got[m].dtype == (F32 if state else dtype), m
        assert_decay(m, got[m], want[m], mag[m], d, dtype, state)
    return got


# (streams, tokens, heads, kv heads, dk, dv): one token, the recurrent form's end, chunk ends, segment ends, odd and whole head sizes
SHAPES = [(3, 1, 4, 4, 32, 32), (2, 1, 2, 1, 17, 5), (2, 2, 1, 1, 1, 1), (2, 15, 3, 3, 40, 72), (2, 16, 4, 2, 128, 128), (2, 17, 4, 2, 32, 32), (1, 63, 2, 2, 64, 64),
          (2, 64, 2, 1, 48, 96), (1, 65, 3, 1, 33, 65), (1, 128, 2, 2, 128, 64), (2, 130, 2, 2, 8, 128), (1, 257, 2, 2, 64, 31), (1, 600, 4, 1, 127, 128), (3, 515, 2, 2, 96, 40)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_decay_forward(gpu_device, shape, dtype):
    _compare(decay_inputs(*shape, dtype, seed=1), dtype)
    _compare(decay_inputs(*shape, dtype, seed=2, state=False), dtype, scale=1.7)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_decay_gradients(gpu_device, shape, dtype):
    _compare(decay_inputs(*shape, dtype, seed=3), dtype, grads=True)
    _compare(decay_inputs(*shape, dtype, seed=4, state=False), dtype, scale=-0.3, grads=True, d_state=False)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T,lengths", [(1, [0, 1, 1, 0]), (10, [0, 10, 3, 9]), (70, [0, 1, 64, 70]), (600, [0, 255, 257, 600]), (600, [599, 1, 65, 512])])
def test_decay_lengths_and_padding(gpu_device, T, lengths, dtype):
    """What lies behind a stream's length -- NaN, infinities, the lowest value -- is not read; its results are zero; its state is the one behind its last token."""
    d = decay_inputs(4, T, 2, 1, 40, 24, dtype, seed=5, lengths=lengths)
    clean = _compare(d, dtype, grads=True)
    dirty = dict(d)
    for m, bad in (("q", float("nan")), ("k", float("inf")), ("v", torch.finfo(dtype).min), ("d_out", float("nan"))):
        t = d[m].clone()
        for i, L in enumerate(lengths):
            t[i, L:] = bad
        dirty[m] = t
    got = _run_decay(dirty, grads=True)
    for m in clean:
        assert torch.equal(got[m], clean[m]), m
    for i, L in enumerate(lengths):
        for m in ("out", "dq", "dk", "dv"):
            assert not got[m][i, L:].any(), m
        if L == 0:
            assert torch.equal(got["new_state"][i].cpu(), d["state"][i]) and torch.equal(got["dstate"][i].cpu(), d["d_state"][i])


def test_decay_lengths_outside_the_range_are_taken_into_it(gpu_device):
    for T in (5, 80):
        a = _run_decay(decay_inputs(2, T, 2, 2, 16, 16, F32, seed=6, lengths=[-3, T + 9]), grads=True)
        b = _run_decay(decay_inputs(2, T, 2, 2, 16, 16, F32, seed=6, lengths=[0, T]), grads=True)
        assert all(torch.equal(a[m], b[m]) for m in a)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T", [1, 9, 100, 520])
def test_decay_extreme_decays(gpu_device, T, dtype):
    """No decay, none kept (-inf), one that underflows within a chunk, one that grows (short)."""
    d = decay_inputs(2, T, 4, 2, 24, 32, dtype, seed=7)
    d["log_decay"] = torch.tensor([0.0, float("-inf"), -30.0, 0.01])
    _compare(d, dtype)
    d["state"] = None
    got = _run_decay(d, grads=True)
    want, mag = decay_exact(d, grads=False), decay_exact(d, absolute=True)
    assert_decay("out", got["out"], want["out"], mag["out"], d, dtype, False)
    assert all(torch.isfinite(t).all() for t in got.values())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("T", [1, 40, 300])
def test_decay_strides(gpu_device, T, dtype):
    """Slices of one projection, head-major tensors, expanded heads and a last dimension that is not dense give the contiguous tensors' bits."""
    from evfly_amd.temporal import decay_attention
    n, H, dk = 2, 4, 32
    g = torch.Generator().manual_seed(8)
    ld = torch.tensor([-0.5, -0.1, -0.01, -0.001]).cuda()
    qkv = torch.randn(n, T, 3 * H * dk, generator=g).to(dtype).cuda()
    q, k, v = (t.unflatten(-1, (H, dk)) for t in qkv.chunk(3, -1))
    ref = decay_attention(q.contiguous(), k.contiguous(), v.contiguous(), ld)
    cases = {"slices": (q, k, v), "head_major": tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)),
             "not_dense": tuple(t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)),
             "unaligned": tuple(torch.cat([t.new_zeros(n, T, H, 1), t], -1)[..., 1:] for t in (q, k, v))}
    for name, (a, b, c) in cases.items():
        got = decay_attention(a, b, c, ld)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1]), name
        lv = [t.detach().requires_grad_() for t in (a, b, c)]
        lr = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
        up = torch.randn(n, T, H, dk, generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
        for x, y in zip(torch.autograd.grad(decay_attention(*lv, ld)[0], lv, up.transpose(1, 2).contiguous().transpose(1, 2)),
                        torch.autograd.grad(decay_attention(*lr, ld)[0], lr, up)):
            assert torch.equal(x, y), name
    one = k[:, :, :1]
    got = decay_attention(q, one.expand(n, T, H, dk), v[:, :, :1].expand(n, T, H, dk), ld)
    sh = decay_attention(q, one, v[:, :, :1], ld)
    assert torch.equal(got[0], sh[0]) and torch.equal(got[1], sh[1])


def test_decay_state_carries_a_recording(gpu_device):
    """In pieces -- windows one by one in place, a few at a time, chunks -- a recording gives what it gives at once."""
    from evfly_amd.temporal import decay_attention, decay_attention_step
    d = decay_inputs(3, 300, 4, 2, 32, 64, F32, seed=10)
    want, mag = decay_exact(d), decay_exact(d, absolute=True)
    c = _cuda(d)
    S, outs, at = c["state"].clone(), [], 0
    for T in (1, 1, 1, 7, 16, 17, 64, 100, 93):
        sl = [c[m][:, at:at + T] for m in "qkv"]
        if T == 1:
            before = S._version
            outs.append(decay_attention_step(*[t[:, 0] for t in sl], c["log_decay"], S)[:, None])
            assert S._version > before
        else:
            o, S = decay_attention(*sl, c["log_decay"], state=S)
            outs.append(o)
        at += T
    assert at == 300
    assert_decay("out", torch.cat(outs, 1), want["out"], mag["out"], d, F32, False)
    assert_decay("state", S, want["new_state"], mag["new_state"], d, F32, True)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 48), (128, 128), (5, 7), (100, 33), (40, 101)])
def test_decay_step(gpu_device, dk, dv, dtype):
    from evfly_amd.temporal import decay_attention_step
    d = decay_inputs(5, 1, 4, 2, dk, dv, dtype, seed=11, lengths=[1, 0, 1, 1, 1])
    want, mag = decay_exact(d), decay_exact(d, absolute=True)
    c = _cuda(d)
    q, k, v = (c[m][:, 0] for m in "qkv")
    keep, new = c["state"].clone(), torch.full_like(c["state"], float("nan"))
    out = decay_attention_step(q, k, v, c["log_decay"], c["state"], lengths=c["lengths"], new_state=new)
    assert torch.equal(c["state"], keep)
    assert_decay("out", out[:, None], want["out"], mag["out"], d, dtype, False)
    assert_decay("state", new, want["new_state"], mag["new_state"], d, dtype, True)
    out2 = decay_attention_step(q, k, v, c["log_decay"], c["state"], lengths=c["lengths"])
    assert torch.equal(out2, out) and torch.equal(c["state"], new)


def test_decay_state_in_place_through_the_abi(gpu_device):
    """state_out may be state_in, also where the sequence runs in segments side by side."""
    from evfly_amd import _lib
    L = _lib.lib()
    for T in (4, 90, 2000):
        d = _cuda(decay_inputs(2, T, 2, 2, 64, 64, F32, seed=12))
        nb = L.evfly_decay_attention_workspace_bytes(2, T, 2, 2, 64, 64, 0, 0)
        ws = torch.empty(max(nb, 1), dtype=torch.uint8, device="cuda")
        res = []
        for same in (False, True):
            S, out = d["state"].clone(), torch.empty(2, T, 2, 64, device="cuda")
            S2 = S if same else torch.empty_like(S)
            _lib.check(L.evfly_decay_attention_forward(d["q"].data_ptr(), d["k"].data_ptr(), d["v"].data_ptr(), None, d["log_decay"].data_ptr(), S.data_ptr(), None, 2, T, 2, 2,
                                                       64, 64, 0.125, 0, out.data_ptr(), S2.data_ptr(), ws.data_ptr(), nb, _lib.cur_stream()))
            res.append((out, S2))
        assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


def test_decay_positions_behind_2_to_31_elements(gpu_device):
    """Rows 2^25 elements apart: offsets pass 32 bits in elements and bytes."""
    from evfly_amd.temporal import decay_attention
    T, step = 70, 1 << 25
    big = torch.empty(T * step, dtype=BF16, device="cuda")
    d = decay_inputs(1, T, 1, 1, 32, 32, BF16, seed=13)
    view = lambda off: big.as_strided((1, T, 1, 32), (T * step, step, 32, 1), off)
    for i, m in enumerate("qkv"):
        view(64 * i).copy_(d[m])
    ld, S = d["log_decay"].cuda(), d["state"].cuda()
    ref = decay_attention(*[d[m].cuda() for m in "qkv"], ld, state=S)
    got = decay_attention(view(0), view(64), view(128), ld, state=S)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_decay_same_bits_every_time_and_untouched_neighbours(gpu_device):
    """No result depends on the order of anything; the rows behind the last one are left as they were."""
    from evfly_amd import _lib
    L = _lib.lib()
    for dtype, code in ((F32, 0), (BF16, 1)):
        d = decay_inputs(2, 300, 4, 2, 40, 24, dtype, seed=14)
        a, b = _run_decay(d, grads=True), _run_decay(d, grads=True)
        assert all(torch.equal(a[m], b[m]) for m in a)
        c = _cuda(d)
        room = torch.full((2 * 300 * 4 * 24 + 512,), 7.0, dtype=dtype, device="cuda")
        nb = L.evfly_decay_attention_workspace_bytes(2, 300, 4, 2, 40, 24, code, 0)
        ws = torch.full((nb + 512,), 7, dtype=torch.uint8, device="cuda")
        _lib.check(L.evfly_decay_attention_forward(c["q"].data_ptr(), c["k"].data_ptr(), c["v"].data_ptr(), None, c["log_decay"].data_ptr(), None, None, 2, 300, 4, 2, 40, 24, 1.0,
                                                   code, room.data_ptr(), None, ws.data_ptr(), nb, _lib.cur_stream()))
        assert (room[-512:] == 7).all() and (ws[nb:] == 7).all()


def test_decay_no_tokens(gpu_device):
    from evfly_amd.temporal import decay_attention
    d = _cuda(decay_inputs(2, 0, 2, 2, 8, 8, F32, seed=15))
    for S in (d["state"], None):
        out, new = decay_attention(d["q"], d["k"], d["v"], d["log_decay"], state=S)
        assert out.shape == (2, 0, 2, 8) and torch.equal(new, S if S is not None else torch.zeros_like(new))
    S = d["state"].requires_grad_()
    _, new = decay_attention(d["q"], d["k"], d["v"], d["log_decay"], state=S)
    assert torch.equal(torch.autograd.grad(new, S, d["d_state"])[0], d["d_state"])
    e = d["q"][:0]
    out, new = decay_attention(e, e, e, d["log_decay"])
    assert out.shape == (0, 0, 2, 8) and new.shape == (0, 2, 8, 8)


def test_decay_other_stream_and_graphs(gpu_device):
    """On a side stream; captured forward and backward, two graphs replayed in turn with eager work between, inputs refreshed in place."""
    from evfly_amd.temporal import decay_attention
    ds = [_cuda(decay_inputs(2, 300, 2, 2, 32, 32, BF16, seed=s)) for s in (16, 17)]
    def step(c):
        lv = [c[m].detach().requires_grad_() for m in "qkv"]
        out, S = decay_attention(*lv, c["log_decay"], state=c["state"])
        return (out, S, *torch.autograd.grad([out, S], lv, [c["d_out"], c["d_state"]]))
    eager = [step(c) for c in ds]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(ds[0])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager[0]))
    graphs = []
    with torch.cuda.stream(side):
        for c in ds:
            step(c)
            side.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                outs = step(c)
            graphs.append((gr, outs))
    torch.cuda.synchronize()
    for i in range(3):
        for c in ds:
            for m in ("q", "d_out"):
                c[m].copy_(torch.roll(c[m], 1, 1))
        want = [step(c) for c in ds]
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (_, outs), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w)), i


def test_decay_refusals(gpu_device):
    from evfly_amd.temporal import decay_attention, decay_attention_step
    c = _cuda(decay_inputs(2, 3, 4, 2, 8, 8, F32, seed=18))
    q, k, v, ld, S = (c[m] for m in ("q", "k", "v", "log_decay", "state"))
    ln = torch.tensor([3, 2], dtype=torch.int32).cuda()
    bad = [(q[0], k, v, ld), (q.cpu(), k, v, ld), (q.double(), k.double(), v.double(), ld), (q, k.to(BF16), v, ld), (q, k[:, :2], v, ld), (q, k[..., :4], v, ld),
           (q[:, :, :3], k, v, ld), (q, k[:1], v, ld), (q, k, v, ld.double()), (q, k, v, ld[:3]), (q, k, v, ld.cpu()), (q, k, v, None), (q, k, v, ld.clone().requires_grad_()),
           (q.new_zeros(2, 3, 4, 129), k.new_zeros(2, 3, 2, 129), v, ld)]
    for a in bad:
        with pytest.raises(ValueError):
            decay_attention(*a)
    for kw in (dict(state=S[:1]), dict(state=S.to(BF16)), dict(state=S.cpu()), dict(lengths=ln.long()), dict(lengths=ln[:1]), dict(lengths=[3, 2]), dict(lengths=ln.cpu()),
               dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            decay_attention(q, k, v, ld, **kw)
    q1, k1, v1 = q[:, 0], k[:, 0], v[:, 0]
    for a, kw in (((q, k, v, ld, S), {}), ((q1, k1, v1, ld, None), {}), ((q1, k1, v1, ld, S.transpose(2, 3)), {}), ((q1, k1, v1, ld, S), dict(new_state=S[:1])),
                  ((q1, k1, v1, ld, S), dict(new_state=S.transpose(2, 3))), ((q1.requires_grad_(), k1, v1, ld, S), {})):
        with pytest.raises(ValueError):
            decay_attention_step(*a, **kw)
    # a state that was written in place after the forward read it does not pass for the one it read
    s = S.clone()
    lv = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out, _ = decay_attention(*lv, ld, state=s)
    decay_attention_step(q1.detach(), k1, v1, ld, s)
    with pytest.raises(RuntimeError):
        out.sum().backward()


@pytest.mark.parametrize("T", [1, 5, 100])
def test_decay_state_at_any_address(gpu_device, T):
    """A state that starts 4 bytes behind a 16-byte boundary."""
    from evfly_amd.temporal import decay_attention, decay_attention_step
    d = _cuda(decay_inputs(3, T, 2, 1, 24, 32, F32, seed=19))
    n = d["state"].numel()
    odd = lambda: torch.zeros(n + 1, device="cuda")[1:].view(d["state"].shape)
    S, N = odd().copy_(d["state"]), odd()
    ref = decay_attention(d["q"], d["k"], d["v"], d["log_decay"], state=d["state"])
    got = decay_attention(d["q"], d["k"], d["v"], d["log_decay"], state=S)
    assert (got[0] - ref[0]).abs().max() <= 128 * EPS32 * 4 * ref[0].abs().max() and (got[1] - ref[1]).abs().max() <= 128 * EPS32 * 4 * ref[1].abs().max()
    if T == 1:
        out = decay_attention_step(d["q"][:, 0], d["k"][:, 0], d["v"][:, 0], d["log_decay"], S, new_state=N)
        assert torch.equal(out, got[0][:, 0]) and torch.equal(N, got[1])


def test_decay_in_inference_mode(gpu_device):
    """Serving code runs under torch.inference_mode: its own tensors (which have no version) and ordinary ones."""
    from evfly_amd.temporal import block_norm, decay_attention, decay_attention_step
    d = _cuda(decay_inputs(2, 1, 2, 2, 16, 16, F32, seed=20))
    q, k, v = (d[m][:, 0] for m in "qkv")
    ref, want = decay_attention(d["q"], d["k"], d["v"], d["log_decay"], state=d["state"])
    with torch.inference_mode():
        for S in (d["state"].clone(), torch.empty_like(d["state"]).copy_(d["state"])):
            out = decay_attention_step(q, k, v, d["log_decay"], S)
            assert torch.equal(out, ref[:, 0]) and torch.equal(S, want)
        y, h = block_norm(out, pre="rms")
        assert torch.equal(y, out) and h.shape == out.shape
    S = d["state"].clone()
    with torch.inference_mode():
        decay_attention_step(q, k, v, d["log_decay"], S)
    assert torch.equal(S, want)


def test_two_host_threads_on_two_streams(gpu_device):
    """Calls from two threads at once, each on its own stream with its own tensors, give the bits of the calls made one after the other."""
    import threading
    from evfly_amd.temporal import block_norm, decay_attention
    ds = [_cuda(decay_inputs(2, 700, 4, 2, 64, 64, BF16, seed=s)) for s in (21, 22)]

    def work(c):
        out, S = decay_attention(c["q"], c["k"], c["v"], c["log_decay"], state=c["state"])
        return out, S, block_norm(out, c["q"], pre="layer")[1]

    want = [work(c) for c in ds]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def run(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(10):
                    got[i].append(work(ds[i]))
            st.synchronize()
        except Exception as e:                                   # (an assert in a thread would be lost)
            errors.append(e)

    ts = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not errors
    for i in range(2):
        assert len(got[i]) == 10 and all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))


def test_no_second_order(gpu_device):
    from evfly_amd.temporal import block_norm, decay_attention
    q = torch.randn(1, 20, 1, 8, device="cuda", requires_grad=True)
    for y in (decay_attention(q, q, q, torch.zeros(1, device="cuda"))[0], block_norm(q, pre="rms")[1]):
        with pytest.raises(RuntimeError, match="no gradients"):
            torch.autograd.grad(y.sum(), q, create_graph=True)


# ---------------------------------------------------------------------------------------- block norm
def _norm_inputs(lead, C, dtype, gate, seed, residual=True, scale=True, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    d = dict(f=(r(*lead, C) + offset).to(dtype), x=(2 * r(*lead, C)).to(dtype) if residual else None, gate=None, res_scale=1 + 0.1 * r(C) if residual and scale else None)
    if gate is not None:
        shape, gdt = gate
        d["gate"] = (0.5 + 0.5 * r(*shape, C)).to(gdt)
    for m in ("post_weight", "pre_weight"):
        d[m] = 1 + 0.1 * r(C)
    for m in ("post_bias", "pre_bias"):
        d[m] = 0.1 * r(C)
    d["dy"], d["dh"] = r(*lead, C).to(dtype), r(*lead, C).to(dtype)
    return d


LEAVES = ("f", "x", "gate", "res_scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


def _norm_call(fn, d, act, post, pre, eps, to, grads=True, use=("dy", "dh")):
    lv = {m: None if d[m] is None or (m.startswith("post") and post is None) or (m.startswith("pre") and pre is None) else to(d[m]).requires_grad_(grads) for m in LEAVES}
    y, h = fn(lv["f"], lv["x"], lv["gate"], act, lv["res_scale"], post=post, post_weight=lv["post_weight"], post_bias=lv["post_bias"], pre=pre, pre_weight=lv["pre_weight"],
              pre_bias=lv["pre_bias"], eps=eps)
    got = {"y": y.detach()}
    if h is not None:
        got["h"] = h.detach()
    if grads:
        pairs = [(o, to(d[u])) for o, u in ((y, "dy"), (h, "dh")) if o is not None and u in use]
        have = [m for m in LEAVES if lv[m] is not None]
        gr = torch.autograd.grad([o for o, _ in pairs], [lv[m] for m in have], [u for _, u in pairs], allow_unused=True)
        got.update({"d_" + m: t for m, t in zip(have, gr) if t is not None})
    return got


def _norm_compare(d, act="none", post="layer", pre="layer", eps=1e-5, grads=True, use=("dy", "dh")):
    """Bounds: every elementwise result is some thirty roundings of 2^-24 on terms no larger than `top` (the largest magnitude of that result's row factors, taken as
    the result's own largest magnitude times the norms' gain), a sum over n columns or rows adds log-depth or sequential roundings: at most n / 8 + 32 steps in
    any lane. The result's own type adds its half step."""
    from evfly_amd.temporal import block_norm
    dtype = d["f"].dtype
    want = _norm_call(ot.block_norm, d, act, post, pre, eps, lambda t: t.double().clone(), grads, use)
    got = _norm_call(block_norm, d, act, post, pre, eps, lambda t: t.cuda(), grads, use)
    assert set(got) >= set(want) and not any(got[m].any() for m in set(got) - set(want)), (set(got) ^ set(want))      # (what an unused output leaves: zeros)
    C, rows = d["f"].shape[-1], d["f"].numel() // d["f"].shape[-1]
    for m, w in want.items():
        g = got[m].double().cpu()
        assert g.shape == w.shape and torch.isfinite(g).all(), m
        like = d[m[2:]].dtype if m.startswith("d_") else dtype
        assert got[m].dtype == like, m
        # magnitudes: a column sum's terms add up to at most the sum of its terms' sizes; rows * the mean size bounds that
        red = rows if m[2:] in ("res_scale", "post_weight", "post_bias", "pre_weight", "pre_bias") else rows // max(1, d["gate"].numel() // C) if m == "d_gate" else 1
        top = w.abs().max().clamp_min(1.0) if red == 1 else torch.tensor(8.0 * red, dtype=torch.float64)
        lim = (C / 8 + red / 8 + 64) * EPS32 * 4 * top + HALF_STEP[like] * w.abs() * 1.001
        worst = ((g - w).abs() / lim).max().item()
        assert worst <= 1.0, (m, worst, (g - w).abs().max().item())
    return got


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 2), (5, 7), (64, 256), (33, 31), (9, 32), (17, 33), (65, 64), (130, 128), (7, 500), (300, 512), (5, 513), (6, 1001), (9, 2048), (3, 4096),
                                    (3, 4100), (2, 8192), (3, 8191), (4000, 24)])
def test_block_norm(gpu_device, rows, C, dtype):
    _norm_compare(_norm_inputs((rows,), C, dtype, None, 1), eps=1e-3)
    _norm_compare(_norm_inputs((rows,), C, dtype, ((rows,), dtype), 2, scale=False), act="sigmoid", post="rms", pre="rms", eps=1e-3)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("gate", ["channel", "stream", "pair", "token"])
@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
@pytest.mark.parametrize("post,pre", [("layer", "rms"), ("rms", None), (None, "layer"), (None, None)])
def test_block_norm_gates(gpu_device, gate, act, post, pre, dtype):
    lead = (3, 5, 37)
    shape = {"channel": (), "stream": (3, 1, 1), "pair": (3, 5, 1), "token": lead}[gate]
    for C, gdt, residual in ((40, dtype, True), (130, F32, False), (1030, dtype, True)):
        _norm_compare(_norm_inputs(lead, C, dtype, (shape, gdt), 3, residual=residual), act, post, pre)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("streams,tokens,C", [(1, 5000, 64), (2, 3001, 128), (700, 3, 32), (600, 9, 64), (40, 100, 2048), (7, 401, 72)])
def test_block_norm_many_rows(gpu_device, streams, tokens, C, dtype):
    """Column sums and a stream's gate row over more rows than one block visits, and gate rows of fewer rows than a block holds."""
    _norm_compare(_norm_inputs((streams, tokens), C, dtype, ((streams, 1), dtype), 4), act="tanh")
    _norm_compare(_norm_inputs((streams, tokens), C, dtype, ((), F32), 5))


@pytest.mark.parametrize("use", [("dy",), ("dh",)])
def test_block_norm_one_output_used(gpu_device, use):
    _norm_compare(_norm_inputs((4, 30), 64, F32, ((4, 1), F32), 6), act="sigmoid", post="rms", pre="layer", use=use)


def test_block_norm_plain_tail_is_layer_norm(gpu_device):
    """post None, pre "layer": evfly's LayerNorm(x + f)."""
    from evfly_amd.temporal import block_norm
    d = _norm_inputs((50,), 128, F32, None, 7, scale=False)
    y, h = block_norm(d["f"].cuda(), d["x"].cuda(), pre="layer", pre_weight=d["pre_weight"].cuda(), pre_bias=d["pre_bias"].cuda())
    assert torch.equal(y.cpu(), d["f"] + d["x"])
    want = torch.nn.functional.layer_norm((d["f"].double() + d["x"].double()), (128,), d["pre_weight"].double(), d["pre_bias"].double())
    assert (h.double().cpu() - want).abs().max() < 64 * EPS32 * 4 * want.abs().max()


def test_block_norm_rows_far_from_zero(gpu_device):
    """A mean a thousand times the spread: the variance is of the differences, so the input's own rounding (1000 * 2^-24 of a spread of one) is all that is lost."""
    from evfly_amd.temporal import block_norm
    f = _norm_inputs((40,), 256, F32, None, 8, offset=1000.0)["f"]
    _, h = block_norm(f.cuda(), pre="layer")
    want = torch.nn.functional.layer_norm(f.double(), (256,))
    # f is exact; the mean's sum of 256 values of 1000 (32 + 8 roundings of 2^-24) and the difference lose 41 * 1000 * 2^-24, over a spread of one
    assert (h.double().cpu() - want).abs().max() < 41 * 1000 * EPS32 + 64 * EPS32 * 4 * want.abs().max()


def test_block_norm_constant_rows(gpu_device):
    """No spread at all: zeros times 1 / sqrt(eps), finite with eps, and a zero row under "rms" likewise."""
    from evfly_amd.temporal import block_norm
    f = torch.full((6, 96), 2.0, device="cuda").requires_grad_()
    _, h = block_norm(f, pre="layer")
    assert not h.any()
    assert torch.isfinite(torch.autograd.grad(h.sum(), f)[0]).all()
    _, h = block_norm(torch.zeros(5, 40, device="cuda", dtype=BF16), pre="rms")
    assert not h.any()
    # one row that is not finite stays alone
    g = torch.randn(9, 33, device="cuda")
    ref = block_norm(g, pre="layer")[1]
    bad = g.clone()
    bad[4, 3] = float("nan")
    got = block_norm(bad, pre="layer")[1]
    assert torch.isnan(got[4]).all() and torch.equal(got[:4], ref[:4]) and torch.equal(got[5:], ref[5:])
    # eps = 0: the rows a block does not have are no rows (their 0 * inf stays out of the sums)
    w = torch.ones(33, device="cuda", requires_grad=True)
    _, h = block_norm(g[:5], post="rms", post_weight=w, pre="layer", pre_weight=w, eps=0.0)
    assert torch.isfinite(torch.autograd.grad(h.square().sum(), w)[0]).all()


def test_block_norm_gate_far_out(gpu_device):
    """Saturated gates: exact ends at +-infinity, right to some ulp of one (absolute) in between, NaN stays NaN; finite gradients wherever the value is finite."""
    from evfly_amd.temporal import block_norm
    z = torch.tensor([0.0, 1e-8, -1e-8, 0.5, -0.5, 10.0, -10.0, 40.0, -40.0, 79.0, -79.0, 81.0, -81.0, 88.0, -88.0, 90.0, -90.0, 104.0, -104.0, 3e38, -3e38, math.inf, -math.inf,
                      math.nan, 20.0, -20.0, 5.0, -5.0, 1.0, -1.0, 2.0, -2.0]).view(1, 32)
    f = torch.ones(1, 32, device="cuda", requires_grad=True)
    for act, want in (("sigmoid", torch.sigmoid(z.double())), ("tanh", torch.tanh(z.double()))):
        g = z.cuda().requires_grad_()
        y, _ = block_norm(f, gate=g, gate_act=act)
        got = y.detach().double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert ((got - want).abs()[ok] <= 8 * EPS32).all()                     # a handful of roundings of values up to one
        if act == "sigmoid":                                                   # and of the value itself where it is small
            mid = ok & (z.abs() <= 79)
            assert ((got - want).abs()[mid] <= 16 * EPS32 * want.abs()[mid]).all()
        df, dg = torch.autograd.grad(y.sum(), [f, g])
        assert torch.isfinite(df.cpu()[ok]).all() and torch.isfinite(dg.cpu()[ok]).all()


def test_block_norm_no_rows_and_strides(gpu_device):
    from evfly_amd.temporal import block_norm
    w = torch.ones(16, device="cuda", requires_grad=True)
    gate = torch.ones(16, device="cuda", requires_grad=True)
    y, h = block_norm(torch.zeros(0, 16, device="cuda"), gate=gate, pre="layer", pre_weight=w)
    assert y.shape == h.shape == (0, 16)
    gw, gg = torch.autograd.grad(h.sum() + y.sum(), [w, gate])
    assert not gw.any() and not gg.any()
    a = torch.randn(8, 6, 40, device="cuda")
    x = torch.randn(6, 8, 40, device="cuda").transpose(0, 1)
    got = block_norm(a[..., 1:33], x[..., 3:35], pre="rms", pre_weight=torch.randn(64, device="cuda")[::2].contiguous())
    torch.manual_seed(0)
    ref = block_norm(a[..., 1:33].contiguous(), x[..., 3:35].contiguous(), pre="rms")
    assert torch.equal(got[0], ref[0])
    buf = torch.randn(1 + 7 * 64, device="cuda")
    un, al = buf[1:].view(7, 64), buf[1:].clone().view(7, 64)                    # rows that start 4 bytes behind a 16-byte boundary
    u, v = block_norm(un, post="layer", pre="rms"), block_norm(al, post="layer", pre="rms")
    assert (u[0] - v[0]).abs().max() < 64 * EPS32 * 4 * 8 and (u[1] - v[1]).abs().max() < 64 * EPS32 * 4 * 8


def test_block_norm_same_bits_and_untouched_neighbours(gpu_device):
    from evfly_amd import _lib
    from evfly_amd.temporal import block_norm
    L = _lib.lib()
    for lead, C, gate in (((600, 9), 64, (600, 1)), ((3, 700), 1000, (3, 1)), ((2000,), 40, ())):
        d = _norm_inputs(lead, C, BF16, (gate, BF16), 9)
        a, b = (_norm_call(block_norm, d, "sigmoid", "layer", "rms", 1e-5, lambda t: t.cuda()) for _ in range(2))
        assert all(torch.equal(a[m], b[m]) for m in a)
    rows, C = 77, 96
    nb = L.evfly_block_norm_workspace_bytes(rows, C, 7, 0)
    f, x, dy, dh = (torch.randn(rows, C, device="cuda") for _ in range(4))
    gate = torch.randn(11, C, device="cuda")
    outs = [torch.full((n * C + 256,), 7.0, device="cuda") for n in (rows, rows, 11, 1, 1, 1, 1, 1)]
    ws = torch.full((nb + 256,), 7, dtype=torch.uint8, device="cuda")
    w = torch.ones(C, device="cuda")
    _lib.check(L.evfly_block_norm_backward(f.data_ptr(), x.data_ptr(), gate.data_ptr(), 7, 0, 0, w.data_ptr(), 1, w.data_ptr(), None, 1, w.data_ptr(), None, 1e-5, dy.data_ptr(),
                                           dh.data_ptr(), rows, C, 0, *[o.data_ptr() for o in outs], ws.data_ptr(), nb, _lib.cur_stream()))
    for o in outs:
        assert (o[-256:] == 7).all() and not (o[:-256] == 7).any()
    assert (ws[nb:] == 7).all()


def test_block_norm_other_stream_and_graph(gpu_device):
    from evfly_amd.temporal import block_norm
    d = {k: None if t is None else t.cuda() for k, t in _norm_inputs((4, 90), 200, BF16, ((4, 1), BF16), 10).items()}
    step = lambda: list(_norm_call(block_norm, d, "sigmoid", "layer", "layer", 1e-5, lambda t: t.detach()).values())
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
        side.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs = step()
    torch.cuda.synchronize()
    for i in range(3):
        d["f"].copy_(torch.roll(d["f"], 1, 1))
        want = step()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_block_norm_refusals(gpu_device):
    from evfly_amd.temporal import block_norm
    f = torch.randn(2, 6, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    for a, kw in (((f.cpu(),), {}), ((f.double(),), {}), ((f.new_zeros(2, 8193),), {}), ((f, f[:1]), {}), ((f, f.to(BF16)), {}), ((f,), dict(post="batch")), ((f,), dict(pre="none")),
                  ((f,), dict(res_scale=w)), ((f,), dict(post_weight=w)), ((f,), dict(pre_bias=w)), ((f,), dict(post="layer", post_weight=w[:8])), ((f,), dict(pre="rms", pre_weight=w.double())),
                  ((f,), dict(gate_act="relu")), ((f,), dict(eps=-1.0)), ((f,), dict(gate=w.to(BF16))), ((f,), dict(gate=w.cpu())), ((f,), dict(gate=f[:1])), ((f,), dict(gate=f[0])),
                  ((f,), dict(gate=w[:8])), (([1.0],), {})):
        with pytest.raises(ValueError):
            block_norm(*a, **kw)


# ---------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_a_block_of_both(gpu_device, dtype):
    """h = norm(x); q, k, v = h W; o = gated per-head norm of decay attention; y, next h = the block's end -- forward, gradients, and the same windows one by one."""
    from evfly_amd.temporal import block_norm, decay_attention, decay_attention_step
    n, T, H, D = 3, 90, 4, 32
    C = H * D
    g = torch.Generator().manual_seed(20)
    r = lambda *s: torch.randn(*s, generator=g)
    x, wqkv, wo, wg = r(n, T, C).to(dtype), (r(C, 3 * C) / C ** 0.5).to(dtype), (r(C, C) / C ** 0.5).to(dtype), (r(C, C) / C ** 0.5).to(dtype)
    n1, n2, hw, al, ld = 1 + 0.1 * r(C), 1 + 0.1 * r(C), 1 + 0.1 * r(D), 1 + 0.1 * r(C), torch.tensor([-0.7, -0.2, -0.05, -0.01])
    up, uh = r(n, T, C).to(dtype), r(n, T, C).to(dtype)

    def block(norm, attend, x, wqkv, wo, wg, n1, n2, hw, al, ld):
        _, h = norm(x, pre="layer", pre_weight=n1)
        q, k, v = ((h @ wqkv).unflatten(-1, (3 * H, D))).chunk(3, -2)
        o = attend(q, k, v, ld)
        o, _ = norm(o, gate=(h @ wg).unflatten(-1, (H, D)), gate_act="sigmoid", post="rms", post_weight=hw)
        return norm(o.flatten(-2) @ wo, x, res_scale=al, post="rms", post_weight=n2, pre="layer", pre_weight=n1)

    ins = (x, wqkv, wo, wg, n1, n2, hw, al)
    lv = [t.double().clone().requires_grad_() for t in ins]
    want = block(ot.block_norm, lambda *a: ot.decay_attention(*a)[0], *lv, ld)
    want = [*want, *torch.autograd.grad(want, lv, [up.double(), uh.double()])]
    lc = [t.cuda().requires_grad_() for t in ins]
    got = block(block_norm, lambda *a: decay_attention(*a)[0], *lc, ld.cuda())
    got = [*got, *torch.autograd.grad(got, lc, [up.cuda(), uh.cuda()])]
    # a chain of some twenty tensors rounded to the tokens' type, each a half step of its largest element, through factors of order one; fp32 sums of 128 .. 270 terms
    tol = 20 * HALF_STEP[dtype] if dtype == BF16 else 20 * 300 * EPS32
    for i, (a, b) in enumerate(zip(got, want)):
        e = (a.detach().double().cpu() - b.detach()).abs().max() / b.detach().abs().max()
        assert e < tol, (i, e.item())
    with torch.no_grad():
        S, ys = torch.zeros(n, H, D, D, device="cuda"), []
        for t in range(T):
            y, _ = block(block_norm, lambda q, k, v, ld: decay_attention_step(q, k, v, ld, S), lc[0][:, t], *lc[1:], ld.cuda())
            ys.append(y)
    e = (torch.stack(ys, 1).double().cpu() - want[0].detach()).abs().max() / want[0].detach().abs().max()
    assert e < tol, e.item()
