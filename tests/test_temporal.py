"""CPU side of the temporal operators: the oracle's definitions against differences and a written-out sum, and every refusal of the C ABI (arguments are checked before
anything touches a device)."""
import ctypes as C
import math

import pytest
import torch

from evfly_amd import _lib
from oracle import temporal as ot


def test_oracle_decay_is_the_written_out_sum():
    g = torch.Generator().manual_seed(1)
    n, T, H, KV, dk, dv = 2, 7, 4, 2, 3, 5
    q, k, v = (torch.randn(n, T, h, e, generator=g) for h, e in ((H, dk), (KV, dk), (KV, dv)))
    ld = torch.tensor([0.0, -0.3, -2.0, float("-inf")])
    S0 = torch.randn(n, H, dk, dv, generator=g)
    lens = torch.tensor([7, 4], dtype=torch.int32)
    out, S = ot.decay_attention(q, k, v, ld, S0, lens, 0.7)
    w = lambda h, m: 1.0 if m == 0 else math.exp(ld[h].item() * m)
    for b in range(n):
        L = int(lens[b])
        for h in range(H):
            for t in range(T):
                want = torch.zeros(dv, dtype=torch.float64)
                if t < L:
                    want = 0.7 * w(h, t + 1) * q[b, t, h].double() @ S0[b, h].double()
                    for s in range(t + 1):
                        want = want + 0.7 * w(h, t - s) * (q[b, t, h].double() @ k[b, s, h // 2].double()) * v[b, s, h // 2].double()
                assert torch.allclose(out[b, t, h], want, rtol=1e-12, atol=1e-12)
            want = w(h, L) * S0[b, h].double()
            for s in range(L):
                want = want + w(h, L - 1 - s) * torch.outer(k[b, s, h // 2].double(), v[b, s, h // 2].double())
            assert torch.allclose(S[b, h], want, rtol=1e-12, atol=1e-12)


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
    ld, lens = torch.tensor([-0.1, -1.0]), torch.tensor([3, 2], dtype=torch.int32)
    assert torch.autograd.gradcheck(lambda q, k, v, s: ot.decay_attention(q, k, v, ld, s, lens, 0.5), (r(2, 3, 2, 2), r(2, 3, 1, 2), r(2, 3, 1, 3), r(2, 2, 2, 3)))
    for post, pre in (("layer", "rms"), ("rms", "layer"), (None, "layer"), ("layer", None)):
        def fn(f, x, gate, al, w, b):
            y, h = ot.block_norm(f, x, gate, "sigmoid", al, post=post, post_weight=w if post else None, post_bias=b if post else None, pre=pre,
                                 pre_weight=b if pre else None, pre_bias=w if pre else None)
            return (y, h) if pre else y
        assert torch.autograd.gradcheck(fn, (r(3, 5), r(3, 5), r(3, 5), r(5), r(5), r(5)))


# ---- refusals: a call with `good` arguments but for one; pointers are never followed
X = 1 << 20          # stands for a device pointer
DECAY = dict(q=X, k=X, v=X, strides=None, log_decay=X, state_in=None, lengths=None, n=1, T=64, H=4, KV=2, dk=32, dv=32, scale=1.0, dtype=0,
             out=X, state_out=None, ws=None, ws_bytes=0, stream=None)
DECAY_BACK = dict(q=X, k=X, v=X, strides=None, log_decay=X, state_in=None, lengths=None, d_out=X, d_state=None, n=1, T=64, H=4, KV=2, dk=32, dv=32, scale=1.0,
                  dtype=0, dq=X, dk_out=X, dv_out=X, ds=None, ws=None, ws_bytes=0, stream=None)
NORM = dict(f=X, x=X, gate=X, rpg=1, gate_f32=0, act=0, alpha=None, post=1, w1=None, b1=None, pre=1, w2=None, b2=None, eps=1e-5, rows=8, C=64, dtype=0, y=X, h=X,
            stream=None)
NORM_BACK = dict(f=X, x=X, gate=X, rpg=1, gate_f32=0, act=0, alpha=None, post=1, w1=None, b1=None, pre=1, w2=None, b2=None, eps=1e-5, dy=X, dh=X, rows=8, C=64,
                 dtype=0, df=X, dx=None, dgate=None, da=None, dw1=None, db1=None, dw2=None, db2=None, ws=X, ws_bytes=1 << 30, stream=None)
BAD_DECAY = [dict(H=3), dict(KV=0), dict(H=0), dict(dk=0), dict(dk=129), dict(dv=0), dict(dv=129), dict(n=-1), dict(T=-1), dict(T=(1 << 30) + 1), dict(dtype=2), dict(dtype=-1),
             dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(k=None), dict(v=None), dict(log_decay=None), dict(n=1 << 30, H=4)]
BAD_NORM = [dict(C=0), dict(C=8193), dict(rows=-1), dict(rows=1 << 31), dict(dtype=2), dict(post=3), dict(pre=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(act=1), dict(act=9),
            dict(rpg=0), dict(rpg=3), dict(rpg=16), dict(f=None), dict(x=None, alpha=X)]
CALLS = ([("evfly_decay_attention_forward", DECAY, b) for b in BAD_DECAY + [dict(out=None), dict(n=1, T=4096, ws=None), dict(n=1, T=4096, ws=X + 4, ws_bytes=1 << 40)]] +
         [("evfly_decay_attention_backward", DECAY_BACK, b) for b in BAD_DECAY + [dict(d_out=None), dict(dq=None), dict(dk_out=None), dict(dv_out=None), dict()]] +
         [("evfly_block_norm_forward", NORM, b) for b in BAD_NORM + [dict(y=None, h=None), dict(h=None), dict(pre=0, y=None, h=None)]] +
         [("evfly_block_norm_backward", NORM_BACK, b) for b in BAD_NORM + [dict(df=None), dict(ws=None), dict(ws_bytes=0), dict(ws=X + 4), dict(x=None, dx=X), dict(x=None, da=X),
                                                                            dict(gate=None, dgate=X), dict(post=0, dw1=X), dict(post=0, db1=X), dict(pre=0, dw2=X), dict(pre=0)]])


@pytest.mark.parametrize("name,good,bad", CALLS, ids=lambda a: a if isinstance(a, str) else ",".join(f"{k}={v}" for k, v in a.items()) if len(a) < 5 else "")
def test_c_entries_refuse(name, good, bad):
    L = _lib.load_library()
    assert getattr(L, name)(*{**good, **bad}.values()) == -1
    assert L.evfly_last_error().decode().startswith(name[len("evfly_"):])


def test_no_streams_and_no_rows_are_nothing_to_do():
    L = _lib.load_library()
    assert L.evfly_decay_attention_forward(*{**DECAY, "n": 0}.values()) == 0
    assert L.evfly_decay_attention_backward(*{**DECAY_BACK, "n": 0}.values()) == 0
    assert L.evfly_block_norm_forward(*{**NORM, "rows": 0}.values()) == 0


def test_workspace_sizes():
    L = _lib.load_library()
    ws = L.evfly_decay_attention_workspace_bytes
    assert ws(64, 1, 8, 8, 32, 32, 0, 0) == 0 and ws(1, 16, 8, 8, 32, 32, 0, 0) == 0
    assert ws(1, 1 << 15, 16, 4, 128, 128, 1, 0) > 0 and ws(1, 1 << 15, 16, 4, 128, 128, 1, 1) > ws(1, 1 << 15, 16, 4, 128, 128, 1, 0)
    assert ws(1, 64, 4, 3, 32, 32, 0, 0) < 0
    bn = L.evfly_block_norm_workspace_bytes
    assert bn(0, 64, 1, 0) == 0 and bn(100, 64, 1, 0) > 0 and bn(100, 9000, 1, 0) < 0


def test_python_entries_need_the_device():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from evfly_amd import temporal
    z = torch.zeros(1, 2, 1, 4)
    for call in (lambda: temporal.decay_attention(z, z, z, torch.zeros(1)), lambda: temporal.decay_attention_step(z[0], z[0], z[0], torch.zeros(1), torch.zeros(2, 1, 4, 4)),
                 lambda: temporal.block_norm(z)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_constants_agree_with_the_header():
    import os
    import re
    from evfly_amd import temporal
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "evfly_hip.h")).read()
    val = lambda n: int(re.search(rf"#define {n} (\d+)", text).group(1))
    assert val("EVFLY_DECAY_MAX_DIM") == temporal.MAX_HEAD_DIM and val("EVFLY_DECAY_STEP_TOKENS") == temporal.STEP_TOKENS
    assert val("EVFLY_BLOCK_NORM_MAX_CHANNELS") == temporal.MAX_CHANNELS
    assert [val("EVFLY_NORM_" + k) for k in ("NONE", "LAYER", "RMS")] == [temporal._NORM[k] for k in (None, "layer", "rms")]
