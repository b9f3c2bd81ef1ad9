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


# ---- what torch does not see of the library's work
@pytest.fixture
def no_device(monkeypatch):
    """The entries on CPU tensors: every argument fits, the library's calls do nothing."""
    class Nothing:
        def __getattr__(self, name):
            return lambda *a: 0
    monkeypatch.setattr(temporal._lib, "lib", lambda: None)
    monkeypatch.setattr(temporal._lib, "load_library", Nothing)
    monkeypatch.setattr(temporal, "_decay_fits", lambda *a: True)
    monkeypatch.setattr(temporal, "_block_fits", lambda *a: True)
    monkeypatch.setattr(temporal, "_getDevice", lambda: -1)
    monkeypatch.setattr(temporal, "_rawStream", lambda i: 0)


Q, LD, S = torch.zeros(1, 3, 2, 4), torch.zeros(2), torch.zeros(1, 2, 4, 4)
ENTRIES = {"decay_attention": lambda x: temporal.decay_attention(x, Q, Q, LD, state=S)[0],
           "decay_attention_step": lambda x: temporal.decay_attention_step(x[:, 0], Q[:, 0], Q[:, 0], LD, S.clone()),
           "block_norm": lambda x: temporal.block_norm(x, Q, pre="rms")[1]}
OF_OTHERS = {"v": (Q, lambda t: temporal.decay_attention(Q, Q, t, LD)), "log_decay": (LD, lambda t: temporal.decay_attention(Q, Q, Q, t)),
             "state": (S, lambda t: temporal.decay_attention(Q, Q, Q, LD, state=t)), "step_state": (S, lambda t: temporal.decay_attention_step(Q[:, 0], Q[:, 0], Q[:, 0], LD, t)),
             "x": (Q, lambda t: temporal.block_norm(Q, t)), "gate": (torch.zeros(4), lambda t: temporal.block_norm(Q, gate=t)),
             "weight": (torch.zeros(4), lambda t: temporal.block_norm(Q, pre="rms", pre_weight=t))}


@pytest.mark.parametrize("name", list(ENTRIES))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(no_device, name, grad):
    call = ENTRIES[name]
    with torch.autograd.forward_ad.dual_level():
        x = Q.clone().requires_grad_(grad and name != "decay_attention_step")
        with pytest.raises(NotImplementedError):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(Q)))
        assert call(Q).shape[-1] == 4                                # a level alone is nothing to refuse
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (Q,), (torch.ones_like(Q),))


@pytest.mark.parametrize("name", list(OF_OTHERS))
def test_forward_mode_of_the_other_arguments_is_refused(no_device, name):
    t, call = OF_OTHERS[name]
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        call(torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t)))


@pytest.mark.parametrize("name", list(ENTRIES))
def test_tracers_are_refused(no_device, name):
    from torch.fx.experimental.proxy_tensor import make_fx
    call = ENTRIES[name]
    with pytest.raises(RuntimeError, match="does not see"):
        torch.jit.trace(call, (Q,), check_trace=False)
    with pytest.raises(RuntimeError, match="does not see"):
        make_fx(call)(Q)
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.stack([Q, Q]))
    if name != "decay_attention_step":
        with pytest.raises(RuntimeError, match="does not see"):
            make_fx(lambda x: call(x.requires_grad_()))(Q.clone())
    assert call(Q).shape[-1] == 4


# ---- state buffers that share memory
def _c_call(name, good, **bad):
    from evfly_amd import _lib
    L = _lib.load_library()
    assert getattr(L, name)(*{**good, **bad}.values()) == -1
    return L.evfly_last_error().decode()


def test_states_that_overlap_in_part_are_refused(no_device):
    buf = torch.zeros(5, 2, 4, 4)
    q = torch.zeros(4, 2, 4)
    for state, new in ((buf[:-1], buf[1:]), (buf[1:], buf[:-1]), (buf.view(-1)[:128].view(4, 2, 4, 4), buf.view(-1)[1:129].view(4, 2, 4, 4))):
        with pytest.raises(ValueError, match="overlap"):
            temporal.decay_attention_step(q, q, q, LD, state, new_state=new)
    whole = torch.zeros(8, 2, 4, 4)
    for state, new in ((whole[:4], whole[4:]), (whole[4:], whole[:4]), (whole[:4], whole[:4])):
        temporal.decay_attention_step(q, q, q, LD, state, new_state=new)


def test_states_that_overlap_in_part_are_refused_by_the_abi():
    from test_temporal import DECAY, X
    size = 4 * 32 * 32 * 4
    for off in (4, 4096, size - 4):
        for a, b in ((X, X + off), (X + off, X)):
            for T in (1, 64, 200):
                assert "overlap" in _c_call("evfly_decay_attention_forward", DECAY, T=T, state_in=a, state_out=b, ws=X, ws_bytes=1 << 40)


def test_the_states_gradient_has_a_buffer_of_its_own():
    """The pass that forms dq reads the state while the one that forms dv writes its gradient."""
    from test_temporal import DECAY_BACK, X
    size = 4 * 32 * 32 * 4
    for other in ("state_in", "d_state"):
        for off in (0, 4, size - 4):
            for a, b in ((X, X + off), (X + off, X)):
                for T in (1, 64, 2000):
                    said = _c_call("evfly_decay_attention_backward", DECAY_BACK, T=T, ws=X, ws_bytes=1 << 40, ds=a, **{other: b})
                    assert "d_state_in" in said and "memory" in said
