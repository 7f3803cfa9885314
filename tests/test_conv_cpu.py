"""Refusals of the short causal convolution, on a machine without a GPU too."""

from __future__ import annotations

import ctypes

import pytest
import torch

from spear_b200.ops.ssm import causal_conv, causal_conv_step

Z = torch.zeros


@pytest.mark.parametrize("args,kw,err,text", [
    ((Z(4, 8), Z(8, 4)), {}, ValueError, "x must be"),
    ((Z(1, 4, 0), Z(0, 4)), {}, ValueError, "x must be"),
    ((Z(1, 4, 8).double(), Z(8, 4)), {}, RuntimeError, "x must be bfloat16"),
    ((Z(1, 4, 8), Z(8, 5)), {}, ValueError, "weight must be"),
    ((Z(1, 4, 8), Z(8, 1)), {}, ValueError, "weight must be"),
    ((Z(1, 4, 8), Z(7, 4)), {}, ValueError, "weight must be"),
    ((Z(1, 4, 8), Z(8, 1, 4)), {}, ValueError, "weight must be"),
    ((Z(1, 4, 8), Z(8, 4).half()), {}, RuntimeError, "weight must have"),
    ((Z(1, 4, 8), Z(8, 4), Z(4)), {}, ValueError, "bias must be"),
    ((Z(1, 4, 8).half(), Z(8, 4), Z(8).half()), {}, RuntimeError, "bias must have"),
    ((Z(1, 4, 8), Z(8, 4)), {"activation": "relu"}, ValueError, "activation"),
    ((Z(1, 4, 8), Z(8, 4)), {"initial_state": Z(1, 4, 8)}, ValueError, "initial_state must be"),
    ((Z(1, 4, 8), Z(8, 4)), {"initial_state": Z(1, 3, 8).half()}, RuntimeError, "initial_state must have"),
    ((Z(2, 4, 8), Z(8, 4)), {"lengths": Z(3, dtype=torch.int32)}, ValueError, "lengths"),
    ((Z(2, 4, 8), Z(8, 4)), {"lengths": Z(2, dtype=torch.int64)}, ValueError, "lengths"),
    ((Z(2, 4, 8), Z(8, 4)), {}, RuntimeError, "no CPU path"),
])
def test_refusals(args, kw, err, text):
    with pytest.raises(err, match=text):
        causal_conv(*args, **kw)


@pytest.mark.parametrize("args,kw,err,text", [
    ((Z(1, 1, 8), Z(1, 3, 8), Z(8, 4)), {}, ValueError, "x_t must be"),
    ((Z(1, 8), Z(1, 2, 8), Z(8, 4)), {}, ValueError, "state must be"),
    ((Z(1, 8), Z(1, 3, 8).half(), Z(8, 4)), {}, ValueError, "state must be"),
    ((Z(2, 8), Z(2, 8, 3).transpose(1, 2), Z(8, 4)), {}, ValueError, "state must be contiguous"),
    ((Z(1, 8), Z(1, 3, 8), Z(8, 4)), {}, RuntimeError, "no CPU path"),
])
def test_step_refusals(args, kw, err, text):
    with pytest.raises(err, match=text):
        causal_conv_step(*args, **kw)


def test_where_the_new_state_may_go():
    from spear_b200.ops.ssm.conv import check_state_out

    pool = Z(3, 3, 8)
    state = pool[:2]
    assert check_state_out("f", state, None).data_ptr() != state.data_ptr()
    assert check_state_out("f", state, state) is state
    again = pool[:2]
    assert check_state_out("f", state, again) is again  # the same memory by another name
    for bad in (pool[1:], Z(2, 3, 9), Z(2, 3, 8).half(), Z(2, 8, 3).transpose(1, 2)):
        with pytest.raises(ValueError, match="state_out"):
            check_state_out("f", state, bad)


def test_entry_refuses_bad_arguments_before_any_launch():
    from spear_b200 import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(16)

    def fwd(x=p, w=p, y=p, B=1, L=4, D=8, W=4, sb=32, st=8, dt=0, wt=0):
        return lib.btp_sm100_causal_conv_forward(x, w, None, None, None, y, None, B, L, D, W, sb, st, 0, dt, wt, None)

    assert fwd(B=0) == -2 and fwd(L=0) == -2 and fwd(D=-1) == -2 and fwd(sb=-1) == -2 and fwd(L=(1 << 30) + 1) == -2
    assert fwd(W=1) == -3 and fwd(W=5) == -3 and fwd(dt=2) == -4 and fwd(dt=0, wt=3) == -4
    assert fwd(x=None) == -1 and fwd(w=None) == -1 and fwd(y=None) == -1
    bwd = lib.btp_sm100_causal_conv_backward
    assert bwd(p, p, None, None, None, p, None, p, p, None, None, None, 1, 4, 8, 4, 32, 8, 0, 0, 0, None) == -1
    step = lib.btp_sm100_causal_conv_step
    assert step(p, p, p, None, p, None, 1, 8, 4, 8, 0, 0, 0, None) == -1
    assert step(p, p, p, None, p, p, 1, 8, 9, 8, 0, 0, 0, None) == -3


@pytest.mark.parametrize("token", ["conv", "scan"])
def test_autograd_learns_of_a_state_that_is_updated_in_place(monkeypatch, token):
    """A tensor that some graph has saved must not change unseen; a tensor with a gradient of its own is not overwritten."""
    from types import SimpleNamespace

    from spear_b200.ops import _call
    from spear_b200.ops.ssm import selective_scan_step

    token_call = lambda *args: (torch.empty_like(args[0]), torch.empty_like(state) if args[-2] is None else args[-2])
    monkeypatch.setattr(_call, "native", lambda: SimpleNamespace(causal_conv_step=token_call, selective_scan_step=token_call))
    monkeypatch.setattr(_call, "on_gpu", lambda what, first, *others: 0)
    if token == "conv":
        state, w = torch.randn(2, 3, 8), torch.nn.Parameter(torch.randn(8, 4))
        step = lambda **kw: causal_conv_step(Z(2, 8), state, w, **kw)
    else:
        state, w = torch.randn(2, 8, 4), torch.nn.Parameter(torch.randn(8, 4))
        step = lambda **kw: selective_scan_step(Z(2, 8), Z(2, 8), w, Z(2, 4), Z(2, 4), state, **kw)
    loss = (state * torch.ones_like(state, requires_grad=True)).sum()  # saves the state
    before = state._version
    y, new = step()
    assert state._version == before and not y.requires_grad and not new.requires_grad
    y, new = step(state_out=state)
    assert new is state and state._version == before + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    other = torch.empty_like(state)
    step(state_out=other)
    assert other._version == 1
    with pytest.raises(ValueError, match="requires grad"):
        step(state_out=torch.empty_like(state).requires_grad_())
    with torch.no_grad():
        step(state_out=torch.empty_like(state).requires_grad_())
    with torch.inference_mode():
        step(state_out=torch.empty_like(state))


@pytest.mark.parametrize("B,L,D", [(2 ** 32 + 1, 1, 1), (1, 2 ** 32 + 5, 1), (1, 1, 2 ** 32 + 8)])
def test_sizes_beyond_32_bits_are_refused_not_cut_off(B, L, D):
    E = lambda *shape: torch.empty(*shape, device="meta")
    with pytest.raises(ValueError, match="below 2\\^31"):
        causal_conv(E(B, L, D), E(D, 4))
    if L == 1:
        with pytest.raises(ValueError, match="below 2\\^31"):
            causal_conv_step(E(B, D), E(B, 3, D), E(D, 4))


def test_entry_refuses_partial_sums_that_it_cannot_store_in_pairs():
    from spear_b200 import _lib

    lib = _lib.load()
    p = ctypes.c_void_p(16)
    for at in (20, 17):
        rc = lib.btp_sm100_causal_conv_backward(p, p, None, None, None, p, None, p, p, None, None, ctypes.c_void_p(at), 1, 4, 8, 4, 32, 8, 0, 0, 0, None)
        assert rc == -5 and "8-byte" in lib.btp_sm100_last_error().decode()
