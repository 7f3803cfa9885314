"""The token-major operators under tracers and other interpreters of torch calls, on a machine without a GPU.

The launches are stood in for: a CPU kernel of each registered op marks its outputs, and a direct call into the library is an
error.  What a tracer records has to hold the registered op, and what it recorded has to run it again on other inputs.
"""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from spear_b200.ops import _call
from spear_b200.ops.norm import rms_norm, rms_norm_8bit
from spear_b200.ops.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step

N = torch.randn
OUTPUTS = {"rms_norm_forward": ("y", "h", "rstd"), "rms_norm_8bit": ("q", "h", "scale"), "rms_norm_backward": ("dx", "dresidual", "dweight"),
           "causal_conv_forward": ("y", "state"), "causal_conv_backward": ("dx", "dweight", "dbias", "dinitial"),
           "causal_conv_step": ("y", "state_out"), "scan_forward": ("y", "state", "checkpoints"),
           "scan_backward": ("dx", "ddelta", "dparams", "dB", "dC", "dz", "dinitial"), "scan_step": ("y", "state_out")}

# name of the op, the call, its inputs
CALLS = {
    "norm": ("rms_norm_forward", lambda x, w: rms_norm(x, w), lambda: (N(4, 8), N(8))),
    "norm residual": ("rms_norm_forward", lambda x, w, r: rms_norm(x, w, r), lambda: (N(2, 4, 8), N(8), N(2, 4, 8))),
    "norm 8 bits": ("rms_norm_8bit", lambda x, w: tuple(t.float() for t in rms_norm_8bit(x, w, block=128)), lambda: (N(4, 8), N(8))),
    "conv": ("causal_conv_forward", lambda x, w: causal_conv(x, w, return_state=True), lambda: (N(2, 5, 8), N(8, 4))),
    "conv token": ("causal_conv_step", lambda x, s, w: causal_conv_step(x, s, w), lambda: (N(2, 8), N(2, 3, 8), N(8, 4))),
    "scan": ("scan_forward", lambda x, d, A, B, C: selective_scan(x, d, A, B, C, return_state=True),
             lambda: (N(2, 5, 8), N(2, 5, 8), N(8, 4), N(2, 5, 4), N(2, 5, 4))),
    "scan token": ("scan_step", lambda x, d, A, B, C, s: selective_scan_step(x, d, A, B, C, s),
                   lambda: (N(2, 8), N(2, 8), N(8, 4), N(2, 4), N(2, 4), N(2, 8, 4))),
}


@pytest.fixture
def stand_in(monkeypatch):
    """Counts the runs of each registered op on CPU tensors; every output becomes its first input's sum."""
    runs = {name: 0 for name in OUTPUTS}
    lib = torch.library.Library("spear_btp", "IMPL")

    def kernel(name):
        schema = getattr(torch.ops.spear_btp, name).default._schema

        @torch.no_grad()
        def run(*args, **kw):
            runs[name] += 1
            given = {a.name: v for a, v in zip(schema.arguments, args)} | kw
            for out in OUTPUTS[name]:
                if given.get(out) is not None:
                    given[out].copy_(args[0].sum().expand(given[out].shape))

        return run

    for name in OUTPUTS:
        lib.impl(name, kernel(name), "CPU")

    def refuse(name, *args):
        raise AssertionError(f"{name} was called past the registered op")

    monkeypatch.setattr(_call, "call", refuse)
    monkeypatch.setattr(_call, "query", refuse)
    monkeypatch.setattr(_call, "native", lambda: refuse("the module"))
    monkeypatch.setattr(_call, "on_gpu", lambda what, first, *others: first.get_device())
    yield runs
    lib._destroy()


def tensors(out):
    return [out] if torch.is_tensor(out) else list(out)


def ops_of(graph):
    return [str(n.target) for n in graph.nodes if "spear_btp" in str(n.target)]


@pytest.mark.parametrize("case", CALLS, ids=str)
def test_make_fx_records_the_op(stand_in, case):
    op, fn, make = CALLS[case]
    traced = make_fx(fn)(*make())
    assert ops_of(traced.graph) == [f"spear_btp.{op}.default"] and stand_in[op] == 1
    args = make()
    got = tensors(traced(*args))
    assert stand_in[op] == 2
    for t in got:
        assert torch.equal(t, args[0].sum().to(torch.float8_e4m3fn).float().expand(t.shape) if case == "norm 8 bits" and t is got[0]
                           else args[0].sum().expand(t.shape))


@pytest.mark.parametrize("case", CALLS, ids=str)
@pytest.mark.filterwarnings("ignore")
def test_jit_trace_records_the_op(stand_in, case):
    op, fn, make = CALLS[case]
    traced = torch.jit.trace(fn, make(), check_trace=False)
    assert f"spear_btp::{op}" in str(traced.graph)
    args = make()
    before = stand_in[op]
    got = tensors(traced(*args))
    assert stand_in[op] == before + 1 and all(torch.isfinite(t).all() for t in got)
    if case != "norm 8 bits":
        assert all(torch.equal(t, args[0].sum().expand(t.shape)) for t in got)


@pytest.mark.parametrize("case,ops", [("norm", ("rms_norm_forward", "rms_norm_backward")), ("conv", ("causal_conv_forward", "causal_conv_backward")),
                                      ("scan", ("scan_forward", "scan_backward"))])
def test_make_fx_records_both_directions(stand_in, case, ops):
    _, fn, make = CALLS[case]

    def step(*args):
        leaves = [a.detach().requires_grad_(True) for a in args]
        outs = tensors(fn(*leaves))
        return torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])

    traced = make_fx(step)(*make())
    assert ops_of(traced.graph) == [f"spear_btp.{op}.default" for op in ops]
    assert all(stand_in[op] == 1 for op in ops)
    args = make()
    # the stand-in of each backward op gives every gradient the sum of its first input: x in all three
    assert all(torch.equal(g, args[0].sum().expand(g.shape)) for g in traced(*args))


@pytest.mark.parametrize("case", CALLS, ids=str)
def test_fake_tensors_reach_no_kernel(stand_in, case):
    _, fn, make = CALLS[case]
    mode = FakeTensorMode()
    args = [mode.from_tensor(t) for t in make()]
    with mode:
        inside = tensors(fn(*args))
    real = tensors(fn(*args))  # outside of the mode: the tensors themselves carry it
    assert not any(stand_in.values())
    assert [t.shape for t in inside] == [t.shape for t in real] and all(hasattr(t, "fake_mode") for t in inside + real)


def test_a_subclass_in_any_place_is_not_read_as_plain_memory(stand_in):
    """A wrapper's data pointer is NULL, which the library takes for "no weight": the call must go through the op."""
    from torch.testing._internal.two_tensor import TwoTensor

    w = torch.nn.Parameter(N(8))
    rms_norm(N(4, 8), TwoTensor(w.detach(), w.detach()))
    assert stand_in["rms_norm_forward"] == 2  # once for each of the wrapped tensors


@pytest.mark.parametrize("case", CALLS, ids=str)
def test_plain_calls_go_straight_to_the_library(stand_in, case):
    _, fn, make = CALLS[case]
    with pytest.raises(AssertionError, match="past the registered op"):
        fn(*make())
    with pytest.raises(AssertionError, match="past the registered op"):
        fn(*(torch.nn.Parameter(t) for t in make()))


@pytest.mark.parametrize("case", CALLS, ids=str)
def test_forward_mode_is_refused(case):
    """A dual tensor in any place; a result without its tangent would be a wrong derivative."""
    from torch.autograd import forward_ad

    _, fn, make = CALLS[case]
    for i in range(len(make())):
        args = list(make())
        with forward_ad.dual_level():
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*args)
            with pytest.raises(RuntimeError, match="no CPU path"):  # an open level alone changes nothing
                fn(*make())
    args = make()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: fn(x, *args[1:]), args[:1], args[:1])


def test_recorded_ops_check_what_they_are_given(monkeypatch):
    """A recorded program runs the op on tensors of other shapes and strides than it was recorded with."""
    from spear_b200.ops.norm import interface as norm
    from spear_b200.ops.ssm import conv, scan

    called = []
    monkeypatch.setattr(_call, "call", lambda name, index, *args: called.append(name))
    monkeypatch.setattr(_call, "query", lambda *a: 4)
    monkeypatch.setattr(_call, "on_gpu", lambda what, first, *others: first.get_device())
    E = torch.empty
    x, w, y, rstd, q = N(4, 8), N(8), E(4, 8), E(4), E(4, 8).to(torch.float8_e4m3fn)
    norm._op_forward(x, None, w, y, None, rstd, 1e-6)
    norm._op_8bit(x, None, w, q, None, E(4), 1e-6, True)
    norm._op_backward(x, w, y, None, rstd, E(4, 8), None, E(8))
    conv._op_forward(N(2, 5, 8), N(8, 4), None, None, None, E(2, 5, 8), None, False)
    conv._op_backward(N(2, 5, 8), N(8, 4), None, None, None, N(2, 5, 8), None, E(2, 5, 8), E(8, 4), None, None, False)
    conv._op_step(N(2, 8), N(2, 3, 8), N(8, 4), None, E(2, 8), E(2, 3, 8), False)
    tokens = (N(2, 5, 8), N(2, 5, 8), N(8, 4), N(2, 5, 4), N(2, 5, 4), None, None, None)
    scan._op_forward(*tokens, None, None, E(2, 5, 8), None, E(2, 1, 8, 4), False)
    back = lambda: [E(2, 1, 8, 4), N(2, 5, 8), None, E(2, 5, 8), E(2, 5, 8), E(48), E(2, 5, 4), E(2, 5, 4), None, None, False]
    scan._op_backward(*tokens, None, *back())
    one = (N(2, 8), N(2, 8), N(8, 4), N(2, 4), N(2, 4))
    scan._op_step(*one, E(2, 8, 4), None, None, None, E(2, 8), E(2, 8, 4), False)
    assert len(called) == 9
    bad = [
        lambda: norm._op_forward(x, None, w, E(3, 8), None, rstd, 1e-6),
        lambda: norm._op_forward(x, None, w, E(8, 4).t(), None, rstd, 1e-6),
        lambda: norm._op_forward(x, None, w, y, None, E(3), 1e-6),
        lambda: norm._op_forward(x, x, w, y, None, rstd, 1e-6),
        lambda: norm._op_forward(x, None, N(7), y, None, rstd, 1e-6),
        lambda: norm._op_8bit(x, None, w, y, None, E(4), 1e-6, False),
        lambda: norm._op_8bit(x, None, w, q, None, E(5), 1e-6, False),
        lambda: norm._op_8bit(x, x, w, q, None, E(4), 1e-6, True),
        lambda: norm._op_backward(x, w, y, None, E(3), E(4, 8), None, E(8)),
        lambda: norm._op_backward(x, None, y, None, rstd, E(4, 8), None, E(8)),
        lambda: norm._op_backward(x, w, y, E(4, 8).half(), rstd, E(4, 8), None, E(8)),
        lambda: conv._op_forward(N(2, 5, 8), N(8, 5), None, None, None, E(2, 5, 8), None, False),
        lambda: conv._op_forward(N(2, 5, 8), N(8, 4), None, None, None, E(2, 4, 8), None, False),
        lambda: conv._op_forward(N(2, 5, 8), N(8, 4), None, None, None, E(2, 5, 8), E(2, 2, 8), False),
        lambda: conv._op_backward(N(2, 5, 8), N(8, 4), None, None, None, N(2, 4, 8), None, E(2, 5, 8), None, None, None, False),
        lambda: conv._op_step(N(2, 8), N(2, 2, 8), N(8, 4), None, E(2, 8), E(2, 3, 8), False),
        lambda: conv._op_step(N(2, 8), N(2, 3, 8), N(8, 4), None, E(1, 8), E(2, 3, 8), False),
        lambda: scan._op_forward(*tokens, None, None, E(2, 5, 8), None, E(2, 2, 8, 4), False),
        lambda: scan._op_forward(*tokens, None, None, E(2, 5, 8), E(2, 8, 3), None, False),
        lambda: scan._op_step(*one, E(2, 8, 4), None, None, None, E(2, 8), E(2, 8, 3), False),
    ]
    for i in (0, 1, 3, 4, 5, 6, 7):  # each buffer of the scan's backward, one element short
        args = back()
        args[i] = args[i].flatten()[:-1]
        bad.append(lambda args=args: scan._op_backward(*tokens, None, *args))
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert len(called) == 9
    # strides that the kernels do not read: the op brings them into order itself
    seen = []
    monkeypatch.setattr(_call, "call", lambda name, index, *args: seen.append(args))
    conv._op_forward(N(2, 8, 5).transpose(1, 2), N(4, 8).t(), None, None, None, E(2, 5, 8), None, False)
    assert seen[0][7:13] == (2, 5, 8, 4, 40, 8)


def test_recorded_ops_without_tokens(monkeypatch):
    """Recorded at some length, run at length 0: states pass through, sums over no tokens are 0, nothing is launched."""
    from spear_b200.ops.norm import interface as norm
    from spear_b200.ops.ssm import conv, scan

    monkeypatch.setattr(_call, "call", lambda name, *args: pytest.fail(name))
    monkeypatch.setattr(_call, "on_gpu", lambda what, first, *others: first.get_device())
    E = lambda *shape: torch.full(shape, 7.0)
    s, ds, out, dw = N(2, 3, 8), N(2, 3, 8), E(2, 3, 8), E(8, 4)
    conv._op_forward(E(2, 0, 8), N(8, 4), None, s, None, E(2, 0, 8), out, False)
    assert torch.equal(out, s)
    conv._op_forward(E(2, 0, 8), N(8, 4), None, None, None, E(2, 0, 8), out, False)
    assert (out == 0).all()
    conv._op_backward(E(2, 0, 8), N(8, 4), None, s, None, E(2, 0, 8), ds, E(2, 0, 8), dw, None, out, False)
    assert torch.equal(out, ds) and (dw == 0).all()
    tokens = (E(2, 0, 8), E(2, 0, 8), N(8, 4), E(2, 0, 4), E(2, 0, 4), None, None, None)
    h, out, dp = N(2, 8, 4), E(2, 8, 4), E(48)
    scan._op_forward(*tokens, h, None, E(2, 0, 8), out, None, False)
    assert torch.equal(out, h)
    scan._op_backward(*tokens, None, E(2, 0, 8, 4), E(2, 0, 8), None, E(2, 0, 8), E(2, 0, 8), dp, E(2, 0, 4), E(2, 0, 4), None, out, False)
    assert (out == 0).all() and (dp == 0).all()
    dw = E(8)
    norm._op_backward(E(0, 8), N(8), E(0, 8), None, E(0), E(0, 8), None, dw)
    assert (dw == 0).all()


@pytest.mark.parametrize("case", ["norm 8 bits", "conv token", "scan token"])
def test_forms_without_gradient_have_none_when_recorded(stand_in, case, recwarn):
    _, fn, make = CALLS[case]
    args = [torch.nn.Parameter(t) for t in make()]
    seen = []

    def run(*args):
        out = tensors(fn(*args))
        seen.extend(t.requires_grad for t in out)
        return out

    with FakeTensorMode(allow_non_fake_inputs=True):
        fake = tensors(fn(*[torch.nn.Parameter(torch.empty(t.shape)) for t in args]))
    traced = make_fx(run)(*args)
    assert not any(seen) and not any(t.requires_grad for t in fake + tensors(traced(*args)))
    assert not [w for w in recwarn.list if "autograd kernel was not registered" in str(w.message)]
