"""Recorded programs of the token-major operators (make_fx, torch.jit.trace, torch.compile without gradients) run the same kernels
as the calls that they were recorded from: the same bits, on other inputs and, where the recorder keeps shapes open, other lengths."""

from __future__ import annotations

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu


def N(*shape):
    return torch.randn(*shape, device="cuda")


def calls():
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit
    from spear_b200.ops.ssm import causal_conv, causal_conv_step, selective_scan, selective_scan_step

    lengths = torch.tensor([5, 70, 0], device="cuda", dtype=torch.int32)
    scan_args = lambda L: (N(3, L, 40), N(3, L, 40), -torch.rand(40, 7, device="cuda"), N(3, L, 7), N(3, L, 7), N(40))
    return {
        "norm": (lambda x, w, r: rms_norm(x, w, r), lambda L: (N(2, L, 72), N(72), N(2, L, 72))),
        "norm 8 bits": (lambda x, w: tuple(t.float() for t in rms_norm_8bit(x, w, block=128)), lambda L: (N(L, 200), N(200))),
        "conv": (lambda x, w, s: causal_conv(x, w, activation="silu", initial_state=s, return_state=True),
                 lambda L: (N(3, L, 24), N(24, 4), N(3, 3, 24))),
        "conv padded": (lambda x, w: causal_conv(x, w, lengths=lengths), lambda L: (N(3, L, 24), N(24, 2))),
        "conv token": (lambda x, s, w: causal_conv_step(x, s, w), lambda L: (N(L, 24), N(L, 3, 24), N(24, 4))),
        "scan": (lambda *a: selective_scan(*a, delta_softplus=True, lengths=lengths, return_state=True), scan_args),
        "scan token": (lambda x, d, A, B, C, s: selective_scan_step(x, d, A, B, C, s, delta_softplus=True),
                       lambda L: (N(L, 24), N(L, 24), -torch.rand(24, 16, device="cuda"), N(L, 16), N(L, 16), N(L, 24, 16))),
    }


CASES = ("norm", "norm 8 bits", "conv", "conv padded", "conv token", "scan", "scan token")


def same(got, want):
    got, want = ([o] if torch.is_tensor(o) else list(o) for o in (got, want))
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("case", CASES)
def test_make_fx(case):
    fn, make = calls()[case]
    traced = make_fx(fn)(*make(70))
    args = make(70)
    assert same(traced(*args), fn(*args))


@pytest.mark.parametrize("case", ["norm", "conv", "conv padded", "scan"])
def test_make_fx_of_a_training_pass(case):
    fn, make = calls()[case]

    def step(*args):
        leaves = [a.detach().requires_grad_(True) for a in args]
        outs = fn(*leaves)
        outs = [outs] if torch.is_tensor(outs) else list(outs)
        return [*outs, *torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])]

    traced = make_fx(step)(*make(70))
    args = make(70)
    assert same([t.detach() for t in traced(*args)], [t.detach() for t in step(*args)])


@pytest.mark.parametrize("case", CASES)
@pytest.mark.filterwarnings("ignore")
def test_jit_trace(case):
    fn, make = calls()[case]
    traced = torch.jit.trace(fn, make(70), check_trace=False)
    for L in (70, 33):
        args = make(L)
        assert same(traced(*args), fn(*args)), L


@pytest.mark.filterwarnings("ignore")
def test_a_recorded_program_on_other_strides():
    """Recorded on dense channels, run on a transposed tensor: the copy that the public call makes is not part of the record."""
    from spear_b200.ops.ssm import causal_conv

    w = N(24, 4)
    fn = lambda x: causal_conv(x, w)
    traced = torch.jit.trace(fn, (N(3, 70, 24),), check_trace=False)
    x = N(3, 24, 70).transpose(1, 2)
    assert same(traced(x), fn(x))


@pytest.mark.parametrize("case", CASES)
def test_compile_without_gradients(case):
    fn, make = calls()[case]
    args = make(70)
    torch._dynamo.reset()
    with torch.no_grad():
        assert same(torch.compile(fn)(*args), fn(*args))


def test_compiled_token_in_place():
    """state and state_out are the same tensor inside a compiled program."""
    from spear_b200.ops.ssm import causal_conv_step, selective_scan_step

    def step(x, w, cs, d, A, B, C, ss):
        y, cs = causal_conv_step(x, cs, w, activation="silu", state_out=cs)
        return selective_scan_step(y, d, A, B, C, ss, delta_softplus=True, state_out=ss)[0]

    args = [N(3, 24), N(24, 4), N(3, 3, 24), N(3, 24), -torch.rand(24, 16, device="cuda"), N(3, 16), N(3, 16), N(3, 24, 16)]
    other = [a.clone() for a in args]
    torch._dynamo.reset()
    with torch.no_grad():
        compiled = torch.compile(step)
        for _ in range(3):
            assert torch.equal(compiled(*args), step(*other))
            assert all(torch.equal(a, b) for a, b in zip(args, other))


def test_functional_transforms_are_refused():
    """A wrapped tensor has no memory of its own: an error, not a result that the transform does not see."""
    from spear_b200.ops.norm import rms_norm
    from spear_b200.ops.ssm import causal_conv, selective_scan_step

    x, w = N(3, 5, 24), N(24, 4)
    for call in (lambda: torch.vmap(rms_norm)(x), lambda: torch.func.grad(lambda t: rms_norm(t).sum())(x),
                 lambda: torch.func.grad(lambda t: causal_conv(x, t).sum())(w), lambda: torch.func.jvp(rms_norm, (x,), (x,)),
                 lambda: torch.vmap(lambda s: selective_scan_step(x[0], x[0], -w, x[0, :, :4], x[0, :, :4], s))(N(2, 5, 24, 4))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


@pytest.mark.parametrize("case", ["norm", "conv", "conv padded", "scan"])
@pytest.mark.filterwarnings("ignore")
def test_jit_trace_of_a_training_pass(case):
    """Traced with inputs that require grad: the outputs and the gradients of the calls themselves, on other inputs."""
    fn, make = calls()[case]
    leaves = lambda: [a.requires_grad_(True) for a in make(70)]
    traced = torch.jit.trace(fn, leaves(), check_trace=False)
    args = leaves()
    got, want = ([o] if torch.is_tensor(o) else list(o) for o in (traced(*args), fn(*args)))
    ups = [torch.randn_like(o) for o in want]
    assert same(got, want)
    assert same(torch.autograd.grad(got, args, ups), torch.autograd.grad(want, args, ups))
