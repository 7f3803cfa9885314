"""What autograd may ask of the operators' training passes: some gradients only, a pass twice, saved tensors elsewhere, a recorded
backward pass, second derivatives (refused), and no memory left behind."""

from __future__ import annotations

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu


def N(*shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda").to(dtype)


def norm(weight=True, residual=True):
    from spear_b200.ops.norm import rms_norm

    args = {"x": N(6, 72), "weight": N(72) if weight else None, "residual": N(6, 72) if residual else None}
    return rms_norm, args


def conv(bias=True, initial=True):
    from spear_b200.ops.ssm import causal_conv

    args = {"x": N(2, 37, 24), "weight": N(24, 4), "bias": N(24) if bias else None, "initial_state": N(2, 3, 24) if initial else None}
    return lambda **kw: causal_conv(**kw, activation="silu", return_state=True), args


def scan(D=True, z=True, bias=True, initial=True):
    from spear_b200.ops.ssm import selective_scan

    args = {"x": N(2, 37, 24), "delta": N(2, 37, 24), "A": -torch.rand(24, 5, device="cuda"), "B": N(2, 37, 5), "C": N(2, 37, 5),
            "D": N(24) if D else None, "z": N(2, 37, 24) if z else None, "delta_bias": N(24) if bias else None,
            "initial_state": N(2, 24, 5) if initial else None}
    return lambda **kw: selective_scan(**kw, delta_softplus=True, return_state=True), args


def outs(result):
    return [result] if torch.is_tensor(result) else list(result)


def grads(fn, args, names, ups=None, **kw):
    leaves = {n: t if t is None else t.detach().requires_grad_(n in names) for n, t in args.items()}
    got = outs(fn(**leaves))
    ups = [torch.ones_like(o) for o in got] if ups is None else ups
    return dict(zip(names, torch.autograd.grad(got, [leaves[n] for n in names], ups, **kw)))


@pytest.mark.parametrize("make", [norm, conv, scan])
def test_every_argument_by_itself_and_any_set_of_options(make):
    """The gradient of one argument has the bits that it has among all, whichever optional arguments are there."""
    for given in itertools.product((True, False), repeat=make.__code__.co_argcount):
        fn, args = make(*given)
        there = [n for n, t in args.items() if t is not None]
        whole = grads(fn, args, there)
        for n in there:
            assert torch.equal(grads(fn, args, [n])[n], whole[n]), (n, given)
            assert whole[n].shape == args[n].shape and whole[n].dtype == args[n].dtype
        # inputs that require grad, of which autograd is asked for one
        leaves = {n: t if t is None else t.detach().requires_grad_(True) for n, t in args.items()}
        got = outs(fn(**leaves))
        for n in there:
            one, = torch.autograd.grad(got, [leaves[n]], [torch.ones_like(o) for o in got], retain_graph=True)
            assert torch.equal(one, whole[n]), (n, given)


@pytest.mark.parametrize("make", [norm, conv, scan])
def test_one_output_of_two(make):
    fn, args = make()
    there = list(args)
    for i in range(2):
        leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
        got = outs(fn(**leaves))
        one = torch.autograd.grad(got[i], list(leaves.values()), torch.ones_like(got[i]), allow_unused=True)
        zero = [torch.ones_like(o) if j == i else torch.zeros_like(o) for j, o in enumerate(got)]
        both = grads(fn, args, there, zero)
        for n, g in zip(there, one):
            assert (torch.zeros_like(both[n]) if g is None else g).sub(both[n]).abs().max() <= 1e-6 * both[n].abs().max(), (i, n)


@pytest.mark.parametrize("make", [norm, conv, scan])
def test_second_derivatives_are_refused_not_zero(make):
    fn, args = make()
    leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
    y = outs(fn(**leaves))[0]
    gx, = torch.autograd.grad(y.sum(), leaves["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (y.sum() + gx.square().sum()).backward()


@pytest.mark.parametrize("make", [norm, conv, scan])
def test_a_pass_runs_no_python_and_twice_the_same(make):
    fn, args = make()
    leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
    got = outs(fn(**leaves))
    assert not isinstance(got[0].grad_fn, torch.autograd.function.BackwardCFunction)
    ups = [torch.randn_like(o) for o in got]
    first = torch.autograd.grad(got, list(leaves.values()), ups, retain_graph=True)
    again = torch.autograd.grad(got, list(leaves.values()), ups)
    assert all(torch.equal(a, b) and a.data_ptr() != b.data_ptr() for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(got, list(leaves.values()), ups)


@pytest.mark.parametrize("make", [norm, conv, scan])
def test_the_python_functions_of_recorded_calls_agree(make):
    """torch.compile and the other recorders take the functions in Python; the same steps, the same bits."""
    from spear_b200.ops.norm import interface as n
    from spear_b200.ops.ssm import conv as c, scan as s

    fn, args = make()
    leaves = [t.detach().requires_grad_(True) for t in args.values()]
    eager = outs(fn(**dict(zip(args, leaves))))
    if make is norm:
        recorded = n._RMSNorm.apply(*leaves, 1e-6)
    elif make is conv:
        recorded = c._CausalConv.apply(*leaves, None, True, True)
    else:
        recorded = s._SelectiveScan.apply(*leaves, None, True, True)
    ups = [torch.randn_like(o) for o in eager]
    for a, b in zip([*eager, *torch.autograd.grad(eager, leaves, ups)], [*recorded, *torch.autograd.grad(list(recorded), leaves, ups)]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("make", [norm, conv, scan])
def test_a_recorded_backward_pass_of_an_eager_forward(make):
    from torch.fx.experimental.proxy_tensor import make_fx

    fn, args = make()
    leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
    got = outs(fn(**leaves))
    back = lambda *ups: torch.autograd.grad(got, list(leaves.values()), list(ups), retain_graph=True)
    traced = make_fx(back)(*(torch.ones_like(o) for o in got))
    assert any("_backward" in str(node.target) and "spear_btp" in str(node.target) for node in traced.graph.nodes)
    ups = [torch.randn_like(o) for o in got]
    assert all(torch.equal(a, b) for a, b in zip(traced(*ups), back(*ups)))


def layer():
    from spear_b200.nn.ssm import SelectiveSSM

    torch.manual_seed(3)
    return SelectiveSSM(64).cuda(), N(2, 50, 64)


def test_checkpointed_and_hooked():
    """Recomputed in the backward pass, and saved tensors kept on the host meanwhile: the same gradients."""
    from torch.utils.checkpoint import checkpoint

    m, u = layer()
    params = list(m.parameters())
    want = torch.autograd.grad(m(u).square().sum(), params)
    again = torch.autograd.grad(checkpoint(m, u, use_reentrant=False).square().sum(), params)
    with torch.autograd.graph.save_on_cpu():
        kept = torch.autograd.grad(m(u).square().sum(), params)
    for a, b, c in zip(want, again, kept):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_compiled_autograd():
    m, u = layer()
    params = list(m.parameters())
    want = torch.autograd.grad(m(u).square().sum(), params)
    loss = m(u).square().sum()
    with torch._dynamo.compiled_autograd._enable(torch.compile(backend="aot_eager")):
        loss.backward()
    for p, g in zip(params, want):
        assert (p.grad - g).norm() <= 1e-5 * g.norm()  # the same kernels, other orders in torch's sums


def test_nothing_is_left_behind():
    m, u = layer()
    fns = [make() for make in (norm, conv, scan)]

    def passes():
        for fn, args in fns:
            grads(fn, args, list(args))
            leaves = {n: t.detach().requires_grad_(True) for n, t in args.items()}
            outs(fn(**leaves))  # a graph that is dropped without a backward pass
        m(u).sum().backward()
        for p in m.parameters():
            p.grad = None

    passes()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        passes()
    assert torch.cuda.memory_allocated() == before


def test_saved_tensors_that_change_are_noticed():
    fn, args = conv()
    leaves = {n: t.detach().requires_grad_(n != "initial_state") for n, t in args.items()}
    y = outs(fn(**leaves))[0]
    leaves["initial_state"].zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_on_a_side_stream():
    m, u = layer()
    params = list(m.parameters())
    want = torch.autograd.grad(m(u).square().sum(), params)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(m(u).square().sum(), params)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_threads_at_once():
    """Passes on four threads, each on a stream of its own, among them the first ones of their thread."""
    import threading

    fn, args = conv()
    ready = torch.cuda.Event()
    ready.record()
    got = [None] * 4

    def work(i):
        stream = torch.cuda.Stream()
        stream.wait_event(ready)
        with torch.cuda.stream(stream):
            for _ in range(50):
                got[i] = grads(fn, args, list(args))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    want = grads(fn, args, list(args))
    assert all(torch.equal(g[n], want[n]) for g in got for n in args)


def test_one_tensor_for_two_arguments():
    from spear_b200.ops.norm import rms_norm
    from spear_b200.ops.ssm import selective_scan

    x, w, up = N(6, 72), N(72), N(6, 72)
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    apart = torch.autograd.grad(list(rms_norm(a, w, b)), [a, b], [up, up])
    both, = torch.autograd.grad(list(rms_norm(a, w, a)), a, [up, up])
    assert torch.equal(both, apart[0] + apart[1])
    sum(o.sum() for o in rms_norm(a, w, b)).backward()
    assert torch.equal(a.grad, b.grad) and a.grad.data_ptr() != b.grad.data_ptr()
    x, m, A = N(2, 37, 24), N(2, 37, 5), -torch.rand(24, 5, device="cuda")
    leaf = lambda t: t.clone().requires_grad_(True)
    x1, x2, m1, m2 = leaf(x), leaf(x), leaf(m), leaf(m)
    apart = torch.autograd.grad(selective_scan(x1, x2, A, m1, m2, delta_softplus=True).sum(), [x1, x2, m1, m2])
    both = torch.autograd.grad(selective_scan(x1, x1, A, m1, m1, delta_softplus=True).sum(), [x1, m1])
    assert torch.equal(both[0], apart[0] + apart[1]) and torch.equal(both[1], apart[2] + apart[3])
