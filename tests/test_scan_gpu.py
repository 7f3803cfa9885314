"""The selective scan against its definition in 64 bits; every tolerance is the running error bound of tests/scan_oracle.py."""

from __future__ import annotations

import pytest
import torch

import scan_oracle

pytestmark = pytest.mark.gpu

NAMES = ("x", "delta", "A", "B", "C", "D", "z", "delta_bias", "initial_state")


def inputs(Bsz, L, dim, N, dtype, *, skip=True, gate=True, bias=True, initial=False, lengths=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    v = {"x": r(Bsz, L, dim).to(dtype), "delta": (r(Bsz, L, dim) - 2).to(dtype), "A": -torch.exp(r(dim, N)),
         "B": r(Bsz, L, N).to(dtype), "C": r(Bsz, L, N).to(dtype), "D": r(dim) if skip else None,
         "z": r(Bsz, L, dim).to(dtype) if gate else None, "delta_bias": r(dim) if bias else None,
         "initial_state": r(Bsz, dim, N) if initial else None, "lengths": None}
    if lengths:
        n = torch.randint(0, L + 1, (Bsz,), generator=g, device="cuda", dtype=torch.int32)
        n[0] = L
        if Bsz > 1:
            n[-1] = 0
        if Bsz > 2:
            n[1] = 1
        v["lengths"] = n
    return v


def run(v, softplus=True, state=True):
    from spear_b200.ops.ssm import selective_scan

    return selective_scan(v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], delta_bias=v["delta_bias"], delta_softplus=softplus,
                          initial_state=v["initial_state"], lengths=v["lengths"], return_state=state)


def oracle(v, softplus=True, **kw):
    return scan_oracle.scan(v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], delta_bias=v["delta_bias"], softplus=softplus,
                            initial=v["initial_state"], lengths=v["lengths"], **kw)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def check(got, want, dtype, name):
    assert got.dtype == dtype and got.shape == want.v.shape, name
    bound = want.to(dtype)
    err = (got.double() - want.v).abs()
    bad = ~((err <= bound) | bound.isinf()).cpu()
    n, worst = bad.sum().item(), (err / bound).nan_to_num(0.0).max().item()
    assert n == 0, f"{name}: {n} of {bad.numel()} outside, worst {worst:.3g} of the bound"


# lengths around the tile of 16 and the step of 4, one token, long enough to be split; channel counts and states that fill no warp
SHAPES = [(1, 1, 1, 1), (1, 1, 32, 16), (2, 2, 8, 4), (1, 3, 33, 16), (2, 15, 40, 16), (3, 16, 64, 8), (2, 17, 130, 16), (1, 31, 24, 32),
          (2, 33, 20, 64), (1, 64, 7, 3), (2, 65, 12, 13), (1, 100, 36, 17), (2, 40, 19, 33), (1, 50, 9, 61), (3, 300, 16, 16), (1, 777, 40, 16),
          (2, 1000, 6, 8), (1, 520, 10, 64), (1, 640, 66, 32), (2, 37, 24, 64), (1, 50, 48, 20), (2, 20, 136, 7)]
VARIANTS = [dict(), dict(skip=False, gate=False, bias=False), dict(initial=True, gate=False), dict(lengths=True, initial=True)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_forward(shape, dtype):
    for i, kw in enumerate(VARIANTS):
        v = inputs(*shape, dtype, seed=i, **kw)
        softplus = i != 2
        if not softplus:  # step sizes as they are: some negative, which is a growing state
            v["delta"] = (v["delta"].float() * 0.05 + 0.1).to(dtype)
            v["delta_bias"] = v["delta_bias"] * 0.05
        y, state = run(v, softplus)
        want = oracle(v, softplus)
        check(y, want["y"], dtype, "y")
        check(state, want["state"], torch.float32, "state")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_backward(shape, dtype):
    Bsz, L, dim, N = shape
    for i, kw in enumerate(VARIANTS):
        v = inputs(*shape, dtype, seed=20 + i, **kw)
        softplus = i != 1
        if not softplus:
            v["delta"] = (v["delta"].float() * 0.05 + 0.1).to(dtype)
        g = torch.Generator(device="cuda").manual_seed(99)
        dy = torch.randn(Bsz, L, dim, generator=g, device="cuda").to(dtype)
        ds = torch.randn(Bsz, dim, N, generator=g, device="cuda")
        names = [n for n in NAMES if v[n] is not None]
        for n in names:
            v[n].requires_grad_(True)
        out = run(v, softplus)
        got = dict(zip(names, torch.autograd.grad(out, [v[n] for n in names], [dy, ds])))
        want = oracle(v, softplus, dy=dy, dstate=ds)
        for n in names:
            key = "d" + {"delta_bias": "bias", "initial_state": "initial"}.get(n, n)
            check(got[n], want[key], v[n].dtype, key)


def test_gradients_of_differences():
    v = inputs(2, 37, 12, 5, torch.float32, initial=True, lengths=True, seed=3)
    v["lengths"] = torch.tensor([37, 21], device="cuda", dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(5)
    dy = torch.randn(2, 37, 12, generator=g, device="cuda")
    dirs = {n: torch.randn(v[n].shape, generator=g, device="cuda") for n in NAMES}
    for n in NAMES:
        v[n].requires_grad_(True)
    grads = dict(zip(NAMES, torch.autograd.grad(run(v, state=False), [v[n] for n in NAMES], dy)))
    bounds = oracle(v, dy=dy)
    got, size, off = 0.0, 0.0, 0.0
    for n in NAMES:
        key = "d" + {"delta_bias": "bias", "initial_state": "initial"}.get(n, n)
        got = got + (grads[n].double() * dirs[n].double()).sum()
        size = size + (grads[n].double() * dirs[n].double()).abs().sum()
        off = off + (bounds[key].to(torch.float32) * dirs[n].double().abs()).sum()

    def f(s):
        w = dict(v)
        for n in NAMES:
            w[n] = v[n].detach().double() + s * dirs[n].double()
        return (oracle(w)["y"].v * dy.double()).sum()

    want = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(got - want) <= off + 1e-7 * size  # differences: about 1e-10 of third derivatives and 1e-11 of rounding, each times up to 100


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 8, 16), (3, 33, 16), (5, 100, 7), (64, 40, 8), (2, 24, 64), (1, 1, 1), (130, 9, 32)], ids=str)
def test_steps_continue_a_prompt(dtype, shape):
    from spear_b200.ops.ssm import selective_scan_step

    Bsz, dim, N = shape
    v = inputs(Bsz, 11, dim, N, dtype, seed=4)
    want = oracle(v)
    cut = {n: (t[:, :6] if n in ("x", "delta", "B", "C", "z") else t) for n, t in v.items()}
    _, state = run(cut)
    inplace = state.clone()
    for t in range(6, 11):
        tok = (v["x"][:, t], v["delta"][:, t], v["A"], v["B"][:, t], v["C"][:, t])
        before = state.clone()
        y, new = selective_scan_step(*tok, state, v["D"], v["z"][:, t], delta_bias=v["delta_bias"], delta_softplus=True)
        assert torch.equal(state, before)
        y2, same = selective_scan_step(*tok, inplace, v["D"], v["z"][:, t], delta_bias=v["delta_bias"], delta_softplus=True, state_out=inplace)
        assert same is inplace and torch.equal(y, y2) and torch.equal(new, inplace)
        check(y, want["y"][:, t], dtype, "y")
        state = new
    check(state, want["state"], torch.float32, "state")


def test_prompt_in_two_parts():
    v = inputs(2, 500, 48, 16, torch.float32, seed=6)
    want = oracle(v)
    part = lambda a, b: {n: (t[:, a:b] if n in ("x", "delta", "B", "C", "z") else t) for n, t in v.items()}  # noqa: E731
    y1, s1 = run(part(0, 211))
    y2, s2 = run({**part(211, 500), "initial_state": s1})
    check(torch.cat([y1, y2], 1), want["y"], torch.float32, "y")
    check(s2, want["state"], torch.float32, "state")


@pytest.mark.parametrize("L", [70, 900])  # in one piece, and split over the tokens
def test_what_lies_behind_the_end_does_not_matter(L):
    v = inputs(4, L, 24, 16, torch.bfloat16, initial=True, seed=7)
    v["lengths"] = torch.tensor([0, 1, 33, L], device="cuda", dtype=torch.int32)
    tok = ("x", "delta", "B", "C", "z")
    dy = torch.randn(4, L, 24, device="cuda").bfloat16()

    def both(w, up):
        leaves = {n: w[n].detach().clone().requires_grad_(True) for n in NAMES}
        out = run({**leaves, "lengths": v["lengths"]})
        return [*out, *torch.autograd.grad(out[0], list(leaves.values()), up)]

    dirty, dyd = dict(v), dy.clone()
    for n in tok:
        dirty[n] = v[n].clone()
    for b in range(4):
        for n in tok:
            dirty[n][b, v["lengths"][b]:] = float("nan") if b % 2 else float("inf")
        dyd[b, v["lengths"][b]:] = float("nan")
    clean = both(v, dy)
    for a, b in zip(clean, both(dirty, dyd)):
        assert torch.equal(a, b)
    assert torch.equal(clean[1][0], v["initial_state"][0]) and (clean[0][0] == 0).all()
    with torch.no_grad():
        y = run({**v, "lengths": torch.tensor([-3, 1, 33, L + 9], device="cuda", dtype=torch.int32)})[0]
    assert torch.equal(y, clean[0])


def test_not_a_number_stays_in_its_sequence_and_channel():
    """An infinite or undefined input reaches its own channel from its token on, and nothing before or beside it."""
    for N in (16, 5):  # full and padded states
        v = inputs(3, 40, 70, N, torch.float32, seed=8)
        y = run(v, state=False)
        w = {n: t.clone() if torch.is_tensor(t) else t for n, t in v.items()}
        w["x"][1, 20, 3], w["x"][1, 10, 69] = float("nan"), float("inf")
        y2 = run(w, state=False)
        same = torch.ones_like(y, dtype=torch.bool)
        same[1, 20:, 3] = False
        same[1, 10:, 69] = False
        assert torch.equal(y[same], y2[same])
        assert y2[1, 20:, 3].isnan().all() and not y2[1, 10, 69].isfinite()
        w = {n: t.clone() if torch.is_tensor(t) else t for n, t in v.items()}
        w["delta"][0, 5, 7] = float("nan")
        w["A"][9, 2] = float("nan")
        y3 = run(w, state=False)
        assert y3[0, 5:, 7].isnan().all() and y3[:, :, 9].isnan().all()
        rest = torch.ones_like(same)
        rest[0, 5:, 7] = False
        rest[:, :, 9] = False
        assert torch.equal(y[rest], y3[rest])


def test_extreme_step_sizes():
    v = inputs(1, 30, 40, 16, torch.float32, seed=9)
    v["delta"][:, ::3] = 60.0    # the state is forgotten
    v["delta"][:, 1::3] = -60.0  # the state is kept as it is
    v["delta"][:, 2, :] = -200.0
    want = oracle(v)
    y, state = run(v)
    # forgotten states underflow to 0 where 64 bits keep them: below float32's least normal number
    for got, q in ((y, want["y"]), (state, want["state"])):
        assert ((got.double() - q.v).abs() <= q.to(torch.float32) + 1e-36).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_offsets(dtype):
    from spear_b200.ops.ssm import selective_scan_step

    v = inputs(3, 45, 40, 16, dtype, seed=10)
    wide = torch.randn(3, 45, 200, device="cuda").to(dtype)
    for off in (0, 8, 3):
        w = dict(v)
        w["x"], w["z"] = wide[:, :, off:off + 40], wide[:, :, off + 41:off + 81]
        w["B"], w["C"] = wide[:, :, off + 82:off + 98], wide[:, :, off + 99:off + 115]
        w["delta"] = v["delta"].transpose(0, 1).contiguous().transpose(0, 1)
        w["A"] = torch.cat([v["A"].new_zeros(off), v["A"].reshape(-1)])[off:].view(40, 16)
        base = torch.randn(3 * 40 * 16 + off, device="cuda")
        w["initial_state"] = base[off:].view(3, 40, 16)
        c = {n: t.clone(memory_format=torch.contiguous_format) if torch.is_tensor(t) else t for n, t in w.items()}
        ya, sa = run(w)
        yb, sb = run(c)
        assert torch.equal(ya, yb) and torch.equal(sa, sb)
        up = torch.randn(40, 45, 3, device="cuda").to(dtype).permute(2, 1, 0)
        grads = []
        for t in (w, c):
            leaves = {n: t[n].detach().requires_grad_(True) for n in NAMES}
            grads.append(torch.autograd.grad(run({**leaves, "lengths": None}, state=False), list(leaves.values()), up))
        assert all(torch.equal(a, b) for a, b in zip(*grads))
        st = torch.randn(3, 40, 16, device="cuda")
        args = lambda q: (q["x"][:, 4], q["delta"][:, 4], q["A"], q["B"][:, 4], q["C"][:, 4], st, q["D"], q["z"][:, 4])  # noqa: E731
        assert torch.equal(selective_scan_step(*args(w))[1], selective_scan_step(*args(c))[1])
    t = dict(v)
    t["x"] = v["x"].transpose(1, 2).contiguous().transpose(1, 2)  # channels not dense: copied
    t["B"] = v["B"][:1].expand(3, -1, -1)
    assert torch.equal(run(t, state=False), run({**t, "x": t["x"].contiguous(), "B": t["B"].contiguous()}, state=False))
    with pytest.raises(ValueError, match="aligned"):
        s = torch.zeros(3 * 40 * 16 + 1, device="cuda")[1:].view(3, 40, 16)
        selective_scan_step(v["x"][:, 0], v["delta"][:, 0], v["A"], v["B"][:, 0], v["C"][:, 0], s)


def test_shared_input_sums_its_gradients():
    """One tensor in two places gets both gradients; a broadcast one the sum over what it was broadcast to."""
    v = inputs(2, 30, 24, 16, torch.float32, gate=True, seed=11)
    dy = torch.randn(2, 30, 24, device="cuda")
    a, b = (v["x"].clone().requires_grad_(True) for _ in range(2))
    ga, gb = torch.autograd.grad(run({**v, "x": a, "z": b}, state=False), [a, b], dy)
    c = v["x"].clone().requires_grad_(True)
    (gc,) = torch.autograd.grad(run({**v, "x": c, "z": c}, state=False), [c], dy)
    with torch.no_grad():
        same = run({**v, "x": a, "z": v["x"]}, state=False)
    assert same.shape == gc.shape
    a2, b2 = (v["x"].clone().requires_grad_(True) for _ in range(2))
    g2 = torch.autograd.grad(run({**v, "x": a2, "z": b2}, state=False), [a2, b2], dy)
    assert torch.equal(gc, g2[0] + g2[1]) and torch.equal(ga, g2[0]) and torch.equal(gb, g2[1])
    B1 = v["B"][:1].clone().requires_grad_(True)
    (g1,) = torch.autograd.grad(run({**v, "B": B1.expand(2, -1, -1)}, state=False), [B1], dy)
    Bf = v["B"][:1].expand(2, -1, -1).clone().requires_grad_(True)
    (gf,) = torch.autograd.grad(run({**v, "B": Bf}, state=False), [Bf], dy)
    assert torch.equal(g1, gf.sum(0, keepdim=True))


def test_streams_graphs_repeatability_and_empty():
    from spear_b200.ops.ssm import selective_scan, selective_scan_step

    v = inputs(2, 1200, 64, 16, torch.bfloat16, seed=12)
    want = run(v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(v)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs, xs = [], [], []
    for _ in range(2):  # two graphs, each with its own buffers, replayed in turn
        x = v["x"].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run({**v, "x": x}))
        graphs.append(graph), xs.append(x)
    xs[0].mul_(2)
    for i in (0, 1, 0):
        graphs[i].replay()
    assert all(torch.equal(a, b) for a, b in zip(outs[1], want))
    assert all(torch.equal(a, b) for a, b in zip(outs[0], run({**v, "x": v["x"] * 2})))
    state, tok = want[1].clone(), v["x"][:, 0].clone()
    args = (v["delta"][:, 0].clone(), v["A"], v["B"][:, 0].clone(), v["C"][:, 0].clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = selective_scan_step(tok, *args, state, v["D"], state_out=state)
    state.copy_(want[1])
    ref = want[1].clone()
    for _ in range(3):
        graph.replay()
        yw, ref = selective_scan_step(tok, *args, ref, v["D"])
        assert same_bits(y, yw) and same_bits(state, ref)  # steps that grow the state without bound: infinite values among them

    def train():
        leaves = {n: v[n].clone().requires_grad_(True) for n in NAMES if v[n] is not None}
        y = run({**v, **leaves}, state=False)
        return torch.autograd.grad(y, list(leaves.values()), torch.ones_like(y))

    assert all(torch.equal(a, b) for a, b in zip(train(), train()))
    e = inputs(2, 4, 8, 16, torch.float32, initial=True, seed=13)
    z = {n: (t[:, :0] if n in ("x", "delta", "B", "C", "z") else t) for n, t in e.items()}
    z["x"] = z["x"].requires_grad_(True)
    y, s = run(z)
    y.sum().backward()
    assert y.shape == (2, 0, 8) and torch.equal(s, e["initial_state"])
    none = {n: (t[:0] if n in ("x", "delta", "B", "C", "z", "initial_state") else t) for n, t in e.items()}
    assert run(none)[1].shape == (0, 8, 16)
    assert selective_scan_step(none["x"][:, 0], none["delta"][:, 0], e["A"], none["B"][:, 0], none["C"][:, 0], none["initial_state"])[0].shape == (0, 8)
    f = torch.compile(lambda x, d: selective_scan(x, d, v["A"], v["B"], v["C"], v["D"], v["z"], delta_softplus=True), backend="eager", fullgraph=True)
    assert torch.equal(f(v["x"], v["delta"]), selective_scan(v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], delta_softplus=True))


def test_captured_training_step():
    """Forward and backward in one graph, on leaves of its own, replayed with other values."""
    v = inputs(2, 100, 64, 16, torch.bfloat16, seed=14)
    names = [n for n in NAMES if v[n] is not None]
    dy = torch.randn(2, 100, 64, device="cuda").bfloat16()

    def grads(w):
        leaves = {n: w[n].detach().clone().requires_grad_(True) for n in names}
        return torch.autograd.grad(run({**v, **leaves}, state=False), list(leaves.values()), dy)

    static = {n: v[n].clone().requires_grad_(True) for n in names}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(run({**v, **static}, state=False), list(static.values()), dy)
    with torch.no_grad():
        static["x"].mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, grads({**v, "x": v["x"] * 0.5})))


def test_more_than_2_31_elements():
    Bsz, L, dim, N = 1, 33, 1 << 26, 1  # x has 2.2e9 elements
    x = torch.zeros(Bsz, L, dim, device="cuda", dtype=torch.bfloat16)
    x[..., -40:] = torch.randn(L, 40, device="cuda").bfloat16()
    d = torch.full((1, 1, dim), 0.5, device="cuda").bfloat16().expand(Bsz, L, dim)
    A = torch.full((dim, N), -0.5, device="cuda")
    B, C = (torch.randn(Bsz, L, N, device="cuda").bfloat16() for _ in range(2))
    from spear_b200.ops.ssm import selective_scan

    y = selective_scan(x, d, A, B, C)
    small = selective_scan(x[..., -40:].contiguous(), d[..., -40:].contiguous(), A[-40:].clone(), B, C)
    assert torch.equal(y[..., -40:], small) and (y[..., :40] == 0).all()


def test_compiled_training_step():
    v = inputs(2, 70, 40, 16, torch.bfloat16, seed=15)
    names = [n for n in NAMES if v[n] is not None]
    dy = torch.randn(2, 70, 40, device="cuda").bfloat16()
    out = []
    for fn in (run, torch.compile(run, backend="aot_eager")):
        leaves = {n: v[n].clone().requires_grad_(True) for n in names}
        y = fn({**v, **leaves}, state=False)
        out.append([y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy)])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def split_inputs():
    """Few channels and many tokens, so that both directions take the tokens in chunks."""
    from spear_b200.ops import _call

    v = inputs(1, 640, 24, 16, torch.float32, gate=False, bias=False, skip=False, initial=True)
    assert _call.query("btp_sm100_scan_carry_floats", 0, 1, 640, 24, 16) > 0
    whole = 2 * 640 * 16 + 24 * 18  # dB and dC of one block of channels and the parameters' row of one chunk
    assert _call.query("btp_sm100_scan_backward_floats", 0, 1, 640, 24, 16) > whole
    return v


def test_chunks_that_would_make_a_state_grow_beyond_a_float():
    """No state before the last 3 tokens and no gradient behind the first 3: what lies between would multiply either by e^4000."""
    v = split_inputs()
    v["A"] = -v["A"].clamp(-2, -1)
    v["delta"] = torch.full_like(v["delta"], 4.0)
    v["initial_state"].zero_()
    v["x"][:, :-3] = 0
    dy = torch.zeros_like(v["x"])
    dy[:, :3] = torch.randn(1, 3, 24, device="cuda")
    names = [n for n in NAMES if v[n] is not None]
    for n in names:
        v[n].requires_grad_(True)
    y, state = run(v, softplus=False)
    got = dict(zip(names, torch.autograd.grad(y, [v[n] for n in names], dy)))
    want = oracle(v, softplus=False, dy=dy)
    check(y.detach(), want["y"], torch.float32, "y")
    check(state.detach(), want["state"], torch.float32, "state")
    assert torch.isfinite(y).all() and torch.isfinite(state).all()
    for n in names:
        key = "d" + {"initial_state": "initial"}.get(n, n)
        check(got[n], want[key], torch.float32, key)
        assert torch.isfinite(got[n]).all(), key


def test_chunks_that_shrink_a_large_state_below_a_floats_reach():
    """1e30 times e^-102 is 5e-15, though e^-102 by itself is no normal float; the same for the final state's gradient."""
    v = split_inputs()
    v["A"] = -1.6 + 0.02 * torch.rand(24, 16, device="cuda")
    v["x"].zero_(), v["delta"].zero_()
    for at, name in ((5, "state"), (610, "dinitial")):  # 16 tokens inside one chunk of whole 32
        v["delta"].detach().zero_()[:, at:at + 16] = 4.0
        v["initial_state"] = torch.full((1, 24, 16), 1e30 if name == "state" else 0.0, device="cuda", requires_grad=True)
        y, state = run(v, softplus=False)
        if name == "state":
            want = oracle(v, softplus=False)
            check(y.detach(), want["y"], torch.float32, "y")
            check(state.detach(), want["state"], torch.float32, name)
        else:
            ds = torch.full_like(state, 1e30)
            got, = torch.autograd.grad(state, [v["initial_state"]], ds)
            check(got, oracle(v, softplus=False, dy=torch.zeros_like(y), dstate=ds)[name], torch.float32, name)


@pytest.mark.parametrize("lo,hi", [(-30, -12), (-12, -7), (-7, -2), (-2, 0), (0, 3), (3, 30)])
def test_step_sizes_are_accurate_where_they_are_small(lo, hi):
    """With a rate of -1e30 nothing is remembered, so y is the step size itself and delta's gradient its slope.

    Relative to 64 bits, u = 2^-24: e^-|v| two units of the special-function unit (4u) and a rounding; the polynomial of
    log(1 + w) 1e-7 as evaluated, its product or sum one rounding.  The slope: e^-|v| as before, 1 + w one rounding, its
    reciprocal a unit (2u), two products, and the state's gradient exactly 1."""
    n, u = 40000, 2.0 ** -24
    v = torch.linspace(lo, hi, n, device="cuda").view(1, n, 1).requires_grad_(True)
    one = torch.ones(1, n, 1, device="cuda")
    from spear_b200.ops.ssm import selective_scan

    y = selective_scan(one, v, torch.full((1, 1), -1e30, device="cuda"), one, one, delta_softplus=True)
    slope, = torch.autograd.grad(y, v, one)
    v64 = v.detach().double()
    want = torch.logaddexp(v64, torch.zeros_like(v64))
    assert ((y.detach().double() - want).abs() <= (6 * u + 1e-7) * want).all()
    want = torch.exp(v64 - want)
    assert ((slope.double() - want).abs() <= 10 * u * want).all()


@pytest.mark.parametrize("way", ["prompt", "chunks", "token", "gradient"])
def test_decays_are_not_off_in_one_direction(way):
    """The product of 4096 decays between 0.98 and 0.998.  A factor's own rounding is random: 4e-8 rms for the special-function
    unit's result and 2e-8 for the product, five deviations of their sum are 5 * sqrt(4096) * 5e-8.  On average a factor may be off by
    4e-9 (the unit alone is low by 2e-8, 8e-5 for the product).  The rate to the base 2 is rounded twice: 2u of the exponent."""
    from spear_b200.ops import _call
    from spear_b200.ops.ssm import selective_scan, selective_scan_step

    L, u = 4096, 2.0 ** -24
    B, D = (1, 8) if way == "chunks" else (64, 512)  # enough warps for all tokens in one piece, or few and so in chunks
    assert (_call.query("btp_sm100_scan_carry_floats", 0, B, L, D, 4) > 0) == (way == "chunks")
    g = torch.Generator(device="cuda").manual_seed(1)
    dt = 0.002 + 0.018 * torch.rand(B, L, D, generator=g, device="cuda")
    A = torch.full((D, 4), -1.0, device="cuda")
    z, zn = torch.zeros(B, L, D, device="cuda"), torch.zeros(B, L, 4, device="cuda")
    one = torch.ones(B, D, 4, device="cuda")
    if way in ("prompt", "chunks"):
        got = selective_scan(z, dt, A, zn, zn, initial_state=one, return_state=True)[1]
    elif way == "token":
        got = one.clone()
        for t in range(L):
            selective_scan_step(z[:, t], dt[:, t], A, zn[:, t], zn[:, t], got, state_out=got)
    else:
        start = one.clone().requires_grad_(True)
        got, = torch.autograd.grad(selective_scan(z, dt, A, zn, zn, initial_state=start, return_state=True)[1], start, one)
    total = dt.double().sum(1)[..., None].expand(B, D, 4)
    rel = got.double() / torch.exp(-total) - 1
    assert (rel.abs() <= 4e-9 * L + 5 * L ** 0.5 * 5e-8 + 2 * u * total).all(), rel.abs().max()
