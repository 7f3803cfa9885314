"""The short causal convolution against its definition in 64 bits.

Tolerances count roundings, u = 2^-24: the sum of W + 1 terms is off by at most (W + 1) u of the sum of their magnitudes;
silu's sigmoid is off by (|pre| + 4) 2u relative (the exponent's rounding and two special-function results of 2 units); a
stored value by half a step of its type.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).tiny * torch.finfo(t).eps


def inputs(B, L, D, W, dtype, wdtype=None, *, bias=True, initial=False, lengths=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    wdtype = dtype if wdtype is None else wdtype
    n = None
    if lengths:
        n = torch.randint(0, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        n[0] = min(L, 1)
        n[-1] = 0 if B > 1 else n[-1]
    return {"x": r(B, L, D).to(dtype), "weight": (r(D, W) / W ** 0.5).to(wdtype), "bias": r(D).to(wdtype) if bias else None,
            "initial_state": r(B, W - 1, D).to(dtype) if initial else None, "lengths": n}


def reference(v, silu):
    """y, state, the pre-activation and the sum of its terms' magnitudes, all in 64 bits; differentiable."""
    x, w = v["x"], v["weight"]
    B, L, D = x.shape
    W = w.shape[1]
    live = torch.ones(B, L, 1, device="cuda", dtype=torch.bool)
    if v["lengths"] is not None:
        live = (torch.arange(L, device="cuda")[None] < v["lengths"][:, None])[..., None]
    front = x.new_zeros(B, W - 1, D) if v["initial_state"] is None else v["initial_state"]
    xx = torch.cat([front, torch.where(live, x, torch.zeros_like(x))], 1)
    b = x.new_zeros(D) if v["bias"] is None else v["bias"]
    pre = b + sum(w[:, k] * xx[:, k:k + L] for k in range(W))
    mag = b.abs() + sum(w[:, k].abs() * xx[:, k:k + L].abs() for k in range(W))
    y = pre * torch.sigmoid(pre) if silu else pre
    y = torch.where(live, y, torch.zeros_like(y))
    ends = [L] * B if v["lengths"] is None else v["lengths"].clamp(0, L).tolist()
    state = torch.stack([xx[i, n:n + W - 1] for i, n in enumerate(ends)])
    return y, state, pre, torch.where(live, mag, torch.zeros_like(mag))


def as64(v):
    return {k: t.detach().double() if t is not None and t.is_floating_point() else t for k, t in v.items()}


def y_bound(y, pre, mag, W, silu, dtype):
    err = (W + 2) * U * mag * (1.1 if silu else 1.0)  # silu's slope is at most 1.1
    if silu:
        err = err + y.abs() * (pre.abs() + 4) * 2 * U
    return err + half(dtype) * (y.abs() + err) + tiny(dtype)


SHAPES = [(1, 1, 1), (1, 1, 8), (2, 2, 16), (3, 3, 24), (1, 5, 7), (2, 64, 40), (3, 65, 33), (1, 130, 264), (5, 31, 1001), (2, 333, 512),
          (1, 2048, 64), (4, 1000, 96)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("W", [2, 3, 4])
def test_forward(shape, dtype, W):
    from spear_b200.ops.ssm import causal_conv

    for i, (silu, bias, initial, lengths, wd) in enumerate([(True, True, False, False, dtype), (False, False, True, False, torch.float32),
                                                            (True, True, True, True, torch.float32), (False, True, False, True, dtype)]):
        v = inputs(*shape, W, dtype, wd, bias=bias, initial=initial, lengths=lengths, seed=i)
        y, state = causal_conv(v["x"], v["weight"], v["bias"], activation="silu" if silu else None, initial_state=v["initial_state"],
                               lengths=v["lengths"], return_state=True)
        yw, sw, pre, mag = reference(as64(v), silu)
        assert y.dtype == dtype and ((y.double() - yw).abs() <= y_bound(yw, pre, mag, W, silu, dtype)).all()
        assert state.dtype == dtype and torch.equal(state.double(), sw)  # a copy: no rounding


@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 2, 8), (3, 3, 24), (1, 5, 7), (2, 64, 40), (3, 65, 33), (3, 700, 264), (2, 333, 130),
                                   (1, 1500, 64)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("W", [2, 3, 4])
def test_backward(shape, dtype, W):
    from spear_b200.ops.ssm import causal_conv

    B, L, D = shape
    for i, (silu, bias, initial, lengths, wd) in enumerate([(True, True, False, False, dtype), (False, False, True, False, torch.float32),
                                                            (True, True, True, True, torch.float32), (False, True, True, True, dtype)]):
        v = inputs(B, L, D, W, dtype, wd, bias=bias, initial=initial, lengths=lengths, seed=10 + i)
        g = torch.Generator(device="cuda").manual_seed(99)
        dy = torch.randn(B, L, D, generator=g, device="cuda").to(dtype)
        ds = torch.randn(B, W - 1, D, generator=g, device="cuda").to(dtype)
        names = [n for n in ("x", "weight", "bias", "initial_state") if v[n] is not None]
        for n in names:
            v[n].requires_grad_(True)
        out = causal_conv(v["x"], v["weight"], v["bias"], activation="silu" if silu else None, initial_state=v["initial_state"],
                          lengths=v["lengths"], return_state=True)
        got = dict(zip(names, torch.autograd.grad(out, [v[n] for n in names], [dy, ds])))
        v64 = as64(v)
        for n in names:
            v64[n].requires_grad_(True)
        yw, sw, pre, mag = reference(v64, silu)
        want = dict(zip(names, torch.autograd.grad([yw, sw], [v64[n] for n in names], [dy.double(), ds.double()])))
        with torch.no_grad():
            # e = dy * slope; the slope is at most 1.1 and changes by at most 0.5 per unit of pre
            live = mag > 0 if v["lengths"] is None else (torch.arange(L, device="cuda")[None] < v["lengths"][:, None])[..., None].expand_as(mag)
            e_abs = dy.double().abs() * live * (1.1 if silu else 1.0)
            e_err = dy.double().abs() * live * ((0.5 * (W + 2) * U * mag + (pre.abs() + 6) * 4 * U * (1 + pre.abs())) if silu else U)
            w = v64["weight"].detach().abs()
            pad = lambda t: torch.cat([t, t.new_zeros(B, W - 1, D)], 1)  # noqa: E731
            tail = lambda t: sum(w[:, k] * pad(t)[:, W - 1 - k:W - 1 - k + L] for k in range(W))  # noqa: E731
            tol = tail(e_err) + (W + 3) * U * (tail(e_abs) + ds.double().abs().amax())
            d = (got["x"].double() - want["x"]).abs()
            assert (d <= tol + half(dtype) * (want["x"].abs() + tol) + tiny(dtype)).all()
            if v["lengths"] is not None:
                for b, n in enumerate(v["lengths"].tolist()):
                    assert (got["x"][b, n:] == 0).all()
            if "initial_state" in got:
                top = (e_err.amax(1, keepdim=True) + (W + 3) * U * e_abs.amax(1, keepdim=True)) * w.sum(1) + W * U * ds.double().abs()
                d = (got["initial_state"].double() - want["initial_state"]).abs()
                assert (d <= top + half(dtype) * (want["initial_state"].abs() + top) + tiny(dtype)).all()
            # sums over B L tokens: at most 64 per thread, 8 runs, then the partial sums in 8 strands
            n_add = 64 + 8 + 8 + B * (L // 64 + 1)
            front = x0 = v64["x"].detach().abs() * live
            xx = torch.cat([torch.zeros(B, W - 1, D, device="cuda", dtype=torch.float64) if v["initial_state"] is None else
                            v64["initial_state"].detach().abs(), front], 1)
            for k in range(W):
                tolw = ((e_err + n_add * U * e_abs) * xx[:, k:k + L]).sum((0, 1))
                d = (got["weight"][:, k].double() - want["weight"][:, k]).abs()
                assert (d <= tolw + half(wd) * (want["weight"][:, k].abs() + tolw) + tiny(wd)).all()
            if "bias" in got:
                tolb = (e_err + n_add * U * e_abs).sum((0, 1))
                assert ((got["bias"].double() - want["bias"]).abs() <= tolb + half(wd) * (want["bias"].abs() + tolb) + tiny(wd)).all()
            del x0


def test_gradients_of_differences():
    from spear_b200.ops.ssm import causal_conv

    v = inputs(2, 19, 12, 4, torch.float32, initial=True, lengths=True, seed=3)
    names = ["x", "weight", "bias", "initial_state"]
    g = torch.Generator(device="cuda").manual_seed(5)
    dy = torch.randn(2, 19, 12, generator=g, device="cuda")
    dirs = {n: torch.randn(v[n].shape, generator=g, device="cuda") for n in names}
    for n in names:
        v[n].requires_grad_(True)
    y = causal_conv(v["x"], v["weight"], v["bias"], activation="silu", initial_state=v["initial_state"], lengths=v["lengths"])
    grads = dict(zip(names, torch.autograd.grad(y, [v[n] for n in names], dy)))
    got = sum((grads[n].double() * dirs[n].double()).sum() for n in names)
    size = sum((grads[n].double() * dirs[n].double()).abs().sum() for n in names)

    def f(s):
        w = as64(v)
        for n in names:
            w[n] = w[n] + s * dirs[n].double()
        return (reference(w, True)[0] * dy.double()).sum()

    want = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(got - want) <= (100 * U + 1e-8) * size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,D", [(1, 8), (3, 33), (64, 520)])
@pytest.mark.parametrize("W", [2, 3, 4])
def test_steps_continue_a_prompt(dtype, B, D, W):
    """A prompt, then single tokens, gives bit for bit what the whole sequence gives: the same sums in the same order."""
    from spear_b200.ops.ssm import causal_conv, causal_conv_step

    v = inputs(B, 12, D, W, dtype, seed=4)
    args = (v["weight"], v["bias"])
    whole, last = causal_conv(v["x"], *args, activation="silu", return_state=True)
    y, state = causal_conv(v["x"][:, :5], *args, activation="silu", return_state=True)
    assert torch.equal(y, whole[:, :5])
    inplace = state.clone()
    for t in range(5, 12):
        before = state.clone()
        y_t, new = causal_conv_step(v["x"][:, t], state, *args, activation="silu")
        assert torch.equal(state, before)
        y_i, same = causal_conv_step(v["x"][:, t], inplace, *args, activation="silu", state_out=inplace)
        assert same is inplace and torch.equal(inplace, new) and torch.equal(y_i, y_t)
        assert torch.equal(y_t, whole[:, t])
        state = new
    assert torch.equal(state, last)
    y, state = causal_conv(v["x"][:, :5], *args, return_state=True)
    y2, state2 = causal_conv(v["x"][:, 5:], *args, initial_state=state, return_state=True)
    assert torch.equal(torch.cat([y, y2], 1), causal_conv(v["x"], *args)) and torch.equal(state2, last)


def test_what_lies_behind_the_end_does_not_matter():
    from spear_b200.ops.ssm import causal_conv

    v = inputs(4, 70, 24, 4, torch.bfloat16, initial=True, seed=6)
    n = torch.tensor([0, 1, 33, 70], device="cuda", dtype=torch.int32)
    v["x"].requires_grad_(True)
    dy = torch.randn_like(v["x"])
    args = dict(activation="silu", initial_state=v["initial_state"], lengths=n, return_state=True)
    y, s = causal_conv(v["x"], v["weight"], v["bias"], **args)
    (g,) = torch.autograd.grad(y, v["x"], dy)
    dirty = v["x"].detach().clone()
    dyd = dy.clone()
    for b in range(4):
        dirty[b, n[b]:] = float("nan") if b % 2 else float("inf")
        dyd[b, n[b]:] = float("nan")
    dirty.requires_grad_(True)
    y2, s2 = causal_conv(dirty, v["weight"], v["bias"], **args)
    (g2,) = torch.autograd.grad(y2, dirty, dyd)
    assert torch.equal(y, y2) and torch.equal(s, s2) and torch.equal(g, g2)
    out_of_range = torch.tensor([-5, 1, 33, 1000], device="cuda", dtype=torch.int32)
    assert torch.equal(causal_conv(v["x"].detach(), v["weight"], v["bias"], **{**args, "lengths": out_of_range})[0], y)
    for b in range(4):  # each sequence alone
        alone, sa = causal_conv(v["x"].detach()[b:b + 1, :n[b]], v["weight"], v["bias"], activation="silu",
                                initial_state=v["initial_state"][b:b + 1], return_state=True)
        assert torch.equal(alone[0], y[b, :n[b]]) and torch.equal(sa[0], s[b])


def test_strides_streams_graphs_and_empty():
    from spear_b200.ops.ssm import causal_conv, causal_conv_step

    v = inputs(3, 40, 64, 4, torch.bfloat16, seed=7)
    wide = torch.randn(3, 40, 200, device="cuda").bfloat16()
    for off, size in ((0, 64), (8, 64), (3, 64), (1, 61)):
        view = wide[:, :, off:off + size]
        w, b = v["weight"][:size], v["bias"][:size]
        want = causal_conv(view.clone(), w, b, activation="silu")
        assert torch.equal(causal_conv(view, w, b, activation="silu"), want)
        t = wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :, off:off + size]
        assert torch.equal(causal_conv(t, w, b, activation="silu"), want)
        a, c = (q.detach().requires_grad_(True) for q in (view, view.clone()))
        up = torch.randn(size, 40, 3, device="cuda").bfloat16().permute(2, 1, 0)
        ga, = torch.autograd.grad(causal_conv(a, w, b, activation="silu"), a, up)
        gc, = torch.autograd.grad(causal_conv(c, w, b, activation="silu"), c, up.contiguous())
        assert torch.equal(ga, gc)
        state = torch.randn(3, 3, size, device="cuda").bfloat16()
        assert torch.equal(causal_conv_step(view[:, 5], state, w, b)[0], causal_conv_step(view[:, 5].clone(), state, w, b)[0])
    assert torch.equal(causal_conv(wide[:, :, ::2][..., :64], v["weight"]), causal_conv(wide[:, :, ::2][..., :64].contiguous(), v["weight"]))
    want, ws = causal_conv(v["x"], v["weight"], v["bias"], return_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = causal_conv(v["x"], v["weight"], v["bias"])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    state, tok = ws.clone(), v["x"][:, 0].clone()
    with torch.cuda.graph(graph):
        y, _ = causal_conv_step(tok, state, v["weight"], v["bias"], state_out=state)
    ref = ws.clone()
    state.copy_(ws)
    for t in range(3):
        tok.copy_(v["x"][:, t])
        graph.replay()
        yw, ref = causal_conv_step(v["x"][:, t], ref, v["weight"], v["bias"])
        assert torch.equal(y, yw) and torch.equal(state, ref)
    x0 = torch.empty(2, 0, 64, device="cuda").bfloat16().requires_grad_(True)
    y, s = causal_conv(x0, v["weight"], v["bias"], initial_state=ws[:2], return_state=True)
    y.sum().backward()
    assert y.shape == x0.shape and torch.equal(s, ws[:2])
    assert causal_conv(torch.empty(0, 5, 64, device="cuda").bfloat16(), v["weight"]).shape == (0, 5, 64)
    assert causal_conv_step(torch.empty(0, 64, device="cuda").bfloat16(), torch.empty(0, 3, 64, device="cuda").bfloat16(), v["weight"])[0].shape == (0, 64)


def test_more_than_2_31_elements():
    from spear_b200.ops.ssm import causal_conv

    L, D = 3, (1 << 31) // 4 // 4096 * 4096 // 4
    B = (1 << 31) // (L * D) + 1
    x = torch.zeros(B, L, D, device="cuda", dtype=torch.bfloat16)
    x[-1] = torch.randn(L, D, device="cuda").bfloat16()
    w = torch.randn(D, 2, device="cuda").bfloat16()
    assert x.numel() > 1 << 31
    y = causal_conv(x, w)
    assert torch.equal(y[-1:], causal_conv(x[-1:].clone(), w)) and (y[0] == 0).all()


def test_compiled_and_repeatable():
    from spear_b200.ops.ssm import causal_conv

    v = inputs(3, 50, 40, 4, torch.bfloat16, initial=True, seed=8)
    f = torch.compile(lambda x, w, b: causal_conv(x, w, b, activation="silu"), backend="eager", fullgraph=True)
    assert torch.equal(f(v["x"], v["weight"], v["bias"]), causal_conv(v["x"], v["weight"], v["bias"], activation="silu"))
    runs = []
    for _ in range(2):
        leaves = [v[n].clone().requires_grad_(True) for n in ("x", "weight", "bias")]
        y = causal_conv(*leaves, activation="silu")
        runs.append(torch.autograd.grad(y, leaves, torch.ones_like(y)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    leaves = [v[n].clone().requires_grad_(True) for n in ("x", "weight", "bias")]
    y = torch.compile(causal_conv, backend="aot_eager")(*leaves, activation="silu")
    assert all(torch.equal(a, b) for a, b in zip(runs[0], torch.autograd.grad(y, leaves, torch.ones_like(y))))


# sequences x channels enough for runs of many tiles, so that the ring of three is gone through many times
@pytest.mark.parametrize("shape", [(8, 1500, 2056), (16, 2999, 1024)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("padded", [False, True])
def test_long_runs(shape, dtype, padded):
    from spear_b200.ops.ssm import causal_conv

    B, L, D = shape
    W = 4
    v = inputs(B, L, D, W, dtype, initial=True, lengths=padded, seed=6)
    if padded:
        v["lengths"][1], v["lengths"][2] = L, L - 1
    dy = torch.randn(B, L, D, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda").to(dtype)
    names = ("x", "weight", "bias", "initial_state")
    for n in names:
        v[n].requires_grad_(True)
    y, state = causal_conv(v["x"], v["weight"], v["bias"], activation="silu", initial_state=v["initial_state"], lengths=v["lengths"],
                           return_state=True)
    got = dict(zip(names, torch.autograd.grad(y, [v[n] for n in names], dy)))
    h = half(dtype)
    for b in range(B):  # sequence by sequence: 64 bits of all of them are tens of GB
        one = {k: (t if k in ("weight", "bias") else None if t is None else t[b:b + 1]) for k, t in v.items()}
        w64 = {k: t.requires_grad_(True) if k in names else t for k, t in as64(one).items()}
        yw, sw, pre, mag = reference(w64, True)
        tol = (W + 1) * U * mag * 1.1 + (pre.abs() + 4) * 2 * U * yw.abs()  # silu's slope is at most 1.1
        assert ((y[b:b + 1].double() - yw).abs() <= tol + h * (yw.abs() + tol) + tiny(dtype)).all(), b
        assert torch.equal(state[b:b + 1], sw.to(dtype)), b
        dx, dw, db, di = torch.autograd.grad(yw, [w64[n] for n in names], dy[b:b + 1].double())
        # e = dy act'(pre): act' is off by 2 (|pre| + 4) u twice and by half of the pre-activation's error, its second derivative's bound;
        # a gradient is the sum of W such terms
        off = dy[b:b + 1].double().abs() * (4 * (pre.abs() + 4) * U + 0.5 * (W + 1) * U * mag)
        if v["lengths"] is not None:
            off = off * (torch.arange(L, device="cuda")[None, :, None] < v["lengths"][b])
        w = v["weight"].detach().double().abs()
        ahead = torch.cat([off, off.new_zeros(1, W - 1, D)], 1)
        size = torch.cat([dy[b:b + 1].double().abs() * 1.1, off.new_zeros(1, W - 1, D)], 1)
        tol = sum(w[:, k] * (ahead + (W + 1) * U * size)[:, W - 1 - k:W - 1 - k + L] for k in range(W))
        assert ((got["x"][b:b + 1].double() - dx).abs() <= tol + h * (dx.abs() + tol) + tiny(dtype)).all(), b
        if b == 0:
            sums = [dw.clone(), db.clone()]
        else:
            sums[0] += dw
            sums[1] += db
    # one thread adds up a run, one strand of eight the runs: at most 3000 + 300 roundings, and each term is off as above; the terms'
    # magnitudes are at most those of dy 1.1 times |xx|
    x = v["x"].detach().double().abs()
    live = 1.0 if v["lengths"] is None else (torch.arange(L, device="cuda")[None, :] < v["lengths"][:, None]).double()[..., None]
    weight = dy.double().abs() * live * (1.1 * 3300 * U + 60 * U)
    size_b = weight.sum((0, 1))
    xmax = x.amax((0, 1)).maximum(v["initial_state"].detach().double().abs().amax((0, 1)))
    assert ((got["bias"].double() - sums[1]).abs() <= size_b + h * (sums[1].abs() + size_b)).all()
    tol = (size_b * xmax)[:, None]
    assert ((got["weight"].double() - sums[0]).abs() <= tol + h * (sums[0].abs() + tol)).all()
