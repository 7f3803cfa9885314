"""The root-mean-square norm against its definition in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of float32.  A row's sum of squares is added up in runs of at
most 32 values per thread, 5 steps in a warp and at most 16 warps, so it is off by at most 53 u relative, its root by
half of that; with the root's and the products' own roundings xhat is off by less than 40 u.  Storing a value rounds it by
half a step of its type (eps / 2).
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-6


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):  # below the normal numbers a step is constant
    return torch.finfo(t).tiny * torch.finfo(t).eps


def inputs(shape, dtype, residual=None, weight=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = r(*shape).to(dtype)
    res = None if residual is None else (3 * r(*shape)).to(residual)
    w = None if weight is None else (1 + 0.3 * r(shape[-1])).to(weight)
    return x, w, res


def reference(x, w, res):
    h = x.double() if res is None else x.double() + res.double()
    rstd = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = h * rstd * (1.0 if w is None else w.double())
    return h, rstd, y


def check_forward(x, w, res, got, h):
    hw, _, yw = reference(x, w, res)
    bound = (half(x.dtype) + 42 * U) * yw.abs() + tiny(x.dtype)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.double() - yw).abs() <= bound).all()
    if res is not None:
        assert h.dtype == res.dtype
        assert ((h.double() - hw).abs() <= (half(res.dtype) + U) * hw.abs() + tiny(res.dtype)).all()


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 3, 24), (5, 250), (4, 256), (7, 257), (2, 512), (3, 1001), (200, 1024), (5, 4096), (160, 4097),
          (2, 8191), (2, 8192), (3, 10008), (1, 16384), (300, 40)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [None, "same", torch.float32])
def test_forward(shape, dtype, residual):
    from spear_b200.ops.norm import rms_norm

    res = dtype if residual == "same" else residual
    for weight in (None, dtype, torch.float32):
        x, w, r = inputs(shape, dtype, res, weight)
        out = rms_norm(x, w, r)
        check_forward(x, w, r, *((out, None) if r is None else out))


@pytest.mark.parametrize("shape", [(1, 8), (3, 100), (6, 128), (5, 129), (9, 1000), (2, 4096), (300, 2048), (2, 16384), (3, 777)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("residual", [False, True])
def test_8bit(shape, dtype, block, residual):
    from spear_b200.ops.norm import rms_norm_8bit

    x, w, r = inputs(shape, dtype, torch.float32 if residual else None, dtype)
    x[0, :] = 0.0  # a row of zeros has scale 1
    if r is not None:
        r[0, :] = 0.0
    out = rms_norm_8bit(x, w, r, block=block)
    assert len(out) == (3 if residual else 2)
    q, scale = out[:2]
    _, _, yw = reference(x, w, r)
    width = shape[-1] if block is None else block
    tops = torch.stack([p.abs().amax(-1) for p in yw.split(width, -1)], -1)
    want = torch.where(tops > 0, tops / 448.0, torch.ones_like(tops))
    got = scale.unsqueeze(-1) if block is None else scale
    assert got.shape == want.shape
    assert ((got.double() - want).abs() <= 44 * U * want).all()
    spread = got.double().repeat_interleave(width, -1)[..., : shape[-1]]
    back = q.double() * spread
    # half a step of e4m3: 2^-4 relative, or 2^-10 of the scale below its normal numbers; the value and its scale add 90 u
    assert ((back - yw).abs() <= (2.0 ** -4 + 90 * U) * yw.abs() + (2.0 ** -10 + 90 * U) * spread).all()
    if residual:
        check_forward(x, w, r, torch.ops.aten.clone(yw.to(dtype)), out[2])


def gradients(x, w, res, dy, dh, h):
    """The formula in 64 bits, and the sum of magnitudes that its roundings are relative to."""
    _, rstd, _ = reference(x, w, res)
    xhat = h.double() * rstd
    g = dy.double() * (1.0 if w is None else w.double())
    m = (g * xhat).mean(-1, keepdim=True)
    mm = (g * xhat).abs().mean(-1, keepdim=True)
    d = rstd * (g - xhat * m)
    mag = rstd * (g.abs() + xhat.abs() * (m.abs() + mm))
    if dh is not None:
        d = d + dh.double()
        mag = mag + dh.double().abs()
    flat = (dy.double() * xhat).reshape(-1, x.shape[-1])
    return d, mag, flat.sum(0), flat.abs().sum(0)


@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 24), (4, 256), (700, 257), (3, 1001), (1500, 512), (5, 4096), (400, 2048),
                                   (2, 8200), (1, 16384)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [None, "same", torch.float32])
def test_backward(shape, dtype, residual):
    from spear_b200.ops.norm import rms_norm

    res = dtype if residual == "same" else residual
    for weight in (None, dtype, torch.float32):
        x, w, r = inputs(shape, dtype, res, weight, seed=1)
        g = torch.Generator(device="cuda").manual_seed(2)
        dy = torch.randn(*shape, generator=g, device="cuda").to(dtype)
        dh = None if r is None else torch.randn(*shape, generator=g, device="cuda").to(r.dtype)
        leaves = [t.requires_grad_(True) for t in (x, w, r) if t is not None]
        out = rms_norm(x, w, r)
        grads = dict(zip([n for n, t in zip(("x", "w", "r"), (x, w, r)) if t is not None],
                         torch.autograd.grad([out] if r is None else list(out), leaves, [dy] if r is None else [dy, dh])))
        with torch.no_grad():
            # the backward reads h as it was stored: the reference differentiates the unrounded sum, and the half step
            # between the two enters through xhat, once directly and once in the mean
            h64 = x.double() if r is None else x.double() + r.double()
            stored = 0.0 if r is None else half(r.dtype)
            d, mag, dw, dwmag = gradients(x, w, r, dy, dh, h64)
            # 60 u for the row's sum, 40 u for xhat twice, a few for the products
            tol = (2.1 * stored + 160 * U) * mag
            assert ((grads["x"].double() - d).abs() <= tol + half(dtype) * (d.abs() + tol) + tiny(dtype)).all()
            if r is not None:
                assert ((grads["r"].double() - d).abs() <= tol + half(r.dtype) * (d.abs() + tol) + tiny(r.dtype)).all()
            if w is not None:
                rows = x.numel() // shape[-1]
                tolw = (1.1 * stored + (50 + min(rows, 600)) * U) * dwmag  # at most 11 rows per thread, 600 partial sums
                assert grads["w"].dtype == w.dtype
                assert ((grads["w"].double() - dw).abs() <= tolw + half(w.dtype) * (dw.abs() + tolw) + tiny(w.dtype)).all()


def test_gradients_of_differences():
    """Directional derivative of a sum of the outputs against central differences in 64 bits."""
    from spear_b200.ops.norm import rms_norm

    x, w, r = inputs((6, 72), torch.float32, torch.float32, torch.float32, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    dy, dh, *dirs = (torch.randn(6, 72, generator=g, device="cuda") for _ in range(4))
    dirs.insert(1, torch.randn(72, generator=g, device="cuda"))
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    grads = torch.autograd.grad(list(rms_norm(x, w, r)), leaves, [dy, dh])
    got = sum((a.double() * b.double()).sum() for a, b in zip(grads, dirs))

    def f(s):
        a, b, c = (t.detach().double() + s * v.double() for t, v in zip((x, w, r), dirs))
        h = a + c
        return (h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * b * dy.double()).sum() + (h * dh.double()).sum()

    want = (f(1e-5) - f(-1e-5)) / 2e-5
    size = sum((a.double() * b.double()).abs().sum() for a, b in zip(grads, dirs))
    assert abs(got - want) <= (200 * U + 1e-8) * size  # differences: 1e-10 from the third derivative, 1e-11 from rounding


def test_only_some_gradients():
    from spear_b200.ops.norm import rms_norm

    x, w, r = inputs((5, 96), torch.bfloat16, torch.float32, torch.bfloat16, seed=5)
    dy = torch.randn(5, 96, device="cuda").bfloat16()
    full = [t.clone().requires_grad_(True) for t in (x, w, r)]
    y, h = rms_norm(*full)
    y.backward(dy)
    for i in range(3):
        part = [t.clone() for t in (x, w, r)]
        part[i].requires_grad_(True)
        rms_norm(*part)[0].backward(dy)
        assert torch.equal(part[i].grad, full[i].grad)
    rr, xx = r.clone().requires_grad_(True), x.clone().requires_grad_(True)
    rms_norm(xx, w, rr)[1].backward(torch.ones_like(r))  # only the sum is used
    assert torch.equal(rr.grad, torch.ones_like(r)) and torch.equal(xx.grad, torch.ones_like(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_offsets_and_broadcast_rows(dtype):
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit

    big, w, _ = inputs((6, 5, 100), dtype, None, dtype, seed=6)
    views = [big[:, :, 3:91], big[::2, 1:4, :64], big.transpose(0, 1), big[..., ::2], big[:1].expand(4, -1, -1), big[:, 2], big[0, 0]]
    for v in views:
        ww = w[: v.shape[-1]]
        want = rms_norm(v.contiguous().clone(), ww.clone(), v.contiguous().clone())
        got = rms_norm(v, ww, v)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(rms_norm(v, w[1:][: v.shape[-1]] if v.shape[-1] < 100 else w), rms_norm(
            v.contiguous().clone(), w[1:][: v.shape[-1]].clone() if v.shape[-1] < 100 else w))
        q, s = rms_norm_8bit(v, ww)
        q2, s2 = rms_norm_8bit(v.contiguous().clone(), ww)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    x = big[:, :, 3:91].clone().requires_grad_(True)
    xs = big.clone().requires_grad_(True)
    up = torch.randn(88, device="cuda").to(dtype).expand(6, 5, 88)  # a broadcast upstream gradient
    rms_norm(x).backward(up)
    rms_norm(xs[:, :, 3:91]).backward(up)
    assert torch.equal(xs.grad[:, :, 3:91], x.grad)


def test_empty_and_extreme_rows():
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit

    x = torch.empty(0, 3, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = rms_norm(x, w)
    y.sum().backward()
    assert y.shape == x.shape and x.grad.shape == x.shape and torch.equal(w.grad, torch.zeros_like(w))
    assert rms_norm_8bit(x)[0].shape == x.shape
    x = torch.randn(6, 200, device="cuda").bfloat16()
    clean = rms_norm(x)
    q0, s0 = rms_norm_8bit(x)
    bad = x.clone()
    bad[1, 5], bad[3, 199], bad[4] = float("nan"), float("inf"), 0.0
    y = rms_norm(bad)
    q, s = rms_norm_8bit(bad)
    keep = [0, 2, 5]
    assert torch.equal(y[keep], clean[keep]) and torch.equal(q.float()[keep], q0.float()[keep]) and torch.equal(s[keep], s0[keep])
    assert y[1].isnan().all() and y[3, 199].isnan() and (y[3, :199] == 0).all() and (y[4] == 0).all()
    assert q[1].float().isnan().all() and (q[4].float() == 0).all() and s[4] == 1
    big = torch.full((2, 64), 2.0 ** 60, device="cuda")  # squares stay inside float32's range up to 2^63
    assert torch.allclose(rms_norm(big), torch.ones_like(big), rtol=1e-5)


def test_streams_graphs_and_repeatability():
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit

    x, w, r = inputs((300, 1536), torch.bfloat16, torch.float32, torch.bfloat16, seed=7)
    want = rms_norm(x, w, r) + rms_norm_8bit(x, w, r, block=128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rms_norm(x, w, r) + rms_norm_8bit(x, w, r, block=128)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(graph):
        cap = rms_norm(xs, w, r) + rms_norm_8bit(xs, w, r, block=128)
    for scale in (1.0, 2.0):
        xs.copy_(x * scale)
        graph.replay()
        want = rms_norm(x * scale, w, r) + rms_norm_8bit(x * scale, w, r, block=128)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cap, want))

    def train():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
        y, h = rms_norm(*leaves)
        return torch.autograd.grad([y, h], leaves, [torch.ones_like(y), torch.ones_like(h)])

    assert all(torch.equal(a, b) for a, b in zip(train(), train()))


def test_rows_beyond_2_31_elements():
    from spear_b200.ops.norm import rms_norm

    rows = (1 << 31) // 8192 + 3
    x = torch.ones(rows, 8192, device="cuda", dtype=torch.bfloat16)
    x[-1] = 3.0
    x[-1, 0] = 5.0
    y = rms_norm(x)
    check_forward(x[-2:], None, None, y[-2:], None)


def test_compiled():
    from spear_b200.ops.norm import rms_norm

    x, w, r = inputs((9, 320), torch.bfloat16, torch.float32, torch.bfloat16, seed=8)
    f = torch.compile(lambda a, b, c: rms_norm(a, b, c), backend="eager", fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(f(x, w, r), rms_norm(x, w, r)))

    dy, dh = torch.randn_like(x), torch.randn_like(r)
    out = []
    for fn in (rms_norm, torch.compile(rms_norm, backend="aot_eager")):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
        out.append(torch.autograd.grad(list(fn(*leaves)), leaves, [dy, dh]))
    assert all(torch.equal(a, b) for a, b in zip(*out))


# several rows per warp or CTA, with a remainder: a row per warp, per CTA of one, two and four runs of columns per thread
TURNS = [(20001, 40), (20003, 256), (5003, 520), (3001, 2048), (2003, 4104), (701, 8200), (603, 16384)]


@pytest.mark.parametrize("shape", TURNS, ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", ["same", torch.float32])
def test_rows_in_turn(shape, dtype, residual):
    """Every row against 64 bits where a warp or CTA takes many of them: the next row fetched ahead, the slots of the sums in turn,
    the weight's gradient over all of a group's rows."""
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit

    res = dtype if residual == "same" else residual
    x, w, r = inputs(shape, dtype, res, torch.float32, seed=3)
    y, h = rms_norm(x, w, r)
    check_forward(x, w, r, y, h)
    check_forward(x, w, None, rms_norm(x, w), None)
    _, _, yw = reference(x, w, r)
    for block in (None, 128):
        q, scale, h8 = rms_norm_8bit(x, w, r, block=block)
        width = shape[-1] if block is None else block
        tops = torch.stack([p.abs().amax(-1) for p in yw.split(width, -1)], -1) / 448.0
        got = scale.unsqueeze(-1) if block is None else scale
        assert ((got.double() - tops).abs() <= 44 * U * tops).all() and torch.equal(h8, h)
        spread = got.double().repeat_interleave(width, -1)[:, : shape[-1]]
        assert ((q.double() * spread - yw).abs() <= (2.0 ** -4 + 90 * U) * yw.abs() + (2.0 ** -10 + 90 * U) * spread).all()
    g = torch.Generator(device="cuda").manual_seed(4)
    dy = torch.randn(*shape, generator=g, device="cuda").to(dtype)
    dh = torch.randn(*shape, generator=g, device="cuda").to(res)
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    dx, dw, dr = torch.autograd.grad(list(rms_norm(x, w, r)), leaves, [dy, dh])
    with torch.no_grad():
        stored = half(res)
        d, mag, want, size = gradients(x, w, r, dy, dh, x.double() + r.double())
        tol = (2.1 * stored + 160 * U) * mag
        assert ((dx.double() - d).abs() <= tol + half(dtype) * (d.abs() + tol) + tiny(dtype)).all()
        assert ((dr.double() - d).abs() <= tol + half(res) * (d.abs() + tol) + tiny(res)).all()
        # a group adds up its rows one by one (at most 20 here), 32 strands the groups' sums (at most 150 each), then the strands
        assert ((dw.double() - want).abs() <= (1.1 * stored + (50 + 20 + 150 + 32) * U) * size).all()


@pytest.mark.parametrize("block", [None, 128])
def test_8bit_values_are_the_rounded_quotients(block):
    """q is e4m3(y / scale), bit for bit, with y as rms_norm returns it in float32 and the quotient rounded to float32: on values at the
    borders between two e4m3 numbers and up to 3 steps of float32 beside them, where a product with the reciprocal goes astray."""
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit

    f8 = torch.arange(1, 127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 2^-9 ... 448
    borders = (f8[1:] + f8[:-1]) / 2
    dim = 16384
    width = 128 if block else dim
    x = torch.ones(1, dim, device="cuda")  # rstd is one number, and the weight sets y
    for seed in range(20):
        g = torch.Generator(device="cuda").manual_seed(seed)
        top = torch.exp(4 * torch.randn(dim // width, 1, generator=g, device="cuda", dtype=torch.float64))
        pick = borders[torch.randint(0, len(borders), (dim // width, width), generator=g, device="cuda")]
        aside = torch.randint(-3, 4, pick.shape, generator=g, device="cuda").double() * 2.0 ** -23
        sign = torch.randint(0, 2, pick.shape, generator=g, device="cuda").double() * 2 - 1
        target = top / 448 * pick * (1 + aside) * sign
        target[:, 5] = top[:, 0]  # the largest of each scale's columns
        w = target.view(dim).float()
        y = rms_norm(x, w)
        q, scale = rms_norm_8bit(x, w, block=block)
        want = (y.view(-1, width) / scale.view(-1, 1)).to(torch.float8_e4m3fn).view(1, dim)
        assert torch.equal(q.view(torch.uint8), want.view(torch.uint8)), seed


def test_a_float16_stream_beyond_its_range():
    """A float16 sum above 65504 is stored as infinity, which the output does not see and the backward pass does: it reads the sum as
    stored.  Only that row's gradients and that column of the weight's are lost."""
    from spear_b200.ops.norm import rms_norm

    x, w, r = inputs((4, 64), torch.float16, torch.float16, torch.float32)
    x[2, 7] = r[2, 7] = 60000.0
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    y, h = rms_norm(x, w, r)
    assert h[2, 7].isinf() and torch.isfinite(y).all()
    with torch.no_grad():
        check_forward(x[:2], w, r[:2], y[:2], h[:2])
    dx, dw, _ = torch.autograd.grad([y, h], leaves, [torch.ones_like(y), torch.ones_like(h)])
    keep = torch.arange(64, device="cuda") != 7
    assert torch.isfinite(dx[[0, 1, 3]]).all() and torch.isfinite(dw[keep]).all() and not torch.isfinite(dw[7])
