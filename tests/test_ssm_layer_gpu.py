"""The operators together, as a model uses them: the selective state space layer, residual blocks around it and around Phalanx,
prompts and tokens, training, captured graphs, an 8-bit projection.

Where two runs differ only in the shape of their matrix products (a prompt against its tokens) the comparison allows 1e-4 of
the norm in float32: four products of at most 256 terms are off by at most 256 * 2^-24 = 1.5e-5 each relative to their terms'
magnitudes, and the convolution and the scan between them by a few 2^-24 per token that they remember.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def close(a, b, tol=1e-4):
    return (a.double() - b.double()).norm() <= tol * b.double().norm()


def layer(dim=64, dtype=torch.float32, **kw):
    from spear_b200.nn.ssm import SelectiveSSM

    torch.manual_seed(0)
    return SelectiveSSM(dim=dim, dtype=dtype, **kw).cuda()


def reference(m, u, lengths=None):
    """The layer in 64 bits, token by token; differentiable."""
    p = {n: t.double() for n, t in m.named_parameters()}
    x, z = (u @ p["in_proj.weight"].t()).split(m.inner, -1)
    B, L, _ = u.shape
    xx = torch.cat([x.new_zeros(B, m.width - 1, m.inner), x], 1)
    pre = p["conv_bias"] + sum(p["conv_weight"][:, k] * xx[:, k:k + L] for k in range(m.width))
    x = torch.nn.functional.silu(pre)
    low, Bt, Ct = (x @ p["x_proj.weight"].t()).split([m.rank, m.state_size, m.state_size], -1)
    dt = torch.nn.functional.softplus(low @ p["dt_proj.weight"].t() + p["dt_bias"])
    A = -torch.exp(p["A_log"])
    h = x.new_zeros(B, m.inner, m.state_size)
    ys = []
    for t in range(L):
        h = torch.exp(dt[:, t, :, None] * A) * h + (dt[:, t] * x[:, t])[..., None] * Bt[:, t, None]
        ys.append((h * Ct[:, t, None]).sum(-1) + p["D"] * x[:, t])
    return (torch.stack(ys, 1) * torch.nn.functional.silu(z)) @ p["out_proj.weight"].t(), h


@pytest.mark.parametrize("kw", [dict(), dict(state_size=8, width=2), dict(state_size=33, width=3, expand=1, rank=7)], ids=str)
def test_layer_against_64_bits(kw):
    m = layer(**kw)
    u = torch.randn(2, 75, 64, device="cuda", requires_grad=True)
    up = torch.randn(2, 75, 64, device="cuda")
    y = m(u)
    names = [n for n, _ in m.named_parameters()]
    grads = torch.autograd.grad(y, [u, *m.parameters()], up)
    u64 = u.detach().double().requires_grad_(True)
    want, _ = reference(m, u64)
    wg = torch.autograd.grad(want, [u64, *m.parameters()], up.double())
    assert close(y, want)
    for n, a, b in zip(["u", *names], grads, wg):
        assert a.dtype == (u if n == "u" else m.get_parameter(n)).dtype and close(a, b, 5e-4), n  # twice the products, there and back


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_then_tokens(dtype):
    m = layer(dtype=dtype, state_size=16)
    u = torch.randn(3, 40, 64, device="cuda").to(dtype)
    # in bfloat16 a product rounds differently by its shape here and there: one step, 2^-8, of a few values on the way
    tol = 1e-4 if dtype == torch.float32 else 3 * 2.0 ** -8
    whole, last = m.prefill(u)
    assert close(m(u), whole, tol)
    out, state = m.prefill(u[:, :25])
    assert close(out, whole[:, :25], tol)
    fixed = state.clone_detached()
    for t in range(25, 40):
        y, new = m.step(u[:, t], state)
        y2, same = m.step(u[:, t], fixed, in_place=True)
        assert same is fixed and torch.equal(y, y2) and torch.equal(fixed.ssm, new.ssm) and torch.equal(fixed.conv, new.conv)
        assert close(y, whole[:, t], tol)
        state = new
    assert close(state.ssm, last.ssm, tol) and close(state.conv, last.conv, tol)
    out2, state2 = m.prefill(u[:, 25:], m.prefill(u[:, :25])[1])
    assert close(out2, whole[:, 25:], tol) and close(state2.ssm, last.ssm, tol)
    y, s = m.step(u[:, 0], m.empty_state(3))
    assert close(y, whole[:, 0], tol)


def test_padded_batch():
    m = layer()
    u = torch.randn(4, 50, 64, device="cuda")
    n = torch.tensor([50, 0, 1, 23], device="cuda", dtype=torch.int32)
    out, state = m.prefill(u, lengths=n)
    dirty = u.clone()
    for b in range(4):
        dirty[b, n[b]:] = 1e9
    out2, state2 = m.prefill(dirty, lengths=n)
    for b, k in enumerate(n.tolist()):
        assert torch.equal(out[b, :k], out2[b, :k]) and (out[b, k:] == 0).all() and torch.equal(state.ssm[b], state2.ssm[b])
        if k:
            alone, s = m.prefill(u[b:b + 1, :k])
            assert close(out[b, :k], alone[0]) and close(state.ssm[b], s.ssm[0])
        else:
            assert (state.ssm[b] == 0).all() and (state.conv[b] == 0).all()


@pytest.mark.parametrize("residual_dtype", [torch.float32, None])
def test_blocks_of_both_mixers_train(residual_dtype):
    """norm -> Phalanx -> norm -> selective scan, a residual stream through both, against the same steps one by one."""
    from spear_b200.nn.block import MixerBlock
    from spear_b200.nn.phalanx import Phalanx
    from spear_b200.ops.norm import rms_norm

    torch.manual_seed(2)
    bf = torch.bfloat16
    blocks = torch.nn.ModuleList([MixerBlock(Phalanx(dim=128, length=64, dtype=bf), 128, dtype=bf, residual_dtype=residual_dtype),
                                  MixerBlock(layer(128, bf), 128, dtype=bf, residual_dtype=residual_dtype)]).cuda()
    x = torch.randn(2, 64, 128, device="cuda").to(bf).requires_grad_(True)

    def run():
        out, h = x, None
        for b in blocks:
            out, h = b(out, h)
        return out, h

    out, h = run()
    assert h.dtype == (residual_dtype or bf) and out.dtype == bf
    a = blocks[0].mixer(rms_norm(x, blocks[0].norm_weight))
    y, hw = rms_norm(a, blocks[1].norm_weight, x if residual_dtype is None else x.to(residual_dtype))
    assert torch.equal(h, hw) and torch.equal(out, blocks[1].mixer(y))
    loss = (out.float() ** 2).sum() + (h.float() ** 2).sum()
    params = [x, *blocks.parameters()]
    grads = torch.autograd.grad(loss, params)
    assert all(g is not None and torch.isfinite(g).all() and g.shape == p.shape and g.dtype == p.dtype for g, p in zip(grads, params))
    out2, h2 = run()
    again = torch.autograd.grad((out2.float() ** 2).sum() + (h2.float() ** 2).sum(), [blocks[1].norm_weight, blocks[1].mixer.A_log])
    keep = {id(p): g for p, g in zip(params, grads)}
    assert torch.equal(again[0], keep[id(blocks[1].norm_weight)]) and torch.equal(again[1], keep[id(blocks[1].mixer.A_log)])


def test_serving_loop_in_a_graph():
    """Prompts of different lengths, then tokens with states updated in place inside one captured graph."""
    from spear_b200.nn.block import MixerBlock

    bf = torch.bfloat16
    blocks = [MixerBlock(layer(64, bf), 64, dtype=bf).cuda() for _ in range(2)]
    u = torch.randn(3, 20, 64, device="cuda").to(bf)
    n = torch.tensor([20, 7, 13], device="cuda", dtype=torch.int32)
    toks = torch.randn(5, 3, 64, device="cuda").to(bf)

    def prompt():
        out, h, states = u, None, []
        for b in blocks:
            out, h, s = b.prefill(out, h, lengths=n)
            states.append(s)
        return states

    def token(t, states, in_place):
        out, h, new = t, None, []
        for b, s in zip(blocks, states):
            out, h, s = b.step(out, h, s, in_place=in_place)
            new.append(s)
        return out + h.to(out.dtype), new

    states, want = prompt(), []
    for t in toks:
        y, states = token(t, states, False)
        want.append(y)
    fixed, tok = prompt(), toks[0].clone()
    start = [s.clone_detached() for s in fixed]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(tok, fixed, True)  # warm-up
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = token(tok, fixed, True)
    for s, o in zip(fixed, start):
        s.ssm.copy_(o.ssm), s.conv.copy_(o.conv)
    for t, w in zip(toks, want):
        tok.copy_(t)
        graph.replay()
        assert torch.equal(y, w)
    assert all(torch.equal(s.ssm, o.ssm) and torch.equal(s.conv, o.conv) for s, o in zip(fixed, states))


def test_8bit_norm_feeds_a_scaled_product():
    """q and its row scales are the left operand of torch's row-scaled 8-bit product."""
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit

    x, r = (torch.randn(64, 512, device="cuda").bfloat16() for _ in range(2))
    w = torch.rand(512, device="cuda") + 0.5
    q, scale, h = rms_norm_8bit(x, w, r)
    y, h2 = rms_norm(x, w, r)
    assert torch.equal(h, h2)
    weight = torch.randn(256, 512, device="cuda")
    ws = weight.abs().amax(1, keepdim=True) / 448
    qw = (weight / ws).to(torch.float8_e4m3fn)
    got = torch._scaled_mm(q, qw.t(), scale_a=scale[:, None].contiguous(), scale_b=ws.t().contiguous(), out_dtype=torch.bfloat16)
    exact = (q.double() * scale.double()[:, None]) @ (qw.double() * ws.double()).t()
    mags = (q.double() * scale.double()[:, None]).abs() @ (qw.double() * ws.double()).abs().t()
    assert ((got.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 512 * 2.0 ** -13 * mags).all()  # the product's own accumulation
    # against the unquantised product: each factor is off by at most 2^-4 (and by less than a scale's 2^-10 where it is small)
    true = y.double() @ weight.double().t()
    off = y.double().abs() @ weight.double().abs().t() * (2 * 2.0 ** -4 + 2.0 ** -8) + 512 * 2.0 ** -10 * scale.double()[:, None] * ws.double().t() * 900
    assert ((exact - true).abs() <= off).all()


@pytest.mark.parametrize("built,cast", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_a_cast_layer_is_a_layer_of_that_type(built, cast):
    """The same parameters, A, D and the step bias rounded by the cast and used in float32 again: the same bits."""
    a = layer(dtype=built).to(cast)
    b = layer(dtype=cast)
    b.load_state_dict(a.state_dict())
    u = torch.randn(2, 30, 64, device="cuda")
    assert torch.equal(a(u), b(u)) and a(u).dtype == cast
    (ya, sa), (yb, sb) = a.prefill(u), b.prefill(u)
    assert torch.equal(ya, yb) and torch.equal(sa.conv, sb.conv) and torch.equal(sa.ssm, sb.ssm)
    assert torch.equal(a.step(u[:, 0], a.empty_state(2))[0], b.step(u[:, 0], b.empty_state(2))[0])


def test_padding_never_reaches_a_gradient():
    """NaN and infinities behind the sequences' ends: outputs and every gradient as with any other padding."""
    m = layer()
    n = torch.tensor([30, 0, 7], device="cuda", dtype=torch.int32)
    u = torch.randn(3, 30, 64, device="cuda")
    up = torch.randn(3, 30, 64, device="cuda")
    dirty = u.clone()
    dirty[1], dirty[2, 7:20], dirty[2, 20:] = float("nan"), float("inf"), -1e30

    def run(v):
        v = v.detach().requires_grad_(True)
        y = m(v, lengths=n)
        return [y.detach(), *torch.autograd.grad(y, [v, *m.parameters()], up)]

    for a, b in zip(run(u), run(dirty)):
        assert torch.equal(a, b) and torch.isfinite(b).all()
