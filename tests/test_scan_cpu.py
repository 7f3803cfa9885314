"""Refusals of the selective scan, on a machine without a GPU too."""

from __future__ import annotations

import ctypes

import pytest
import torch

from spear_b200.ops.ssm import selective_scan, selective_scan_step

Z = torch.zeros


def call(fn=selective_scan, **over):
    a = {"x": Z(2, 4, 8), "delta": Z(2, 4, 8), "A": Z(8, 16), "B": Z(2, 4, 16), "C": Z(2, 4, 16)}
    a.update(over)
    return fn(**a)


@pytest.mark.parametrize("over,err,text", [
    ({"x": Z(4, 8)}, ValueError, "x must be"),
    ({"x": Z(2, 4, 0)}, ValueError, "x must be"),
    ({"x": Z(2, 4, 8).double()}, RuntimeError, "x must be bfloat16"),
    ({"delta": Z(2, 4, 9)}, ValueError, "delta must be"),
    ({"delta": Z(2, 4, 8).half()}, RuntimeError, "delta must have"),
    ({"A": Z(8, 65)}, ValueError, "A must be"),
    ({"A": Z(8, 0)}, ValueError, "A must be"),
    ({"A": Z(7, 16)}, ValueError, "A must be"),
    ({"A": Z(8, 16).bfloat16()}, RuntimeError, "A must be float32"),
    ({"B": Z(2, 4, 15)}, ValueError, "B must be"),
    ({"B": Z(2, 4, 1, 16)}, ValueError, "B must be"),
    ({"C": Z(2, 5, 16)}, ValueError, "C must be"),
    ({"C": Z(2, 4, 16).half()}, RuntimeError, "C must have"),
    ({"D": Z(9)}, ValueError, "D must be"),
    ({"D": Z(8).half()}, RuntimeError, "D must be float32"),
    ({"delta_bias": Z(1)}, ValueError, "delta_bias must be"),
    ({"z": Z(2, 1, 8)}, ValueError, "z must be"),
    ({"initial_state": Z(2, 8, 15)}, ValueError, "initial_state"),
    ({"initial_state": Z(2, 8, 16).bfloat16()}, ValueError, "initial_state"),
    ({"lengths": Z(2)}, ValueError, "lengths"),
    ({"lengths": Z(1, dtype=torch.int32)}, ValueError, "lengths"),
    ({}, RuntimeError, "no CPU path"),
])
def test_refusals(over, err, text):
    with pytest.raises(err, match=text):
        call(**over)


def step(**over):
    a = {"x_t": Z(2, 8), "delta_t": Z(2, 8), "A": Z(8, 16), "B_t": Z(2, 16), "C_t": Z(2, 16), "state": Z(2, 8, 16)}
    a.update(over)
    return selective_scan_step(**a)


@pytest.mark.parametrize("over,err,text", [
    ({"x_t": Z(2, 1, 8)}, ValueError, "x_t must be"),
    ({"delta_t": Z(2, 7)}, ValueError, "delta_t must be"),
    ({"B_t": Z(2, 8)}, ValueError, "B_t must be"),
    ({"C_t": Z(2, 16).half()}, RuntimeError, "C_t must have"),
    ({"z_t": Z(2, 9)}, ValueError, "z_t must be"),
    ({"state": Z(2, 8, 15)}, ValueError, "state must be"),
    ({"state": Z(2, 8, 16).half()}, ValueError, "state must be"),
    ({"state": Z(2, 16, 8).transpose(1, 2)}, ValueError, "state must be contiguous"),
    ({}, RuntimeError, "no CPU path"),
])
def test_step_refusals(over, err, text):
    with pytest.raises(err, match=text):
        step(**over)


def test_entry_refuses_bad_arguments_before_any_launch():
    from spear_b200 import _lib

    lib = _lib.load()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(20)

    def fwd(x=p, d=p, A=p, B=p, C=p, y=p, init=None, sizes=(1, 4, 8, 16), st=8, dt=0):
        return lib.btp_sm100_scan_forward(x, d, A, B, C, None, None, None, init, None, y, None, None, None, *sizes, *([st] * 10), 0, dt, None)

    assert fwd(sizes=(0, 4, 8, 16)) == -2 and fwd(sizes=(1, 0, 8, 16)) == -2 and fwd(sizes=(1, 4, 0, 16)) == -2
    assert fwd(sizes=(1, 4, 8, 0)) == -2 and fwd(sizes=(1, 4, 8, 65)) == -2 and fwd(sizes=(1, (1 << 30) + 1, 8, 16)) == -2
    assert fwd(st=-1) == -2 and fwd(dt=2) == -4
    assert fwd(x=None) == -1 and fwd(A=None) == -1 and fwd(y=None) == -1
    assert fwd(A=odd) == -5 and fwd(init=odd) == -5

    def bwd(ck=p, buf=p, z=None, dz=None):
        return lib.btp_sm100_scan_backward(p, p, p, p, p, None, z, None, None, ck, p, None, p, p, p, p, p, dz, None, buf, 1, 4, 8, 16,
                                           *([8] * 10), 0, 0, None)

    assert bwd(ck=None) == -1 and bwd(buf=None) == -1 and bwd(z=p) == -1 and bwd(buf=odd) == -5
    assert lib.btp_sm100_scan_step(p, p, p, p, p, None, None, None, p, p, odd, 1, 8, 16, 8, 8, 16, 16, 0, 0, 0, None) == -5
    assert lib.btp_sm100_scan_step(p, p, p, p, p, None, None, None, None, p, p, 1, 8, 16, 8, 8, 16, 16, 0, 0, 0, None) == -1


def test_oracle_agrees_with_autograd():
    """The formulas that the GPU tests compare with, against differentiation of the recurrence in 64 bits."""
    import scan_oracle

    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    Bsz, L, dim, N = 2, 7, 3, 4
    v = {"x": r(Bsz, L, dim), "delta": r(Bsz, L, dim), "A": -r(dim, N).exp(), "B": r(Bsz, L, N), "C": r(Bsz, L, N), "D": r(dim),
         "z": r(Bsz, L, dim), "delta_bias": r(dim), "initial": r(Bsz, dim, N)}
    lengths = torch.tensor([7, 4], dtype=torch.int32)
    dy, ds = r(Bsz, L, dim), r(Bsz, dim, N)
    got = scan_oracle.scan(**v, softplus=True, lengths=lengths, dy=dy, dstate=ds)
    w = {k: t.clone().requires_grad_(True) for k, t in v.items()}
    dt = torch.nn.functional.softplus(w["delta"] + w["delta_bias"])
    ys, ends = [], []
    for b, n in enumerate(lengths.tolist()):
        h = w["initial"][b]
        rows = []
        for t in range(n):
            h = torch.exp(dt[b, t, :, None] * w["A"]) * h + (dt[b, t] * w["x"][b, t])[:, None] * w["B"][b, t]
            rows.append(((h * w["C"][b, t]).sum(-1) + w["D"] * w["x"][b, t]) * torch.nn.functional.silu(w["z"][b, t]))
        ys.append(torch.cat([torch.stack(rows), torch.zeros(L - n, dim, dtype=torch.float64)])), ends.append(h)
    grads = torch.autograd.grad([torch.stack(ys), torch.stack(ends)], list(w.values()), [dy, ds])
    assert torch.allclose(got["y"].v, torch.stack(ys)) and torch.allclose(got["state"].v, torch.stack(ends))
    for name, gr in zip(w, grads):
        assert torch.allclose(got["d" + {"delta_bias": "bias"}.get(name, name)].v, gr, atol=1e-12), name


@pytest.mark.parametrize("B,L,D", [(2 ** 32 + 1, 1, 1), (1, 2 ** 32 + 5, 1), (1, 1, 2 ** 32 + 8)])
def test_sizes_beyond_32_bits_are_refused_not_cut_off(B, L, D):
    from spear_b200.ops.ssm import selective_scan, selective_scan_step

    E = lambda *shape: torch.empty(*shape, device="meta")
    with pytest.raises(ValueError, match="below 2\\^31"):
        selective_scan(E(B, L, D), E(B, L, D), E(D, 2), E(B, L, 2), E(B, L, 2))
    if L == 1:
        with pytest.raises(ValueError, match="below 2\\^31"):
            selective_scan_step(E(B, D), E(B, D), E(D, 2), E(B, 2), E(B, 2), E(B, D, 2))
