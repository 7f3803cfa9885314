"""The selective scan and its gradients in 64 bits, each value with a bound on the error that a float32 computation of the
same formula makes.

A quantity is (v, e): v in 64 bits, e >= |float32 result - v|.  Every operation adds its own rounding, u = 2^-24 relative, to
what it passes on, so the bounds are arithmetic and not a fit.  `u` is taken twice as large as it is, which covers products
of two errors, the special-function unit's two units in the last place and the other order of sums that a split over chunks has.

A value beyond float32's largest number has no float32 result near it (a state that grows with a negative step size can get
there): its bound, and that of what is computed from it, is infinite.  The same holds for what is stored in a type whose largest
number it exceeds.
"""

from __future__ import annotations

import torch

U = 2.0 ** -23


LARGEST = torch.finfo(torch.float32).max


class Q:
    def __init__(self, v, e=None):
        e = torch.zeros_like(v) if e is None else e
        # v.abs() + e beyond the range, or inf * 0 in e: no bound
        self.v, self.e = v, torch.where(v.abs() + e < LARGEST, e, torch.inf)

    def __add__(self, o):
        v = self.v + o.v
        return Q(v, self.e + o.e + U * v.abs())

    def __mul__(self, o):
        v = self.v * o.v
        return Q(v, self.e * o.v.abs() + o.e * self.v.abs() + U * v.abs())

    def sum(self, dim, adds):
        return Q(self.v.sum(dim), self.e.sum(dim) + adds * U * self.v.abs().sum(dim))

    def __getitem__(self, i):
        return Q(self.v[i], self.e[i])

    def exp(self):
        v = self.v.exp()  # argument scaled by log2 e: two roundings of it, then two units of the result
        return Q(v, v * (self.e + 2 * U * self.v.abs() + 2 * U))

    def sigmoid(self):
        v = torch.sigmoid(self.v)
        return Q(v, v * (1 - v) * (self.e + 2 * U * self.v.abs()) + 3 * U * v)

    def softplus(self):
        v = torch.nn.functional.softplus(self.v, threshold=1e9)
        return Q(v, torch.sigmoid(self.v) * (self.e + 2 * U * self.v.abs()) + 6 * U * v)

    def where(self, m):
        return Q(torch.where(m, self.v, 0.0), torch.where(m, self.e, 0.0))

    def to(self, dtype):
        """The bound on a value that is stored in dtype."""
        f = torch.finfo(dtype)
        bound = self.e + f.eps / 2 * (self.v.abs() + self.e) + f.tiny * f.eps
        return torch.where(self.v.abs() + bound < f.max, bound, torch.inf)


def stack(qs, dim):
    return Q(torch.stack([q.v for q in qs], dim), torch.stack([q.e for q in qs], dim))


def scan(x, delta, A, B, C, D=None, z=None, *, delta_bias=None, softplus=False, initial=None, lengths=None, dy=None, dstate=None):
    """{"y", "state"} and, with dy, {"dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "dbias", "dinitial"}, all Q."""
    q = lambda t: None if t is None else Q(t.detach().double())  # noqa: E731
    Bsz, L, dim = x.shape
    N = A.shape[1]
    live = torch.ones(Bsz, L, 1, device=x.device, dtype=torch.bool)
    if lengths is not None:
        live = (torch.arange(L, device=x.device)[None] < lengths[:, None])[..., None]
    keep = lambda t: None if t is None else Q(torch.where(live, t.detach().double(), 0.0))  # noqa: E731
    X, Bq, Cq, Z, Aq = keep(x), keep(B), keep(C), keep(z), q(A)
    raw = keep(delta)
    if delta_bias is not None:
        raw = raw + q(delta_bias)
    dt = (raw.softplus() if softplus else raw).where(live)
    u = dt * X
    h = Q(torch.zeros(Bsz, dim, N, device=x.device, dtype=torch.float64)) if initial is None else q(initial)
    hs, decayed, decays = [], [], []
    for t in range(L):
        a = (dt[:, t, :, None] * Aq).exp()
        a = Q(torch.where(live[:, t, :, None], a.v, 1.0), torch.where(live[:, t, :, None], a.e, 0.0))
        w = a * h
        h = w + u[:, t, :, None] * Bq[:, t, None, :]
        hs.append(h), decayed.append(w), decays.append(a)
    out = {"state": h}
    H = stack(hs, 1)
    y0 = (H * Cq[:, :, None, :]).sum(-1, N)
    if D is not None:
        y0 = y0 + q(D) * X
    gate = None if Z is None else Z * Z.sigmoid()
    out["y"] = (y0 if gate is None else y0 * gate).where(live)
    if dy is None:
        return out
    up = keep(dy)
    e = up if gate is None else up * gate
    if gate is not None:
        s = Z.sigmoid()
        one = Q(torch.ones_like(s.v))
        slope = s * (one + Z * (one + Q(-s.v, s.e)))
        out["dz"] = (up * y0 * slope).where(live)
    G = Q(torch.zeros(Bsz, dim, N, device=x.device, dtype=torch.float64)) if dstate is None else q(dstate)
    gs = [None] * L
    for t in range(L - 1, -1, -1):
        gs[t] = G + Cq[:, t, None, :] * e[:, t, :, None]
        G = gs[t] * decays[t]
    out["dinitial"] = G
    g, w = stack(gs, 1), stack(decayed, 1)
    adds = 64 + L // 16 + 4 * Bsz  # a tile, the tiles of a chunk, the chunks and sequences
    ww = g * w
    du = (g * Bq[:, :, None, :]).sum(-1, N)
    out["dB"] = (g * u[..., None]).sum(2, 12 + dim // 32).where(live)
    out["dC"] = (H * e[..., None]).sum(2, 12 + dim // 32).where(live)
    skip = e * q(D) if D is not None else None
    out["dx"] = (du * dt + skip if skip is not None else du * dt).where(live)
    dd = (ww * Aq).sum(-1, N) + du * X
    if softplus:
        dd = dd * raw.sigmoid()
    out["ddelta"] = dd.where(live)
    two = lambda t: t.sum((0, 1), adds)  # noqa: E731
    out["dA"] = two(ww * dt[..., None])
    out["dD"], out["dbias"] = two(e * X), two(out["ddelta"])
    return out
