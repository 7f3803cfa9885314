"""Cases of the selective state space operators and of the root-mean-square norm, with their plain forms.

Three operators, each in the directions a program uses it in:

  conv   short causal convolution over tokens, one filter per channel (prompt, training pass, single token)
  scan   selective state space scan (prompt, training pass, single token)
  norm   root-mean-square norm with the residual's addition, in the activations' type (also its training pass) or in
         8 bits with one scale per row or per 128 columns

Activations are token-major, [batch, length, channels], as the projections of a layer leave them.
"""

from __future__ import annotations

import math

import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
BLOCK = 128  # columns that share a scale in the blockwise 8-bit form
EPS = 1e-6

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
_BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}


# ---------------------------------------------------------------------------------------------------- cases
def _conv(name, mode, batch, length, dim, width=4, dtype="bfloat16", silu=True, ragged=False):
    return {"name": name, "op": "conv", "mode": mode, "batch": batch, "length": length, "dim": dim, "width": width,
            "dtype": dtype, "silu": silu, "ragged": ragged}


def _scan(name, mode, batch, length, dim, states=16, dtype="bfloat16", gate=True, ragged=False):
    return {"name": name, "op": "scan", "mode": mode, "batch": batch, "length": length, "dim": dim, "states": states,
            "dtype": dtype, "gate": gate, "ragged": ragged}


def _norm(name, mode, rows, dim, dtype="bfloat16", residual="same"):
    return {"name": name, "op": "norm", "mode": mode, "rows": rows, "dim": dim, "dtype": dtype, "residual": residual}


def listed():
    return [
        # one training pass of the convolution over a batch of full-length samples
        _conv("conv train 8x2048x2048", "train", 8, 2048, 2048),
        # prompts of different lengths in one padded batch, an odd length and a channel count that is no power of two
        _conv("conv prompts 6x1999x1504", "prompt", 6, 1999, 1504, ragged=True),
        # one new token for each of many open requests
        _conv("conv token 256x4096", "step", 256, 1, 4096),
        # one training pass of the scan: the largest case
        _scan("scan train 8x2048x2048", "train", 8, 2048, 2048),
        # a batch of prompts as a server takes them in
        _scan("scan prompts 8x2048x2048", "prompt", 8, 2048, 2048),
        # one long document: few channels' worth of work side by side, a long axis
        _scan("scan document 1x16384x1024", "prompt", 1, 16384, 1024),
        # a padded batch with odd sizes in 32 bits, without the gate
        _scan("scan prompts 5x777x1001 float32", "prompt", 5, 777, 1001, dtype="float32", gate=False, ragged=True),
        # one new token of one request: latency
        _scan("scan token 1x1024", "step", 1, 1, 1024),
        # one new token for each of many open requests: the states' traffic
        _scan("scan token 256x4096", "step", 256, 1, 4096),
        # one training pass of the norm in front of a layer, residual stream in 32 bits
        _norm("norm train 16384x2048", "train", 16384, 2048, residual="float32"),
        # the norm in front of an 8-bit projection for a few new tokens, one scale per row
        _norm("norm 8-bit rows 16x4096", "rows8", 16, 4096),
        # the same for prompts, one scale per 128 columns
        _norm("norm 8-bit blocks 16384x4096", "block8", 16384, 4096),
    ]


def _size(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _dim(rng, low, high):
    """A channel count over the whole range: mostly multiples of 8 or 64, now and then an odd one."""
    d = _size(rng, low, high)
    step = rng.choice([1, 8, 64, 64])
    return max(low, min(high, d // step * step))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "norm":
        mode = rng.choice(["plain", "train", "rows8", "block8"])
        dim = _dim(rng, 64, 8192)
        rows = _size(rng, 1, min(32768, 16384 * 2048 // dim))
        residual = rng.choice(["none", "same", "float32"])
        return {"op": op, "mode": mode, "rows": rows, "dim": dim, "dtype": dtype, "residual": residual}
    mode = rng.choice(["train", "prompt", "step"])
    dim = _dim(rng, 64, 4096)
    states = rng.choice([8, 16, 16, 16, 32, 64])
    most = 8 * 2048 * 2048 * 16 // (2 if dtype == "float32" else 1)
    if mode == "step":
        length, batch = 1, _size(rng, 1, 256)
    else:
        most //= dim * (states if op == "scan" else 16)
        length = _size(rng, 1, min(16384, max(1, most)))
        batch = _size(rng, 1, max(1, min(16, most // length)))
    ragged = mode != "step" and rng.random() < 0.3
    case = {"op": op, "mode": mode, "batch": batch, "length": length, "dim": dim, "dtype": dtype}
    if op == "conv":
        return {**case, "width": rng.choice([2, 3, 4, 4]), "silu": rng.random() < 0.75, "ragged": ragged}
    return {**case, "states": states, "gate": rng.random() < 0.6, "ragged": ragged}


# ---------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lengths(case, g):
    """Tokens per sequence of a padded batch: one full sequence, the others anywhere from none to all."""
    if not case["ragged"]:
        return None
    n = torch.randint(0, case["length"] + 1, (case["batch"],), generator=g, device="cuda", dtype=torch.int32)
    n[0] = case["length"]
    return n


def prepare(case, seed):
    g = _generator(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)

    s = {"case": dict(case)}
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        s["x"] = normal(rows, dim)
        s["weight"] = normal(dim, scale=0.1, shift=1.0)
        s["residual"] = None
        if case["residual"] != "none":  # the residual stream has grown over the layers before
            s["residual"] = normal(rows, dim, dtype=torch.float32 if case["residual"] == "float32" else dt, scale=3.0)
        if case["mode"] == "train":
            s["dy"] = normal(rows, dim)
            s["dh"] = None if s["residual"] is None else normal(rows, dim, dtype=s["residual"].dtype)
        return s
    B, L, D = case["batch"], case["length"], case["dim"]
    step = case["mode"] == "step"
    tokens = (B,) if step else (B, L)
    s["lengths"] = None if step else _lengths(case, g)
    if case["op"] == "conv":
        W = case["width"]
        s["x"] = normal(*tokens, D)
        s["weight"] = normal(D, W, scale=1.0 / math.sqrt(W))
        s["bias"] = normal(D, scale=0.1)
        s["state"] = normal(B, W - 1, D) if step else None
        if case["mode"] == "train":
            s["dy"] = normal(*tokens, D)
        return s
    N = case["states"]
    x = torch.randn(*tokens, D, generator=g, device="cuda")
    s["x"] = (x * torch.sigmoid(x)).to(dt)  # what the convolution's activation leaves
    s["delta"] = normal(*tokens, D, scale=0.5)
    s["B"], s["C"] = normal(*tokens, N), normal(*tokens, N)
    s["z"] = normal(*tokens, D) if case["gate"] else None
    # decay rates 1 ... N with some spread, step sizes spread over 0.001 ... 0.1 by the bias before the softplus
    rates = torch.arange(1, N + 1, device="cuda", dtype=torch.float32).log() + 0.1 * torch.randn(D, N, generator=g, device="cuda")
    s["A"] = -torch.exp(rates)
    size = torch.exp(torch.empty(D, device="cuda").uniform_(math.log(1e-3), math.log(1e-1), generator=g))
    s["bias"] = size + torch.log(-torch.expm1(-size))
    s["D"] = 1.0 + 0.1 * torch.randn(D, generator=g, device="cuda")
    s["state"] = torch.randn(B, D, N, generator=g, device="cuda") if step else None
    if case["mode"] == "train":
        s["dy"] = normal(*tokens, D)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _valid(lengths, L):
    """[B, L, 1] truth values: the tokens of each sequence that are there."""
    return (torch.arange(L, device="cuda")[None, :] < lengths[:, None])[..., None]


def _plain_conv_inputs(s):
    """Inputs in 32 bits: [B, W-1+L, D] with the zeros (or the state) in front, and each output's window [B, L, D, W]."""
    W = s["case"]["width"]
    x = s["x"].float()
    if s["lengths"] is not None:
        x = torch.where(_valid(s["lengths"], x.shape[1]), x, 0.0)
    xx = torch.cat([torch.zeros_like(x[:, :1]).expand(-1, W - 1, -1), x], dim=1)
    return xx, xx.unfold(1, W, 1)


def _plain_conv_state(s, xx):
    """The W-1 inputs before each sequence's end."""
    W, L = s["case"]["width"], s["x"].shape[1]
    end = torch.full((xx.shape[0],), L, device="cuda") if s["lengths"] is None else s["lengths"].long()
    at = end[:, None] + torch.arange(W - 1, device="cuda")[None, :]
    return torch.gather(xx, 1, at[..., None].expand(-1, -1, xx.shape[2])).to(s["x"].dtype)


def _plain_conv(s):
    case, dt = s["case"], s["x"].dtype
    weight, bias = s["weight"].float(), s["bias"].float()
    if case["mode"] == "step":
        window = torch.cat([s["state"], s["x"][:, None]], dim=1)
        pre = (window.float() * weight.t()).sum(1) + bias
        y = pre * torch.sigmoid(pre) if case["silu"] else pre
        return {"y": y.to(dt), "state": window[:, 1:].contiguous()}
    xx, windows = _plain_conv_inputs(s)
    pre = (windows * weight).sum(-1) + bias
    sig = torch.sigmoid(pre)
    y = pre * sig if case["silu"] else pre
    if s["lengths"] is not None:
        y = torch.where(_valid(s["lengths"], y.shape[1]), y, 0.0)
    out = {"y": y.to(dt)}
    if case["mode"] == "prompt":
        out["state"] = _plain_conv_state(s, xx)
        return out
    e = s["dy"].float()
    if case["silu"]:
        e = e * sig * (1.0 + pre * (1.0 - sig))
    if s["lengths"] is not None:
        e = torch.where(_valid(s["lengths"], e.shape[1]), e, 0.0)
    W = case["width"]
    ahead = torch.cat([e, torch.zeros_like(e[:, :1]).expand(-1, W - 1, -1)], dim=1).unfold(1, W, 1)
    dx = (ahead * weight.flip(1)).sum(-1)
    if s["lengths"] is not None:
        dx = torch.where(_valid(s["lengths"], e.shape[1]), dx, 0.0)
    out["dx"] = dx.to(dt)
    out["dweight"] = (windows * e[..., None]).sum((0, 1)).to(s["weight"].dtype)
    out["dbias"] = e.sum((0, 1)).to(s["bias"].dtype)
    return out


def _plain_step_size(s):
    """Softplus of the step size's input; it does not overflow for large ones."""
    v = s["delta"].float() + s["bias"]
    return v, torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))


def _plain_scan(s):
    case, dt = s["case"], s["x"].dtype
    x, Bt, Ct = s["x"].float(), s["B"].float(), s["C"].float()
    v, delta = _plain_step_size(s)
    if case["mode"] == "step":
        h = torch.exp(delta[..., None] * s["A"]) * s["state"] + (delta * x)[..., None] * Bt[:, None, :]
        y = (h * Ct[:, None, :]).sum(-1) + s["D"] * x
        if s["z"] is not None:
            z = s["z"].float()
            y = y * z * torch.sigmoid(z)
        return {"y": y.to(dt), "state": h}
    Bsz, L, D = x.shape
    N = s["A"].shape[1]
    valid = None if s["lengths"] is None else _valid(s["lengths"], L)
    if valid is not None:
        delta = torch.where(valid, delta, 0.0)
        x = torch.where(valid, x, 0.0)
    u = delta * x
    a = torch.exp(delta[..., None] * s["A"])
    drive = u[..., None] * Bt[:, :, None, :]
    hs = torch.empty_like(drive)
    h = torch.zeros(Bsz, D, N, device="cuda")
    for t in range(L):  # the recurrence itself
        h = torch.addcmul(drive[:, t], a[:, t], h, out=hs[:, t])
    del drive
    state = h.clone()
    y0 = (hs * Ct[:, :, None, :]).sum(-1) + s["D"] * x
    if s["z"] is not None:
        z = s["z"].float()
        sig = torch.sigmoid(z)
        y = y0 * z * sig
    else:
        y = y0
    if valid is not None:
        y = torch.where(valid, y, 0.0)
    out = {"y": y.to(dt)}
    if case["mode"] == "prompt":
        out["state"] = state
        return out
    dy = s["dy"].float()
    if valid is not None:
        dy = torch.where(valid, dy, 0.0)
    if s["z"] is not None:
        out["dz"] = (dy * y0 * sig * (1.0 + z * (1.0 - sig))).to(dt)
        dy = dy * z * sig
    g = Ct[:, :, None, :] * dy[..., None]
    for t in range(L - 2, -1, -1):
        g[:, t].addcmul_(a[:, t + 1], g[:, t + 1])
    q = g * a
    q[:, 1:] *= hs[:, :-1]
    q[:, 0] = 0.0
    out["dC"] = torch.einsum("bldn,bld->bln", hs, dy)
    out["dB"] = torch.einsum("bldn,bld->bln", g, u)
    du = (g * Bt[:, :, None, :]).sum(-1)
    ddelta = (q * s["A"]).sum(-1) + du * x
    out["dx"] = (du * delta + dy * s["D"]).to(dt)
    out["dA"] = torch.einsum("bldn,bld->dn", q, delta)
    out["dD"] = (dy * x).sum((0, 1))
    draw_ = ddelta * torch.sigmoid(v)
    if valid is not None:
        draw_ = torch.where(valid, draw_, 0.0)
        out["dB"], out["dC"] = torch.where(valid, out["dB"], 0.0), torch.where(valid, out["dC"], 0.0)
    out["ddelta"] = draw_.to(dt)
    out["dbias"] = draw_.sum((0, 1))
    out["dB"], out["dC"] = out["dB"].to(dt), out["dC"].to(dt)
    return out


def _plain_norm(s):
    case, dt = s["case"], s["x"].dtype
    h = s["x"].float()
    out = {}
    if s["residual"] is not None:
        h = h + s["residual"].float()
        out["h"] = h.to(s["residual"].dtype)
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    weight = s["weight"].float()
    xhat = h * r
    y = xhat * weight
    if case["mode"] in ("rows8", "block8"):
        rows, dim = y.shape
        width = dim if case["mode"] == "rows8" else BLOCK
        pad = -dim % width
        blocks = torch.cat([y, y.new_zeros(rows, pad)], dim=1).view(rows, -1, width)
        top = blocks.abs().amax(-1)
        scale = torch.where(top > 0, top / F8_MAX, 1.0)
        q = (blocks / scale[..., None]).view(rows, -1)[:, :dim]
        out["q"] = q.clamp(-F8_MAX, F8_MAX).to(F8)
        out["scale"] = scale[:, 0] if case["mode"] == "rows8" else scale
        return out
    out["y"] = y.to(dt)
    if case["mode"] == "train":
        dy = s["dy"].float()
        wdy = dy * weight
        dh = r * (wdy - xhat * (wdy * xhat).mean(-1, keepdim=True))
        if s["dh"] is not None:
            dh = dh + s["dh"].float()
            out["dresidual"] = dh.to(s["residual"].dtype)
        out["dx"] = dh.to(dt)
        out["dweight"] = (dy * xhat).sum(0).to(s["weight"].dtype)
    return out


# ---------------------------------------------------------------------------------------------------- the framework's operators
def _leaves(s, names):
    """The tensors that get gradients, as leaves of this pass."""
    return {n: s[n].detach().requires_grad_(True) for n in names if s[n] is not None}


def _own_conv(s):
    from spear_b200.ops.ssm import causal_conv, causal_conv_step

    case = s["case"]
    act = "silu" if case["silu"] else None
    if case["mode"] == "step":
        y, state = causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation=act)
        return {"y": y, "state": state}
    if case["mode"] == "prompt":
        y, state = causal_conv(s["x"], s["weight"], s["bias"], activation=act, lengths=s["lengths"], return_state=True)
        return {"y": y, "state": state}
    v = _leaves(s, ("x", "weight", "bias"))
    y = causal_conv(v["x"], v["weight"], v["bias"], activation=act, lengths=s["lengths"])
    dx, dweight, dbias = torch.autograd.grad(y, [v["x"], v["weight"], v["bias"]], s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}


def _own_scan(s):
    from spear_b200.ops.ssm import selective_scan, selective_scan_step

    case = s["case"]
    if case["mode"] == "step":
        y, state = selective_scan_step(s["x"], s["delta"], s["A"], s["B"], s["C"], s["state"], s["D"], s["z"],
                                       delta_bias=s["bias"], delta_softplus=True)
        return {"y": y, "state": state}
    if case["mode"] == "prompt":
        y, state = selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], delta_bias=s["bias"],
                                  delta_softplus=True, lengths=s["lengths"], return_state=True)
        return {"y": y, "state": state}
    v = _leaves(s, ("x", "delta", "A", "B", "C", "D", "z", "bias"))
    y = selective_scan(v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v.get("z"), delta_bias=v["bias"],
                       delta_softplus=True, lengths=s["lengths"])
    grads = torch.autograd.grad(y, list(v.values()), s["dy"])
    return {"y": y.detach(), **{"d" + n: gr for n, gr in zip(v, grads)}}


def _own_norm(s):
    from spear_b200.ops.norm import rms_norm, rms_norm_8bit

    case = s["case"]
    if case["mode"] in ("rows8", "block8"):
        got = rms_norm_8bit(s["x"], s["weight"], s["residual"], eps=EPS, block=BLOCK if case["mode"] == "block8" else None)
        return dict(zip(("q", "scale", "h"), got))
    if case["mode"] == "plain":
        got = rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
        return {"y": got} if s["residual"] is None else {"y": got[0], "h": got[1]}
    v = _leaves(s, ("x", "weight", "residual"))
    got = rms_norm(v["x"], v["weight"], v.get("residual"), eps=EPS)
    if s["residual"] is None:
        outs, ups, out = [got], [s["dy"]], {"y": got.detach()}
    else:
        outs, ups, out = list(got), [s["dy"], s["dh"]], {"y": got[0].detach(), "h": got[1].detach()}
    grads = torch.autograd.grad(outs, list(v.values()), ups)
    return {**out, **{"d" + n: gr for n, gr in zip(v, grads)}}


_PLAIN = {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}
_OWN = {"conv": _own_conv, "scan": _own_scan, "norm": _own_norm}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------- least work
def work(case):
    e = _BYTES[case["dtype"]]
    train = case["mode"] == "train"
    if case["op"] == "norm":
        n = case["rows"] * case["dim"]
        r = 0 if case["residual"] == "none" else (4 if case["residual"] == "float32" else e)
        out = e if case["mode"] in ("plain", "train") else 1
        move = n * (e + 2 * r + out) + case["dim"] * e
        if case["mode"] == "rows8":
            move += 4 * case["rows"]
        if case["mode"] == "block8":
            move += 4 * case["rows"] * -(-case["dim"] // BLOCK)
        if train:  # dy and the residual's gradient read, the inputs' gradients written, the weight's gradient
            move += n * (e + r + e + r) + case["dim"] * e
        return {"bytes": move, "flops": n * (14 if train else 5)}
    B, L, D = case["batch"], case["length"], case["dim"]
    n = B * L * D
    if case["op"] == "conv":
        W = case["width"]
        move = 2 * n * e + D * (W + 1) * e
        ops = 2 * W + (4 if case["silu"] else 0)
        if case["mode"] == "step":
            move += 2 * B * (W - 1) * D * e
        if case["mode"] == "prompt":
            move += B * (W - 1) * D * e
        if train:
            move += 2 * n * e + D * (W + 1) * e
            ops = 3 * ops
        return {"bytes": move, "flops": n * ops}
    N = case["states"]
    acts = 3 + (1 if case["gate"] else 0)  # x, delta, y and the gate
    move = n * acts * e + 2 * B * L * N * e + D * (N + 2) * 4
    ops = 7 * N + 12
    if case["mode"] == "step":
        move += 2 * B * D * N * 4
    if case["mode"] == "prompt":
        move += B * D * N * 4
    if train:  # dy read; gradients of x, delta, the gate, B, C, A, D and the bias written
        move += n * acts * e + 2 * B * L * N * e + D * (N + 2) * 4
        ops = ops + 20 * N + 20
    return {"bytes": move, "flops": n * ops}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    return {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[case["op"]](s)


def _exact_conv(s):
    """Tap by tap: each tap is a shifted copy of the inputs; gradients by differentiating that sum."""
    case = s["case"]
    W, train = case["width"], case["mode"] == "train"
    step = case["mode"] == "step"
    x = s["x"][:, None] if step else s["x"]
    B, L, D = x.shape
    if s["lengths"] is not None:
        live = torch.arange(L, device="cuda").expand(B, L) < s["lengths"][:, None]
        x = x * live[..., None]
    with torch.enable_grad():
        leaves = [t.detach().requires_grad_(train) for t in (x, s["weight"], s["bias"])]
        xs, weight, bias = leaves
        front = s["state"] if step else x.new_zeros(B, W - 1, D)
        xx = torch.cat([front, xs], dim=1)
        y = bias.expand(B, L, D)
        for k in range(W):
            y = y + weight[:, k] * xx[:, k:k + L]
        if case["silu"]:
            y = y / (1.0 + torch.exp(-y))
        if s["lengths"] is not None:
            y = y * live[..., None]
        grads = torch.autograd.grad(y, leaves, s["dy"]) if train else ()
    out = {"y": y.detach()[:, 0] if step else y.detach()}
    if train:
        if s["lengths"] is not None:
            grads = (grads[0] * live[..., None],) + grads[1:]
        return {**out, **dict(zip(("dx", "dweight", "dbias"), grads))}
    ends = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    out["state"] = torch.stack([xx[b, n:n + W - 1] for b, n in enumerate(ends)]).detach()
    return out


def _doubling(a, b):
    """All prefixes of h = a h + b along the first axis, by doubling the stretch that each entry covers."""
    a, b = a.clone(), b.clone()
    k = 1
    while k < a.shape[0]:
        b[k:] = b[k:] + a[k:] * b[:-k]
        a[k:] = a[k:] * a[:-k]
        k *= 2
    return b


def _exact_scan(s):
    """Sequence by sequence, each only as long as it is, every recurrence by doubling."""
    case = s["case"]
    A, skip = s["A"], s["D"]
    D, N = A.shape
    v = s["delta"] + s["bias"]
    delta = torch.logaddexp(v, torch.zeros_like(v))
    if case["mode"] == "step":
        h = torch.exp(delta[:, :, None] * A) * s["state"] + (delta * s["x"])[:, :, None] * s["B"][:, None]
        y = torch.einsum("bdn,bn->bd", h, s["C"]) + s["x"] * skip
        if s["z"] is not None:
            y = y * s["z"] / (1.0 + torch.exp(-s["z"]))
        return {"y": y, "state": h}
    Bsz, L, _ = s["x"].shape
    train = case["mode"] == "train"
    names = ["y"] + (["dx", "ddelta", "dB", "dC"] + (["dz"] if s["z"] is not None else []) if train else [])
    out = {n: torch.zeros(Bsz, L, N if n in ("dB", "dC") else D, device="cuda", dtype=torch.float64) for n in names}
    if train:
        out.update(dA=torch.zeros_like(A), dD=torch.zeros_like(skip), dbias=torch.zeros_like(skip))
    else:
        out["state"] = torch.zeros(Bsz, D, N, device="cuda", dtype=torch.float64)
    ends = [L] * Bsz if s["lengths"] is None else s["lengths"].tolist()
    for b, n in enumerate(ends):
        if n == 0:
            continue
        x, dl, Bt, Ct = s["x"][b, :n], delta[b, :n], s["B"][b, :n], s["C"][b, :n]
        a = torch.exp(dl[:, :, None] * A)
        h = _doubling(a, (dl * x)[:, :, None] * Bt[:, None, :])
        y = torch.einsum("ldn,ln->ld", h, Ct) + x * skip
        gate = None if s["z"] is None else s["z"][b, :n] / (1.0 + torch.exp(-s["z"][b, :n]))
        out["y"][b, :n] = y if gate is None else y * gate
        if not train:
            out["state"][b] = h[-1]
            continue
        dy = s["dy"][b, :n]
        if gate is not None:
            sig = 1.0 / (1.0 + torch.exp(-s["z"][b, :n]))
            out["dz"][b, :n] = dy * y * (sig + gate * (1.0 - sig))
            dy = dy * gate
        # adjoint: backwards in time each entry takes the decay of its successor
        back = torch.ones_like(a)
        back[1:] = a.flip(0)[:-1]
        g = _doubling(back, (dy[:, :, None] * Ct[:, None, :]).flip(0)).flip(0)
        before = torch.zeros_like(h)
        before[1:] = h[:-1]
        w = g * a * before
        du = torch.einsum("ldn,ln->ld", g, Bt)
        out["dx"][b, :n] = du * dl + dy * skip
        dd = (torch.einsum("ldn,dn->ld", w, A) + du * x) / (1.0 + torch.exp(-v[b, :n]))
        out["ddelta"][b, :n] = dd
        out["dB"][b, :n] = torch.einsum("ldn,ld->ln", g, dl * x)
        out["dC"][b, :n] = torch.einsum("ldn,ld->ln", h, dy)
        out["dA"] += torch.einsum("ldn,ld->dn", w, dl)
        out["dD"] += (dy * x).sum(0)
        out["dbias"] += dd.sum(0)
        del a, h, back, g, before, w
    return out


def _exact_norm(s):
    case = s["case"]
    train = case["mode"] == "train"
    with torch.enable_grad():
        leaves = {n: s[n].detach().requires_grad_(train) for n in ("x", "weight", "residual") if s[n] is not None}
        h = leaves["x"] if s["residual"] is None else leaves["x"] + leaves["residual"]
        y = leaves["weight"] * h / torch.sqrt(h.square().sum(-1, keepdim=True) / h.shape[-1] + EPS)
        if train:
            ups = [s["dy"]] + ([] if s["dh"] is None else [s["dh"]])
            grads = torch.autograd.grad([y] + ([] if s["dh"] is None else [h]), list(leaves.values()), ups)
    out = {} if s["residual"] is None else {"h": h.detach()}
    y = y.detach()
    if case["mode"] in ("rows8", "block8"):
        width = case["dim"] if case["mode"] == "rows8" else BLOCK
        parts = y.split(width, dim=1)
        scales = [p.abs().max(dim=1).values / F8_MAX for p in parts]
        scales = [torch.where(c == 0, torch.ones_like(c), c) for c in scales]
        out["q"] = torch.cat([(p / c[:, None]).clamp(-F8_MAX, F8_MAX) for p, c in zip(parts, scales)], dim=1).float().to(F8).float()
        out["scale"] = scales[0] if case["mode"] == "rows8" else torch.stack(scales, dim=1)
        return out
    out["y"] = y
    if train:
        out.update({"d" + n: g for n, g in zip(leaves, grads)})
    return out
