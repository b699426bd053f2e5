"""The feed-forward operators in 64 bits, with a bound on what an implementation that
works as documented may be off: fp32 sums (a product of depth k errs by at most 2 k
half steps of its sum of magnitudes, tensor cores may truncate), activations to a few
fp32 steps, and one rounding to 16 bits per stored value."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}       # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}     # half the smallest step
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
SLOPE = 1.13   # no activation is steeper (gelu: 1.129)
EPS = 2.0 ** -24


def act(name, z):
    """(act(z), act'(z)) in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z), (z > 0).to(z.dtype)
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(8 / math.pi)
        p = torch.sigmoid(c * (z + 0.044715 * z ** 3))
        q = torch.sigmoid(-c * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * q * c * (1 + 3 * 0.044715 * z * z)
    p, q = torch.sigmoid(z), torch.sigmoid(-z)
    return (p, p * q) if name == "sigmoid" else (z * p, p + z * p * q)


def act_error(z):
    """Of act and act' in fp32: the exponent's argument, e^x and 1/x, a few steps each, and
    the argument's own rounding, which grows with it."""
    return 64 * EPS * (1 + z.abs())


def product(a, b, ea=None, eb=None):
    """(a b^T, bound) of operands that err by ea, eb."""
    s = a.abs() @ b.abs().t()
    e = 2 * EPS * (a.shape[1] + 8) * s
    if ea is not None:
        e = e + ea @ (b.abs() if eb is None else b.abs() + eb).t()
    if eb is not None:
        e = e + a.abs() @ eb.t()
    return a @ b.t(), e


def rounded(v, e, dtype):
    """(v, bound) once v, which errs by e, was rounded to dtype."""
    return v, e + HALF[dtype] * (v.abs() + e) + TINY[dtype]


def linear(x, w, b=None, r=None, name="none"):
    """[(y, bound), (pre, bound)]"""
    dt = x.dtype
    z, e = product(x.double(), w.double())
    if b is not None:
        z = z + b.double()
        e = e + 2 * EPS * z.abs()
    a, _ = act(name, z)
    ea = SLOPE * e + (act_error(z) if name != "none" else 0)
    y = a
    if r is not None:
        y = a + r.double()
        ea = ea + EPS * y.abs()
    return [rounded(y, ea, dt), rounded(z, e, dt)]


def linear_backward(grad, x, w, pre=None, name="none"):
    """[(dx, bound), (dw, bound), (db, bound)]"""
    dt = x.dtype
    g = grad.double()
    dz, e = g, torch.zeros_like(g)
    if name != "none":
        _, d = act(name, pre.double())
        dz = g * d
        e = g.abs() * act_error(pre.double()) + 2 * EPS * dz.abs()
    db = dz.sum(0), e.sum(0) + 2 * EPS * (len(dz) + 8) * dz.abs().sum(0)
    if name != "none":
        dz, e = rounded(dz, e, dt)
    dx = product(dz, w.double().t(), e)
    dw = product(dz.t(), x.double().t(), e.t())
    return [rounded(*v, dt) for v in (dx, dw, db)]


def gated(x, wg, wu, name="silu"):
    """[(h, bound), (g, bound), (u, bound)]"""
    dt = x.dtype
    g, eg = product(x.double(), wg.double())
    u, eu = product(x.double(), wu.double())
    a, _ = act(name, g)
    ea = SLOPE * eg + act_error(g)
    h = a * u, (a.abs() + ea) * eu + ea * u.abs() + EPS * (a * u).abs()
    return [rounded(*v, dt) for v in (h, (g, eg), (u, eu))]


def gated_backward(dh, edh, x, wg, wu, gate, up, name):
    """([(dx, bound), (dwg, bound), (dwu, bound)], (h, bound)); dh errs by edh."""
    dt = x.dtype
    g, u = gate.double(), up.double()
    a, d = act(name, g)
    ee = act_error(g)
    dg = rounded(dh * u * d, (edh * d.abs() + (dh.abs() + edh) * ee) * u.abs() + 3 * EPS * (dh * u * d).abs(), dt)
    du = rounded(dh * a, edh * a.abs() + (dh.abs() + edh) * ee + EPS * (dh * a).abs(), dt)
    h = rounded(a * u, ee * u.abs() + EPS * (a * u).abs(), dt)
    both = torch.cat([dg[0], du[0]], 1), torch.cat([dg[1], du[1]], 1)
    dx = product(both[0], torch.cat([wg, wu]).double().t(), both[1])
    xt = x.double().t()
    out = [dx, product(dg[0].t(), xt, dg[1].t()), product(du[0].t(), xt, du[1].t())]
    return [rounded(*v, dt) for v in out], h


def ffn(x, wg, wu, wd, r=None, name="silu"):
    dt = x.dtype
    h, eh = gated(x, wg, wu, name)[0]
    y, e = product(h, wd.double(), eh)
    if r is not None:
        y = y + r.double()
        e = e + EPS * y.abs()
    return rounded(y, e, dt)


def ffn_backward(grad, x, wg, wu, wd, gate, up, name="silu"):
    """[(dx), (dwg), (dwu), (dwd)], each with its bound"""
    dh, edh = product(grad.double(), wd.double().t())
    out, h = gated_backward(dh, edh, x, wg, wu, gate, up, name)
    dwd = product(grad.double().t(), h[0].t(), None, h[1].t())
    return out + [rounded(*dwd, x.dtype)]


def check(got, want, what=""):
    """got within the bound of want = (value, bound)."""
    v, e = want
    assert got.shape == v.shape, (what, got.shape, v.shape)
    off = (got.double() - v).abs()
    bad = ~(off <= e)
    if bad.any():
        i = (off / e.clamp(min=1e-300)).nan_to_num(nan=float("inf")).argmax().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {i}: got "
                             f"{got.flatten()[i].item()}, want {v.flatten()[i].item()} +- "
                             f"{e.flatten()[i].item()}")
