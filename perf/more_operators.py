"""Cases and plain forms of the feed-forward operators: a linear layer with bias,
activation and residual in the product's epilogue, and a gated feed-forward block
(both projections, the activation and their product in one kernel), each with its
backward pass and its form for few tokens.

`own = False` computes the plain form with elementary torch operations in 32 bits;
`own = True` makes the calls that a user makes of sion_b200. Both take the state that
`prepare` gives.

    linear        y = act(x W^T + b) + r                      x [T, K], W [N, K]
    linear_back   z' = dy * act'(z); dx = z' W, dW = z'^T x, db = sum z'
    gated         h = act(x Wg^T) * (x Wu^T)                  Wg, Wu [F, K]
    gated_back    dg = dh u act'(g), du = dh act(g); dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
    ffn           y = h Wd^T + r                              Wd [K, F]
    ffn_back      dh = dy Wd, then as gated_back, and dWd = dy^T h

z, g, u are the values in front of the activations, which the forward pass has saved in
16 bits.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one conversation answered alone: a projection back into the residual stream
        {"name": "linear_one", "kind": "linear", "tokens": 1, "inner": 4096, "outer": 4096,
         "act": "none", "bias": True, "residual": True, "save": False, "dtype": "f16"},
        # a decode batch's first product of a plain feed-forward layer
        {"name": "linear_batch", "kind": "linear", "tokens": 24, "inner": 4096, "outer": 16384,
         "act": "gelu", "bias": True, "residual": False, "save": False, "dtype": "bf16"},
        # a short prompt through a layer whose sizes fit no tile and no vector
        {"name": "linear_odd", "kind": "linear", "tokens": 777, "inner": 1021, "outer": 5003,
         "act": "relu", "bias": True, "residual": True, "save": False, "dtype": "f16"},
        # the same layer in training: what the backward pass needs is written too
        {"name": "linear_train", "kind": "linear", "tokens": 8192, "inner": 4096, "outer": 16384,
         "act": "gelu_tanh", "bias": True, "residual": False, "save": True, "dtype": "bf16"},
        # its backward pass
        {"name": "linear_back", "kind": "linear_back", "tokens": 8192, "inner": 4096, "outer": 16384,
         "act": "gelu_tanh", "bias": True, "dtype": "bf16"},
        # a small model's layer, a ragged batch
        {"name": "linear_back_small", "kind": "linear_back", "tokens": 1031, "inner": 768,
         "outer": 2312, "act": "gelu", "bias": True, "dtype": "f16"},
        # one conversation: the gated half of a block
        {"name": "gated_one", "kind": "gated", "tokens": 1, "inner": 4096, "outer": 11264,
         "act": "silu", "save": False, "dtype": "bf16"},
        # gradients of the gated half alone, at sizes that fit no tile
        {"name": "gated_back_odd", "kind": "gated_back", "tokens": 515, "inner": 1032, "outer": 2747,
         "act": "gelu", "dtype": "f16"},
        # a decode batch through the whole block
        {"name": "ffn_batch", "kind": "ffn", "tokens": 61, "inner": 4096, "outer": 11264,
         "act": "silu", "residual": True, "save": False, "dtype": "f16"},
        # a prompt of ordinary length through the whole block
        {"name": "ffn_prompt", "kind": "ffn", "tokens": 500, "inner": 4096, "outer": 11264,
         "act": "silu", "residual": True, "save": False, "dtype": "bf16"},
        # training, forward and backward
        {"name": "ffn_train", "kind": "ffn", "tokens": 8192, "inner": 4096, "outer": 11264,
         "act": "silu", "residual": True, "save": True, "dtype": "bf16"},
        {"name": "ffn_back", "kind": "ffn_back", "tokens": 8192, "inner": 4096, "outer": 11264,
         "act": "silu", "dtype": "bf16"},
    ]


ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")


def draw(rng):
    def spread(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    kind = rng.choice(("linear", "linear", "linear_back", "gated", "gated_back", "ffn", "ffn_back"))
    c = {"kind": kind, "tokens": spread(1, 8192), "inner": spread(64, 8192),
         "outer": spread(64, 16384), "dtype": rng.choice(("f16", "bf16"))}
    # most layers have sizes that are multiples of 8, some of 64, a few have any
    step = rng.choice((1, 8, 8, 64, 64, 128))
    for k in ("inner", "outer"):
        c[k] = max(step, c[k] // step * step)
    if kind.startswith("linear"):
        c["act"], c["bias"] = rng.choice(ACTS), rng.random() < 0.6
    else:
        c["act"] = rng.choice(("silu", "silu", "gelu", "gelu_tanh", "relu", "sigmoid", "none"))
    if kind in ("linear", "ffn"):
        c["residual"] = rng.random() < 0.5
    if kind in ("linear", "gated", "ffn"):
        c["save"] = rng.random() < 0.4
    most = work(listed()[-1])
    while any(work(c)[k] > most[k] for k in most):
        c["tokens"] = (c["tokens"] + 1) // 2
        c["outer"] = max(step, c["outer"] * 3 // 4 // step * step)
    return c


def _matrices(kind):
    return 1 if kind.startswith("linear") else 2 if kind.startswith("gated") else 3


def work(case):
    t, k, n, kind = case["tokens"], case["inner"], case["outer"], case["kind"]
    product = 2 * t * k * n
    weights = _matrices(kind) * n * k
    if kind == "linear":
        values = t * k + weights + t * n * (1 + case["save"] + case["residual"]) + n * case["bias"]
        return {"bytes": 2 * values, "flops": product}
    if kind == "linear_back":
        saved = t * n if case["act"] != "none" else 0
        return {"bytes": 2 * (2 * t * k + t * n + saved + 2 * weights + n * case["bias"]),
                "flops": 2 * product}
    if kind == "gated":
        return {"bytes": 2 * (t * k + weights + t * n * (3 if case["save"] else 1)),
                "flops": 2 * product}
    if kind == "gated_back":
        return {"bytes": 2 * (2 * t * k + 3 * t * n + 2 * weights), "flops": 4 * product}
    if kind == "ffn":
        values = weights + t * k * (2 + case["residual"]) + t * n * 2 * case["save"]
        return {"bytes": 2 * values, "flops": 3 * product}
    return {"bytes": 2 * (3 * t * k + 2 * t * n + 2 * weights), "flops": 6 * product}


# ----------------------------------------------------------------- the inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 7919 + 17)
    t, k, n, kind = case["tokens"], case["inner"], case["outer"], case["kind"]
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=gen).mul_(scale).to(dtype)

    # activations behind a norm: channels of different size, a few of them large
    channel = torch.exp(0.4 * torch.randn(k, device=dev, generator=gen))
    s = {"case": dict(case)}
    s["x"] = torch.randn(t, k, device=dev, generator=gen).mul_(channel).to(dtype)
    near = 1.0 / math.sqrt(k)
    if kind.startswith("linear"):
        s["w"] = normal(n, k, scale=near)
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
    else:
        s["wg"], s["wu"] = normal(n, k, scale=near), normal(n, k, scale=near)
    if kind.startswith("ffn"):
        s["wd"] = normal(k, n, scale=1.0 / math.sqrt(n))
    wide = kind.startswith("linear")
    if case.get("residual"):
        s["r"] = normal(t, n if wide else k)
    else:
        s["r"] = None
    if kind.endswith("_back"):  # gradients under a loss scale
        s["dy"] = normal(t, k if kind == "ffn_back" else n, scale=0.5)
        if wide:
            s["z"] = normal(t, n, scale=1.3) if case["act"] != "none" else None
        else:
            s["g"], s["u"] = normal(t, n, scale=1.3), normal(t, n, scale=1.3)
    return s


# ------------------------------------------------------------- the plain forms
_ROOT = math.sqrt(2.0 / math.pi)


def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return z * (z > 0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(_ROOT * (z + 0.044715 * z * z * z)))
    s = 1.0 / (1.0 + torch.exp(-z))
    return s if name == "sigmoid" else z * s


def _slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return (0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) * (0.5 * math.sqrt(2.0 / math.pi)))
    if name == "gelu_tanh":
        h = torch.tanh(_ROOT * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + h) + 0.5 * z * (1.0 - h * h) * _ROOT * (1.0 + 3 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 - s) if name == "sigmoid" else s * (1.0 + z * (1.0 - s))


def _plain(s):
    c = s["case"]
    kind, act, dtype = c["kind"], c["act"], s["x"].dtype
    x = s["x"].float()
    if kind == "linear":
        z = x @ s["w"].float().t()
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _act(act, z)
        if s["r"] is not None:
            y = y + s["r"].float()
        return [y.to(dtype), z.to(dtype)] if c["save"] else [y.to(dtype)]
    if kind == "linear_back":
        dz = s["dy"].float()
        if act != "none":
            dz = dz * _slope(act, s["z"].float())
        out = [(dz @ s["w"].float()).to(dtype), (dz.t() @ x).to(dtype)]
        if s["b"] is not None:
            out.append(dz.sum(0, dtype=torch.float64).to(dtype))
        return out
    wg, wu = s["wg"].float(), s["wu"].float()
    if kind in ("gated", "ffn"):
        g, u = x @ wg.t(), x @ wu.t()
        y = _act(act, g) * u
        if kind == "ffn":
            y = y @ s["wd"].float().t()
            if s["r"] is not None:
                y = y + s["r"].float()
        return [v.to(dtype) for v in ((y, g, u) if c["save"] else (y,))]
    g, u, dy = s["g"].float(), s["u"].float(), s["dy"].float()
    dh = dy @ s["wd"].float() if kind == "ffn_back" else dy
    dg, du = dh * u * _slope(act, g), dh * _act(act, g)
    out = [dg @ wg + du @ wu, dg.t() @ x, du.t() @ x]
    if kind == "ffn_back":
        out.append(dy.t() @ (_act(act, g) * u))
    return [v.to(dtype) for v in out]


def _calls(s):
    import sion_b200 as sion

    c = s["case"]
    kind, act = c["kind"], c["act"]
    if kind == "linear":
        call = sion.linear_save if c["save"] else sion.linear
        y = call(s["x"], s["w"], s["b"], s["r"], activation=act)
        return list(y) if c["save"] else [y]
    if kind == "linear_back":
        dx, dw, db = sion.linear_backward(s["dy"], s["x"], s["w"], s["z"], activation=act,
                                          bias=s["b"] is not None)
        return [dx, dw] if db is None else [dx, dw, db]
    if kind == "gated":
        call = sion.gated_linear_save if c["save"] else sion.gated_linear
        h = call(s["x"], s["wg"], s["wu"], activation=act)
        return list(h) if c["save"] else [h]
    if kind == "gated_back":
        return list(sion.gated_linear_backward(s["dy"], s["x"], s["wg"], s["wu"], s["g"], s["u"],
                                               activation=act))
    if kind == "ffn":
        call = sion.gated_ffn_save if c["save"] else sion.gated_ffn
        y = call(s["x"], s["wg"], s["wu"], s["wd"], s["r"], activation=act)
        return list(y) if c["save"] else [y]
    return list(sion.gated_ffn_backward(s["dy"], s["x"], s["wg"], s["wu"], s["wd"], s["g"], s["u"],
                                        activation=act))


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    act, kind = case["act"], case["kind"]

    def value_and_slope(z):
        """The activation and its derivative, from the definitions."""
        if act == "none":
            return z, torch.ones_like(z)
        if act == "relu":
            return torch.clamp(z, min=0), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
        if act == "gelu":  # z Phi(z), Phi + z phi(z)
            area = torch.special.ndtr(z)
            return z * area, area + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        if act == "gelu_tanh":  # z sigma(2 a)
            a = math.sqrt(8 / math.pi) * (z + 0.044715 * z.pow(3))
            p = torch.special.expit(a)
            return z * p, p + z * p * torch.special.expit(-a) * math.sqrt(8 / math.pi) * (1 + 0.134145 * z.square())
        p, q = torch.special.expit(z), torch.special.expit(-z)
        return (p, p * q) if act == "sigmoid" else (z * p, p + z * p * q)

    if kind.startswith("linear"):
        if kind == "linear":
            z = torch.einsum("tk,nk->tn", s["x"], s["w"])
            z = z if s["b"] is None else z.add_(s["b"])
            y = value_and_slope(z)[0]
            y = y if s["r"] is None else y + s["r"]
            return [y, z] if case["save"] else [y]
        dz = s["dy"] if act == "none" else value_and_slope(s["z"])[1].mul_(s["dy"])
        out = [torch.einsum("tn,nk->tk", dz, s["w"]), torch.einsum("tn,tk->nk", dz, s["x"])]
        return out if s["b"] is None else out + [dz.sum(0)]
    if not kind.endswith("_back"):
        g = torch.einsum("tk,fk->tf", s["x"], s["wg"])
        u = torch.einsum("tk,fk->tf", s["x"], s["wu"])
        y = value_and_slope(g)[0] * u
        if kind == "ffn":
            y = torch.einsum("tf,kf->tk", y, s["wd"])
            y = y if s["r"] is None else y + s["r"]
        return [y, g, u] if case["save"] else [y]
    a, slope = value_and_slope(s["g"])
    dh = torch.einsum("tk,kf->tf", s["dy"], s["wd"]) if kind == "ffn_back" else s["dy"]
    dg, du = dh * s["u"] * slope, dh * a
    dx = torch.einsum("tf,fk->tk", dg, s["wg"]) + torch.einsum("tf,fk->tk", du, s["wu"])
    out = [dx, torch.einsum("tf,tk->fk", dg, s["x"]), torch.einsum("tf,tk->fk", du, s["x"])]
    if kind == "ffn_back":
        out.append(torch.einsum("tk,tf->kf", s["dy"], a * s["u"]))
    return out
