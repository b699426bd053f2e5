"""The activations and their derivatives in 64 bits with a bound that is relative, tails
included: what the steps that activation.cuh takes in fp32 may be off, in units of
EPS = 2^-24, half a step of fp32.

  The approximate 2^x is good to 4, 1 / x to 2 (their documented bounds), other steps to 1;
  a constant is off by less than 1 / 4. An error d of x is one of d ln 2 in 2^x.
  logistic(s), of an s that is good to i: e^-s to (i + 1.25) |s| + 4, where e^-s < 1 only
  s e^-s < 0.4 of that |s| counts; the sum 1, the reciprocal 2.
  gelu: e^(-z^2 / 2) has an exponent of two roundings: 1.125 z^2 + 4; t is good to 3.25, which
  t c(t) takes at most 2.5 times; the polynomial's steps 6, its fit 25, two products.
  Sums (the derivatives) are bounded by their terms' errors, 1 - p by p's and its own step."""
import math

import torch

from ffn_ref import EPS, HALF, TINY

SLOPE = math.sqrt(8 / math.pi)
NAMES = ("gelu", "gelu_tanh", "silu", "sigmoid")
# What is smaller may be lost: past an exponent of 88.7 e^-s is infinite in fp32 and the
# logistic function 0, where act and act' are still up to 10 x 24 x e^-88.7 (gelu_tanh's slope).
LOST = 1e-36


def both(name, z):
    """((act, error), (act', error)), errors in EPS."""
    m = z.abs()
    if name == "gelu":
        # (torch.special.ndtr loses the tail: its 1 + erf cancels)
        area, density = torch.special.erfc(-z / math.sqrt(2)) / 2, torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        e = 1.125 * z * z + 4
        ea = e + 43
        d = area + z * density
        return (z * area, (ea + 1) * (z * area).abs()), \
            (d, (e + 3) * m * density + ea * area + d.abs())
    inner = SLOPE * (z + 0.044715 * z ** 3) if name == "gelu_tanh" else z
    p, q = torch.sigmoid(inner), torch.sigmoid(-inner)
    i = 4 if name == "gelu_tanh" else 0  # roundings of the argument
    e = (i + 1.25) * ((-inner).clamp(min=0) + 0.4) + 7
    if name == "sigmoid":
        return (p, e * p), (p * q, (1.25 * m + 17) * p * q)
    s = SLOPE * (1 + 3 * 0.044715 * z * z) if name == "gelu_tanh" else torch.ones_like(z)
    d = p + z * p * q * s
    return (z * p, (e + 1) * m * p), \
        (d, m * p * s * (q * (e + 6) + p * e) + p * e + d.abs())


def bounds(name, z, dtype):
    """((act, bound), (act', bound)), each rounded once to dtype."""
    out = []
    for v, e in both(name, z.double()):
        e = e * EPS
        out.append((v, e + HALF[dtype] * (v.abs() + e) + TINY[dtype] + LOST))
    return out


def every(dtype, limit=100):
    """Every value of the type from -limit to limit."""
    z = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    return z[z.double().abs() <= limit]
