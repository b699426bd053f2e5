"""Activations and derivatives of the feed-forward kernels at every 16-bit value up to 100, with
a relative bound (ffn_tails.py): products of depth 1 or with unit vectors hand the values
through unchanged."""
import pytest
import torch

import ffn_ref as R
import ffn_tails as A
from test_ffn_gpu import DTYPES

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    import sion_b200
    return sion_b200


def values(dtype, width):
    z = A.every(dtype)
    z = z[:len(z) // width * width]
    return z.cuda()


@pytest.mark.parametrize("name", A.NAMES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 20, 130])
def test_activations(S, name, dtype, T):
    # x = 1, weights = the values: z itself in front of the activation, in every token
    z = values(dtype, 8)
    x, w, one = (torch.ones(s, dtype=dtype, device="cuda") for s in ((T, 1), (1, 1), (len(z), 1)))
    want, _ = A.bounds(name, z, dtype)
    want = tuple(t.expand(T, -1) for t in want)
    for y in (S.linear(x, z[:, None], None, None, name),
              S.gated_linear(x, z[:, None], one, name)):
        R.check(y, want, name)
    if T == 130:  # tokens carry the values
        R.check(S.linear(z[:, None], w, None, None, name)[:, 0], A.bounds(name, z, dtype)[0], name)


@pytest.mark.parametrize("name", A.NAMES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [64, 61])
def test_derivatives(S, name, dtype, n):
    # n rows or columns of values; 61: rows that are no whole vectors
    z = values(dtype, n).view(-1, n)
    eye = torch.eye(n, dtype=dtype, device="cuda")
    a, d = A.bounds(name, z, dtype)
    one = torch.ones_like(z)
    x = torch.zeros_like(z)
    # dx = dz I; a column's sum of one row each
    R.check(S.linear_backward(one, x, eye, z, name)[0], d, "dz")
    row = z[len(z) // 3:][:1]
    db = S.linear_backward(one[:1], x[:1], eye, row, name, bias=True)[2]
    R.check(db, tuple(t[len(z) // 3] for t in d), "db")
    # dw = (dg, du)^T I
    zt, ones = z.t(), one.t()
    w = torch.zeros(len(z), n, dtype=dtype, device="cuda")
    _, dg, du = S.gated_linear_backward(ones, eye, w, w, zt, ones, name)
    R.check(dg, d, "dg")
    R.check(du, a, "du")
    # dh = 1 as the product of a unit vector and a row of ones; h in dwd's first row
    dy = torch.zeros(n, n, dtype=dtype, device="cuda")
    dy[:, 0] = 1
    wd = torch.zeros(n, len(z), dtype=dtype, device="cuda")
    wd[0] = 1
    _, dg, du, _ = S.gated_ffn_backward(dy, eye, w, w, wd, zt, ones, name)
    R.check(dg, d, "ffn dg")
    R.check(du, a, "ffn du")
    dwd = S.gated_ffn_backward(eye, eye, w, w, wd, zt, ones, name)[3]
    R.check(dwd, (a[0].t(), a[1].t()), "h")
