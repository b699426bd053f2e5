"""The bound of tests/ffn_tails.py holds for the same steps in fp32 and is narrow enough to
tell a lost tail."""
import numpy as np
import pytest
import torch

import ffn_ref as R
import ffn_tails as A


@pytest.mark.parametrize("name", A.NAMES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_formulas_and_width(name, dtype):
    z = A.every(dtype, 30)
    a, d = A.bounds(name, z, dtype)
    want = R.act(name, z.double())
    for (v, _), w in zip((a, d), want):
        assert (v - w).abs().max() < 1e-12
    # every value that the type holds with all its bits is told from 0 and from one that is
    # off by three roundings (the bounds leave one)
    normal = max(torch.finfo(dtype).tiny, 1e4 * A.LOST)
    for v, e in (a,) if name != "sigmoid" else (a, d):
        held = (v.abs() >= normal) & (z > -10)
        assert held.any() and (e[held] < 0.5 * v.abs()[held]).all()
        assert (e[held] < 3 * R.HALF[dtype] * v.abs()[held]).all()
    tail = (z >= -5) & (z <= -4)
    assert (a[1][tail] < 1.1 * (R.HALF[dtype] * a[0][tail].abs() + R.TINY[dtype])).all()


def test_the_polynomial_of_the_normal_tail():
    """normal_area of activation.cuh with numpy's fp32 steps, against 64 bits."""
    f = np.float32
    z = -np.arange(0.01, 13, 0.01).astype(f)
    e = np.exp2((f(-0.721347520) * z) * z)
    t = f(1) / (np.abs(z) * f(0.353553391) + f(1))
    c = np.full_like(z, f(0.04410203546))
    for k in (-0.17836862803, 0.19461159408, 0.01894582063, 0.14075168967, 0.13879109917,
              0.14116570354):
        c = c * t + f(k)
    tail = torch.from_numpy((c * t * e).astype(np.float64))
    z = torch.from_numpy(z.astype(np.float64))
    want = torch.special.erfc(-z / 2 ** 0.5) / 2
    off = ((tail - want) / want).abs()
    assert (off <= (1.125 * z * z + 47) * R.EPS).all()
    assert off[z > -5].max() < 2.5e-6 and off.max() < 8e-6
