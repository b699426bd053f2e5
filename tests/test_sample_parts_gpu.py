"""Sampling where a cluster's CTA has the largest part of a row that it can have."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

# 65535 = round(exp(-16 / T) 2^31): all the low half of a mass, the value for which
# sums of low halves come nearest to the end of 32 bits
LOW = 65535


def temperature():
    t = np.float32(-16 / np.log(LOW / 2.0 ** 31))
    for t in (t, np.nextafter(t, np.float32(0)), np.nextafter(t, np.float32(9))):
        z = np.float32(-16) / t
        if np.rint(np.float32(np.exp(z.astype(np.float64))) * np.float32(2.0 ** 31)) == LOW:
            return t
    raise AssertionError


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [131072, 131073, 262144, 262145, 262147, 131071])
def test_masses_of_a_full_part_are_summed_exactly(V, dtype):
    rows, p, t = 100, 0.5, temperature()
    x = torch.zeros(rows, V, dtype=dtype, device="cuda")
    x[:, 5] = 16
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    args = dict(temperature=torch.full((rows,), float(t), device="cuda"),
                top_p=torch.full((rows,), p, device="cuda"))
    tok, lp = (a.cpu().numpy() for a in sample(x, torch.from_numpy(u).cuda(), **args))
    # token 5, then the others by index while less than p of all is before them
    total = 2 ** 31 + (V - 1) * LOW
    others = int(np.ceil((p * total - 2 ** 31) / LOW))
    mass = np.full(others + 1, LOW, np.int64)
    mass[5] = 2 ** 31
    upto = np.cumsum(mass)
    want = np.searchsorted(upto, np.floor(u.astype(np.float64) * upto[-1]).astype(np.int64), "right")
    np.testing.assert_array_equal(tok, want)
    for i in (0, 50, 99):
        one = {k: v[i:i + 1].contiguous() for k, v in args.items()}
        a, b = sample(x[i:i + 1], torch.from_numpy(u[i:i + 1]).cuda(), **one)
        assert int(a) == tok[i] and float(b) == lp[i]


def sample(*a, **k):
    import sion_b200
    return sion_b200.sample(*a, **k)
