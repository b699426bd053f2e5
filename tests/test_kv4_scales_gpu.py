"""kv4_attention over values of very different size, against plain 64-bit sums.

Tolerance, elementwise. With p the probabilities before their division by S = sum(p):
A = sum p |V| / S. Weights are rounded to 11 bits, a relative 2^-11 each, in the
sum and in its divisor: 2^-11 (A + |O|) <= 2^-10 A. Exponents carry 2e-5 of fp32
rounding, on both sides: 4e-5 A. What a weight below fp16's normal range loses of
(code - 8) is at most 2^-25 * 8 where the row's largest weight is 2^6 or more:
n 2^-28 B with B = max p ||V||_inf / S. Sums are fp32, of terms up to 15 p scale <=
2 p ||V||_inf that cancel where a value is near 0: the matrix unit adds 32 tokens
and as many offsets at a time, each cut at 2^-23 of the largest, 2^7 2^-23 B, and each
step of 32 tokens is one fp32 addition more: (2^-16 + n 2^-28) B. The result is
rounded once, 2^-11 or 2^-8 of it, half of fp16's smallest step at the bottom."""
import numpy as np
import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu

TYPES = {"f16": (torch.float16, 2.0 ** -11), "bf16": (torch.bfloat16, 2.0 ** -8)}


def sion():
    import sion_b200
    return sion_b200


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def filled(k, v, page):
    """A pool of one slot that holds k, v [heads, tokens, D], its table and lens."""
    kvh, n, D = k.shape
    need = R.pages_for(n, page)
    pool = torch.zeros(need, sion().kv4_page_bytes(kvh, D, page), dtype=torch.uint8, device="cuda")
    table = np.random.default_rng(n).permutation(need).astype(np.int32)[None]
    dev = [torch.from_numpy(x).half()[None].cuda() for x in (k, v)]
    sion().kv4_append(pool, i32(table), i32([n]), *dev)
    return pool, table


def held(pool, table, n, page, kvh, D):
    K, V = R.decode(pool.cpu().numpy(), page, kvh, D)
    at = np.arange(n)
    return [x[table[0][at // page], :, at % page].transpose(1, 0, 2) for x in (K, V)]


def check(pool, table, n, q, kvh, page):
    """One slot's attention against 64 bits; q [1, heads, rows, D] on the host."""
    D, H, rows = q.shape[3], q.shape[1], q.shape[2]
    eps = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    o, lse = sion().kv4_attention_lse(q.cuda(), pool, i32(table), i32([n]), kvh)
    o, lse = o.double().cpu().numpy()[0], lse.double().cpu().numpy()[0]
    K, V = held(pool, table, n, page, kvh, D)
    x = q.double().numpy()[0]
    for h in range(H):
        k, v = K[h // (H // kvh)], V[h // (H // kvh)]
        for i in range(rows):
            m = n - rows + i + 1
            s = k[:m] @ x[h, i] / np.sqrt(D)
            p = np.exp(s - s.max())
            S = p.sum()
            ref, A = p @ v[:m] / S, p @ np.abs(v[:m]) / S
            B = (p * np.abs(v[:m]).max(1)).max() / S
            tol = (2.0 ** -10 + 4e-5) * A + (2.0 ** -16 + 2 * m * 2.0 ** -28) * B + \
                eps * np.abs(ref) + 2.0 ** -25
            err = np.abs(o[h, i] - ref)
            assert (err <= tol).all(), (h, i, float((err / tol).max()))
            want = s.max() + np.log(S)
            assert abs(lse[h, i] - want) <= 2e-5 + 1e-6 * abs(want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,rows,group", [(128, 1, 4), (64, 1, 8), (64, 5, 8), (128, 3, 4)])
@pytest.mark.parametrize("big,small", [(30000.0, 1e-3), (30000.0, 1e-5), (30000.0, 1e-6),
                                       (3000.0, 1e-6), (1.0, 1e-6)])
def test_equal_probabilities(dtype, D, rows, group, big, small):
    # one token's values far above the others', or the others' above one's: each
    # counts for its probability, wherever it lies
    rng = np.random.default_rng(int(D + rows + big))
    page = 16
    for n in (11, 100, 700):
        for where in (0, n // 2, n - rows):
            for one, rest in ((big, small), (small, big)):
                v = rng.standard_normal((1, n, D)) * rest
                v[0, where] = rng.standard_normal(D) * one
                if rest == small:
                    v[0, :where] += small * 3  # not around zero
                pool, table = filled(np.zeros((1, n, D)), np.clip(v, -65504, 65504), page)
                q = torch.zeros(1, group, rows, D, dtype=TYPES[dtype][0])
                check(pool, table, n, q, 1, page)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,rows,group", [(128, 1, 4), (64, 5, 8)])
@pytest.mark.parametrize("score", [8.0, 16.0, 24.0])
def test_unlikely_large_values_and_likely_small_ones(dtype, D, rows, group, score):
    # the small tokens are exp(score) times as likely as the large one, whose values
    # are about that much larger, so that both make the result; and the reverse
    rng = np.random.default_rng(int(score))
    page, ratio = 32, float(np.exp(score))
    for n in (40, 3000):
        for where in (0, n - rows):
            for sign in (1.0, -1.0):
                k = np.zeros((1, n, D))
                k[0, where] = -sign * score / np.sqrt(D)
                big = min(30000.0, 0.02 * ratio)
                v = rng.standard_normal((1, n, D)) * (big / ratio) / 30
                v[0, where] = rng.standard_normal(D) * big / 4
                if sign < 0:
                    v[0, where] /= ratio
                v[0, 1::3] += big / ratio  # bases well above their scales
                pool, table = filled(k, v, page)
                q = torch.ones(1, group, rows, D, dtype=TYPES[dtype][0])
                q[:, 1::2] *= 0.5
                check(pool, table, n, q, 1, page)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,group", [(1, 8), (5, 8)])
def test_unlikely_tokens_of_large_bases(dtype, rows, group):
    # scales are alike: one likely token around zero, 4000 unlikely ones around 1000,
    # whose sum is well above what the result is rounded to
    rng = np.random.default_rng(4)
    n, D, page = 4001, 64, 64
    for where in (0, n - rows):
        for bits in (22, 28, 33):
            k, v = np.zeros((1, n, D)), rng.standard_normal((1, n, D)) + 1000.0
            k[0, where] = bits * np.log(2) / np.sqrt(D)
            v[0, where] -= 1000.0
            pool, table = filled(k, v, page)
            check(pool, table, n, torch.ones(1, group, rows, D, dtype=TYPES[dtype][0]), 1, page)
