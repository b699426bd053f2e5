"""Feed-forward operators bit for bit: inputs are small integers, of which every sum, in any
order, is an integer below 2^24 and so exact in fp32; what is left are the documented
roundings to 16 bits, which the oracle makes at the same places. One term of a sum left
out, taken twice or taken from a neighbour changes results, whatever the depth."""
import pytest
import torch

from test_ffn_calls_gpu import SHAPES
from test_ffn_gpu import DTYPES, GATED, LINEAR

pytestmark = pytest.mark.gpu

# few-token and narrow kernels with their depth in 2, 4 and 8 parts, and depths that end one
# instruction (16), one block of 64 and one element behind a stage
DEEP = [(1, 4112, 40), (8, 8193, 24), (20, 4096, 4096), (24, 8192, 1024), (40, 8256, 520),
        (64, 8208, 1000), (61, 11264, 4096), (128, 2064, 512), (130, 4161, 264), (300, 20001, 136)]


@pytest.fixture(scope="module")
def S():
    import sion_b200
    return sion_b200


def ints(*shape, terms, dtype, seed):
    """-1, 0 or 1, of which about `terms` in 1 are not 0."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    sign = torch.randint(0, 2, shape, device="cuda", generator=g) * 2 - 1
    return (sign * (torch.rand(*shape, device="cuda", generator=g) < terms)).to(dtype)


def small(*shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype)


def product(a, b):
    """a b^T; no partial sum reaches 2^24."""
    a, b = a.double(), b.double()
    assert (a.abs() @ b.abs().t()).max() < 2 ** 24
    return a @ b.t()


def same(got, want, what):
    want = want.to(got.dtype)
    if not torch.equal(got, want):
        bad = (got != want).nonzero()
        i = tuple(bad[0].tolist())
        raise AssertionError(f"{what}: {len(bad)} of {got.numel()} differ, first {i}: "
                             f"{got[i].item()}, not {want[i].item()}")


def densities(total, a, b):
    """Of one operand that is summed with a second one over a, with a third one over b: so
    that about `total` terms of a sum are not 0."""
    one = min(1.0, (total / max(a, b)) ** 0.5)
    return one, min(1.0, total / (a * one)), min(1.0, total / (b * one))


@pytest.mark.parametrize("T,K,N", LINEAR + SHAPES + DEEP)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(S, T, K, N, dtype):
    d = min(1.0, (600 / K) ** 0.5)
    x, w = ints(T, K, terms=d, dtype=dtype, seed=1), ints(N, K, terms=d, dtype=dtype, seed=2)
    b, r = small(N, dtype=dtype, seed=3), small(T, N, dtype=dtype, seed=4)
    plain = product(x, w)
    same(S.linear(x, w), plain, "plain")
    z = plain + b.double()
    same(S.linear(x, w, b, r, "relu"), z.relu() + r.double(), "relu")
    y, pre = S.linear_save(x, w, b, r, "relu")
    same(y, z.relu() + r.double(), "y")
    same(pre, z, "pre")


@pytest.mark.parametrize("T,K,N", LINEAR + SHAPES + [(9001, 64, 72), (20000, 8, 1000), (33, 40, 9000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_backward(S, T, K, N, dtype):
    dg, dw, dx = densities(600, N, T)
    grad, pre = ints(T, N, terms=dg, dtype=dtype, seed=1), small(T, N, dtype=dtype, seed=2)
    w, x = ints(N, K, terms=dw, dtype=dtype, seed=3), ints(T, K, terms=dx, dtype=dtype, seed=4)
    for name in ("none", "relu"):
        dz = grad.double() * (pre > 0) if name == "relu" else grad.double()
        got = S.linear_backward(grad, x, w, pre, name, bias=True)
        for g, want, what in zip(got, (product(dz, w.t()), product(dz.t(), x.t()), dz.sum(0)),
                                 ("dx", "dw", "db")):
            same(g, want, f"{name} {what}")


BLOCKS = GATED + [(100, 4096, 1024), (500, 1024, 4096), (33, 4096, 11264), (479, 128, 8192),
                  (4100, 72, 184), (20, 1024, 3000)]


@pytest.mark.parametrize("T,K,F", BLOCKS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated(S, T, K, F, dtype):
    d = min(1.0, (30 / K) ** 0.5)
    x = ints(T, K, terms=d, dtype=dtype, seed=1)
    wg, wu = (ints(F, K, terms=d, dtype=dtype, seed=i) for i in (2, 3))
    wd, r = ints(K, F, terms=min(1.0, 60 / F), dtype=dtype, seed=4), small(T, K, dtype=dtype, seed=5)
    g, u = product(x, wg), product(x, wu)
    for name in ("none", "relu"):
        h = ((g.relu() if name == "relu" else g) * u).to(dtype)
        got = S.gated_linear_save(x, wg, wu, name)
        for a, want, what in zip(got, (h, g, u), ("h", "gate", "up")):
            same(a, want, f"{name} {what}")
        same(S.gated_ffn(x, wg, wu, wd, r, name), product(h, wd) + r.double(), f"{name} y")


@pytest.mark.parametrize("T,K,F", BLOCKS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_backward(S, T, K, F, dtype):
    dt, dy_dx, _ = densities(200, T, F)
    gate, up = small(T, F, dtype=dtype, seed=1), small(T, F, dtype=dtype, seed=2)
    x = ints(T, K, terms=dy_dx, dtype=dtype, seed=3)
    wg, wu = (ints(F, K, terms=min(1.0, 100 / F), dtype=dtype, seed=i) for i in (4, 5))
    dy = ints(T, K, terms=min(1.0, (20 / K) ** 0.5, (200 / T) ** 0.5), dtype=dtype, seed=6)
    wd = ints(K, F, terms=min(1.0, (20 / K) ** 0.5), dtype=dtype, seed=7)
    dh16 = ints(T, F, terms=dt, dtype=dtype, seed=8)
    for name in ("none", "relu"):
        a, slope = (gate.double().relu(), (gate > 0).double()) if name == "relu" else \
            (gate.double(), torch.ones_like(gate).double())
        h = (a * up.double()).to(dtype)

        def gradients(dh):
            dg, du = (dh * up.double() * slope).to(dtype), (dh * a).to(dtype)
            dx = product(torch.cat([dg, du], 1), torch.cat([wg, wu]).t())
            return dx, product(dg.t(), x.t()), product(du.t(), x.t())

        for got, want, what in zip(S.gated_linear_backward(dh16, x, wg, wu, gate, up, name),
                                   gradients(dh16.double()), ("dx", "dwg", "dwu")):
            same(got, want, f"{name} {what}")
        want = (*gradients(product(dy, wd.t())), product(dy.t(), h.t()))
        for got, ref, what in zip(S.gated_ffn_backward(dy, x, wg, wu, wd, gate, up, name), want,
                                  ("dx", "dwg", "dwu", "dwd")):
            same(got, ref, f"{name} ffn {what}")


# more columns than there are counters for the bias gradient's sums (33 rows of 1.2 million, in
# vectors or not), and more rows than 32 a block can hold (2.2 million)
@pytest.mark.parametrize("T,K,N", [(33, 8, 1200000), (40, 3, 140001), (2200001, 8, 8), (2200001, 7, 9)])
def test_very_many_rows_or_columns(S, T, K, N):
    for dtype in DTYPES:
        test_linear(S, T, K, N, dtype)
        test_linear_backward(S, T, K, N, dtype)
        if N < 100:
            test_gated(S, T, K, N, dtype)
            test_gated_backward(S, T, K, N, dtype)
