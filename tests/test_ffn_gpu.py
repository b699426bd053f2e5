"""Feed-forward operators on the GPU against 64 bits, elementwise (ffn_ref.py)."""
import pytest
import torch

import ffn_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def S():
    import sion_b200
    return sion_b200


@pytest.fixture(autouse=True)
def watchdog():
    yield
    from sion_b200 import abi
    assert abi.watchdog_status(clear=True) == 0


def rand(*shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def linear_inputs(T, K, N, dtype, seed=0):
    x = rand(T, K, dtype=dtype, seed=seed + 1)
    w = rand(N, K, dtype=dtype, seed=seed + 2, scale=K ** -0.5)
    b = rand(N, dtype=dtype, seed=seed + 3)
    r = rand(T, N, dtype=dtype, seed=seed + 4)
    return x, w, b, r


def gated_inputs(T, K, F, dtype, seed=0):
    x = rand(T, K, dtype=dtype, seed=seed + 1)
    wg = rand(F, K, dtype=dtype, seed=seed + 2, scale=K ** -0.5)
    wu = rand(F, K, dtype=dtype, seed=seed + 3, scale=K ** -0.5)
    wd = rand(K, F, dtype=dtype, seed=seed + 4, scale=F ** -0.5)
    return x, wg, wu, wd


# tokens from one to several tiles; sizes on and off the borders of 8, 16, 32, 64, 128, 256
LINEAR = [(1, 1, 1), (1, 8, 8), (1, 64, 128), (3, 7, 5), (8, 65, 33), (16, 128, 256), (17, 200, 130),
          (31, 264, 31), (32, 512, 100), (33, 1000, 257), (64, 4096, 64), (65, 72, 1000),
          (128, 128, 128), (129, 63, 129), (256, 320, 384), (300, 1021, 515), (513, 256, 2056),
          (1000, 520, 777), (2048, 1024, 1536), (4096, 64, 64), (257, 8192, 264), (700, 2048, 5000)]


@pytest.mark.parametrize("T,K,N", LINEAR)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(S, T, K, N, dtype):
    x, w, b, r = linear_inputs(T, K, N, dtype)
    R.check(S.linear(x, w), R.linear(x, w)[0], "plain")
    y, pre = S.linear_save(x, w, b, r, "silu")
    want = R.linear(x, w, b, r, "silu")
    R.check(y, want[0], "y")
    R.check(pre, want[1], "pre")


@pytest.mark.parametrize("name", R.ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 200])
def test_every_activation(S, name, dtype, T):
    x, w, b, r = linear_inputs(T, 96, 168, dtype)
    x = x * 3  # into both tails
    y, pre = S.linear_save(x, w, b, None, name)
    want = R.linear(x, w, b, None, name)
    R.check(y, want[0], name)
    R.check(pre, want[1], name)
    x, wg, wu, wd = gated_inputs(T, 96, 168, dtype)
    h, g, u = S.gated_linear_save(x * 3, wg, wu, name)
    for got, ref in zip((h, g, u), R.gated(x * 3, wg, wu, name)):
        R.check(got, ref, name)
    assert torch.equal(S.gated_linear(x * 3, wg, wu, name), h)


@pytest.mark.parametrize("T,K,N", LINEAR)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_backward(S, T, K, N, dtype):
    x, w, b, r = linear_inputs(T, K, N, dtype)
    grad, pre = rand(T, N, dtype=dtype, seed=8), rand(T, N, dtype=dtype, seed=9)
    for name in ("none", "gelu"):
        got = S.linear_backward(grad, x, w, pre, name, bias=True)
        for g, want, what in zip(got, R.linear_backward(grad, x, w, pre, name), ("dx", "dw", "db")):
            R.check(g, want, f"{name} {what}")


@pytest.mark.parametrize("name", R.ACTS)
def test_every_derivative(S, name):
    for dtype in DTYPES:
        x, w, b, r = linear_inputs(70, 48, 56, dtype)
        grad, pre = rand(70, 56, dtype=dtype, seed=8), rand(70, 56, dtype=dtype, seed=9, scale=4)
        pre[0, :3] = torch.tensor([0.0, -0.0, 30.0])
        for g, want in zip(S.linear_backward(grad, x, w, pre, name, bias=True),
                           R.linear_backward(grad, x, w, pre, name)):
            R.check(g, want, name)
        x, wg, wu, wd = gated_inputs(70, 48, 56, dtype)
        up, dy = rand(70, 56, dtype=dtype, seed=10), rand(70, 48, dtype=dtype, seed=11)
        for g, want in zip(S.gated_ffn_backward(dy, x, wg, wu, wd, pre, up, name),
                           R.ffn_backward(dy, x, wg, wu, wd, pre, up, name)):
            R.check(g, want, name)


GATED = [(1, 1, 1), (1, 64, 64), (2, 9, 3), (16, 256, 128), (33, 72, 65), (64, 512, 1000),
         (65, 130, 127), (128, 128, 128), (200, 264, 392), (257, 1000, 513), (515, 520, 1032),
         (1024, 256, 768), (2000, 768, 2312), (300, 4096, 520)]


@pytest.mark.parametrize("T,K,F", GATED)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated(S, T, K, F, dtype):
    x, wg, wu, wd = gated_inputs(T, K, F, dtype)
    r = rand(T, K, dtype=dtype, seed=7)
    h, g, u = S.gated_linear_save(x, wg, wu)
    for got, ref, what in zip((h, g, u), R.gated(x, wg, wu), "hgu"):
        R.check(got, ref, what)
    y, g2, u2 = S.gated_ffn_save(x, wg, wu, wd, r)
    R.check(y, R.ffn(x, wg, wu, wd, r), "ffn")
    assert torch.equal(g, g2) and torch.equal(u, u2)
    assert torch.equal(S.gated_ffn(x, wg, wu, wd, r), y)


@pytest.mark.parametrize("T,K,F", GATED)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_backward(S, T, K, F, dtype):
    x, wg, wu, wd = gated_inputs(T, K, F, dtype)
    gate, up = rand(T, F, dtype=dtype, seed=8), rand(T, F, dtype=dtype, seed=9)
    dh, dy = rand(T, F, dtype=dtype, seed=10), rand(T, K, dtype=dtype, seed=11)
    want = R.gated_backward(dh.double(), torch.zeros_like(dh).double(), x, wg, wu, gate, up, "gelu_tanh")[0]
    for got, ref, what in zip(S.gated_linear_backward(dh, x, wg, wu, gate, up, "gelu_tanh"), want,
                              ("dx", "dwg", "dwu")):
        R.check(got, ref, what)
    want = R.ffn_backward(dy, x, wg, wu, wd, gate, up, "silu")
    for got, ref, what in zip(S.gated_ffn_backward(dy, x, wg, wu, wd, gate, up), want,
                              ("dx", "dwg", "dwu", "dwd")):
        R.check(got, ref, "ffn " + what)


def test_calls_of_few_tokens_leave_the_shared_counters_alone(S):
    # h of the few-token block lies in the library's scratch, whose head holds the split
    # products' counters
    x, wg, wu, wd = gated_inputs(200, 1024, 256, torch.float16)
    want = S.gated_ffn(x, wg, wu, wd)
    for T in (1, 7, 32):
        S.gated_ffn(x[:T], wg, wu, wd)
        assert torch.equal(S.gated_ffn(x, wg, wu, wd), want)
