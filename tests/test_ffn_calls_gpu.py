"""Feed-forward operators on the GPU: layouts, masks of padding, scratch, streams, graphs,
threads, and the sizes at which the kernels change."""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest
import torch

import ffn_ref as R
from sion_b200 import abi
from test_ffn_gpu import DTYPES, gated_inputs, linear_inputs, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    import sion_b200
    return sion_b200


@pytest.fixture(autouse=True)
def watchdog():
    yield
    assert abi.watchdog_status(clear=True) == 0


# tokens x depth x features for one shape of tiles each: clusters of 2, 4 and 8 parts of single
# tiles, pairs in parts, wide tiles, several waves from the queue, columns past the last tile
SHAPES = [(128, 2048, 4096), (128, 4096, 4096), (100, 8192, 1024), (256, 4096, 4096),
          (500, 8192, 4096), (4096, 512, 8200), (8192, 512, 5120), (9000, 264, 2056),
          (700, 4096, 130),
          # few tiles and great depth: as many parts as a tile may have
          (256, 16384, 2048), (250, 16000, 1024), (512, 16384, 512), (130, 20000, 256)]


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_linear_shapes(S, T, K, N):
    for dtype in DTYPES:
        x, w, b, r = linear_inputs(T, K, N, dtype)
        for name in ("relu", "gelu"):  # wide tiles take relu, not gelu
            y = S.linear(x, w, b, r, name)
            R.check(y, R.linear(x, w, b, r, name)[0], name)
            assert torch.equal(S.linear(x, w, b, r, name), y)


@pytest.mark.parametrize("T,K,F", [(100, 4096, 1024), (300, 4096, 512), (500, 1024, 4096),
                                   (2100, 512, 5128), (33, 4096, 11264)])
def test_gated_shapes(S, T, K, F):
    for dtype in DTYPES:
        x, wg, wu, wd = gated_inputs(T, K, F, dtype)
        h, g, u = S.gated_linear_save(x, wg, wu, "gelu")
        for got, want in zip((h, g, u), R.gated(x, wg, wu, "gelu")):
            R.check(got, want)
        dy = rand(T, K, dtype=dtype, seed=5)
        got = S.gated_ffn_backward(dy, x, wg, wu, wd, g, u, "gelu")
        for a, want in zip(got, R.ffn_backward(dy, x, wg, wu, wd, g, u, "gelu")):
            R.check(a, want)
        for a, again in zip(got, S.gated_ffn_backward(dy, x, wg, wu, wd, g, u, "gelu")):
            assert torch.equal(a, again)


@pytest.mark.parametrize("T,K,N", [(4200, 512, 4096), (512, 4096, 4096), (130, 1024, 300)])
def test_backward_shapes(S, T, K, N):
    for dtype in DTYPES:
        x, w, b, r = linear_inputs(T, K, N, dtype)
        grad = rand(T, N, dtype=dtype, seed=8)
        got = S.linear_backward(grad, x, w, bias=True)
        for a, want in zip(got, R.linear_backward(grad, x, w)):
            R.check(a, want)
        for a, again in zip(got, S.linear_backward(grad, x, w, bias=True)):
            assert torch.equal(a, again)


@pytest.mark.parametrize("T,K,F", [(479, 128, 8192), (70, 64, 4104), (4100, 72, 184)])
def test_backward_of_very_different_depths(S, T, K, F):
    # gradients of tokens and of weights of which one sums over far more than the other
    for dtype in DTYPES:
        x, wg, wu, wd = gated_inputs(T, K, F, dtype)
        gate, up = (rand(T, F, dtype=dtype, seed=i) for i in (6, 7))
        dy = rand(T, K, dtype=dtype, seed=8)
        got = S.gated_ffn_backward(dy, x, wg, wu, wd, gate, up)
        for a, want in zip(got, R.ffn_backward(dy, x, wg, wu, wd, gate, up)):
            R.check(a, want)
        for a, again in zip(got, S.gated_ffn_backward(dy, x, wg, wu, wd, gate, up)):
            assert torch.equal(a, again)
        got = S.linear_backward(gate, x, wg, bias=True)
        for a, want in zip(got, R.linear_backward(gate, x, wg)):
            R.check(a, want)


# ------------------------------------------------------------------------ layouts
def layouts(t):
    """The same values in other layouts: rows with room behind them, an odd stride, an odd
    address, columns first."""
    n, k = t.shape
    room = torch.full((n, k + 24), float("nan"), dtype=t.dtype, device="cuda")
    room[:, :k] = t
    yield room[:, :k]
    odd = torch.full((n, k + 5), float("nan"), dtype=t.dtype, device="cuda")
    odd[:, 3:3 + k] = t
    yield odd[:, 3:3 + k]
    yield t.t().contiguous().t()


@pytest.mark.parametrize("T", [1, 5, 40, 200])
@pytest.mark.parametrize("dtype", DTYPES)
def test_inputs_of_any_layout(S, T, dtype):
    x, w, b, r = linear_inputs(T, 136, 264, dtype)
    want = R.linear(x, w, b, r, "silu")[0]
    for i, t in enumerate((x, w, r)):
        for v in layouts(t):
            a = [x, w, r]
            a[i] = v
            R.check(S.linear(a[0], a[1], b, a[2], "silu"), want, f"argument {i}")
    x, wg, wu, wd = gated_inputs(T, 136, 264, dtype)
    dy, (h, g, u) = rand(T, 136, dtype=dtype, seed=5), S.gated_linear_save(x, wg, wu)
    want = R.ffn_backward(dy, x, wg, wu, wd, g, u)
    base = [dy, x, wg, wu, wd, g, u]
    for i, t in enumerate(base):
        for v in layouts(t):
            a = list(base)
            a[i] = v
            for got, ref in zip(S.gated_ffn_backward(*a), want):
                R.check(got, ref, f"argument {i}")


def test_leading_dimensions_and_repeated_rows(S):
    x, w, b, r = linear_inputs(24, 64, 72, torch.bfloat16)
    y = S.linear(x, w, b, r)
    assert torch.equal(S.linear(x.view(2, 3, 4, 64), w, b, r.view(2, 3, 4, 72)).view(24, 72), y)
    assert torch.equal(S.linear(x[0], w, b, r[0]), S.linear(x[:1], w, b, r[:1])[0])
    swapped = x.view(4, 6, 64).transpose(0, 1)
    assert torch.equal(S.linear(swapped, w), S.linear(swapped.contiguous(), w))
    for T in (6, 200):  # one row for all tokens: stride 0
        one = x[:1].expand(T, 64)
        R.check(S.linear(one, w, b, r[:1].expand(T, 72)),
                R.linear(one, w, b, r[:1].expand(T, 72))[0])
        grad = r[:1].expand(T, 72)
        for got, want in zip(S.linear_backward(grad, one, w, bias=True), R.linear_backward(grad, one, w)):
            R.check(got, want)


def test_no_tokens(S):
    x, w, b, r = linear_inputs(3, 40, 56, torch.float16)
    assert S.linear(x[:0], w, b, r[:0], "gelu").shape == (0, 56)
    y, pre = S.linear_save(x.view(3, 1, 40)[:0], w)
    assert y.shape == pre.shape == (0, 1, 56)
    dx, dw, db = S.linear_backward(r[:0], x[:0], w, r[:0], "gelu", bias=True)
    assert dx.shape == (0, 40) and dw.shape == w.shape and not dw.any() and not db.any()
    x, wg, wu, wd = gated_inputs(3, 40, 56, torch.float16)
    assert S.gated_ffn(x[:0], wg, wu, wd).shape == (0, 40)
    h = S.gated_linear(x[:0], wg, wu)
    d = S.gated_ffn_backward(x[:0], x[:0], wg, wu, wd, h, h)
    assert d[0].shape == (0, 40) and all(not t.any() and t.shape == w.shape
                                         for t, w in zip(d[1:], (wg, wu, wd)))


def test_what_is_not_wanted(S):
    x, w, b, r = linear_inputs(70, 64, 72, torch.float16)
    grad = rand(70, 72, dtype=torch.float16, seed=1)
    full = S.linear_backward(grad, x, w, bias=True)
    for i, kw in enumerate((dict(need_weight=False), dict(need_x=False), dict(need_x=False, need_weight=False))):
        for bias in (False, True):
            got = S.linear_backward(grad, x, w, bias=bias, **kw)
            for a, f, wanted in zip(got, full, (kw.get("need_x", True), kw.get("need_weight", True), bias)):
                assert torch.equal(a, f) if wanted else a is None
    x, wg, wu, wd = gated_inputs(70, 64, 72, torch.float16)
    h, g, u = S.gated_linear_save(x, wg, wu)
    dy = rand(70, 64, dtype=torch.float16, seed=2)
    full = S.gated_ffn_backward(dy, x, wg, wu, wd, g, u)
    assert torch.equal(S.gated_ffn_backward(dy, x, wg, wu, wd, g, u, need_weights=False)[0], full[0])
    part = S.gated_ffn_backward(dy, x, wg, wu, wd, g, u, need_x=False)
    assert part[0] is None and all(torch.equal(a, f) for a, f in zip(part[1:], full[1:]))
    assert S.gated_linear_backward(h, x, wg, wu, g, u, need_x=False, need_weights=False) == (None,) * 3


def test_refusals(S):
    x, w, b, r = linear_inputs(4, 16, 24, torch.float16)
    wd = rand(16, 24, dtype=torch.float16, seed=1)
    for text, call in [
            ("CUDA", lambda: S.linear(x.cpu(), w)), ("float16 or bfloat16", lambda: S.linear(x.float(), w.float())),
            ("must be Half", lambda: S.linear(x, w.bfloat16())), ("must be \\[out, 16\\]", lambda: S.linear(x, w[:, :8])),
            ("2D", lambda: S.linear(x, w[0])), ("one entry per", lambda: S.linear(x, w, b[:5])),
            ("shape", lambda: S.linear(x, w, b, r[:2])), ("unknown activation", lambda: S.linear(x, w, activation="elu")),
            ("not empty", lambda: S.linear(x[:, :0], w[:, :0])), ("not be empty", lambda: S.linear(x, w[:0])),
            ("linear_save", lambda: S.linear_backward(r, x, w, None, "gelu")),
            ("shape", lambda: S.linear_backward(r[:, :8], x, w)),
            ("w_up must be", lambda: S.gated_linear(x, w, w[:8])),
            ("w_down must be", lambda: S.gated_ffn(x, w, w, w)),
            ("shape", lambda: S.gated_ffn(x, w, w, wd, r)),
            ("shape", lambda: S.gated_ffn_backward(x, x, w, w, wd, r, r[:2]))]:
        with pytest.raises(RuntimeError, match=text):
            call()


# ------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("T", [3, 30, 150, 600])
def test_rows_do_not_mix(S, T):
    x, w, b, r = linear_inputs(T, 256, 200, torch.bfloat16)
    clean = S.linear(x, w, b, r, "gelu")
    bad = x.clone()
    bad[0, 5], bad[T // 2, 7] = float("nan"), float("inf")
    y = S.linear(bad, w, b, r, "gelu")
    rows = torch.tensor([i for i in range(T) if i not in (0, T // 2)], device="cuda")
    assert torch.equal(y[rows], clean[rows])
    assert y[0].isnan().all() and not y[T // 2].isfinite().any()
    assert S.linear(bad, w, None, None, "relu")[0].isnan().all()  # relu keeps what is not a number


def test_padding_is_not_read(S):
    # rows behind the last token and columns behind the last feature hold anything
    T, K, N = 130, 72, 104
    x, w, b, r = linear_inputs(T, K, N, torch.float16)
    wide = [torch.full((t.shape[0] + 200, t.shape[1] + 64), float("nan"), dtype=t.dtype, device="cuda")
            for t in (x, w, r)]
    for big, t in zip(wide, (x, w, r)):
        big[:t.shape[0], :t.shape[1]] = t
    xs, ws, rs = [big[:t.shape[0], :t.shape[1]] for big, t in zip(wide, (x, w, r))]
    assert torch.equal(S.linear(xs, ws, b, rs), S.linear(x, w, b, r))
    for a, c in zip(S.linear_backward(rs, xs, ws, rs, "silu", bias=True),
                    S.linear_backward(r, x, w, r, "silu", bias=True)):
        assert torch.equal(a, c)


# ------------------------------------------------------------------------- the C ABI
def test_outputs_with_strides_aliases_and_scratch(S):
    for T, K, N, pad in ((5, 64, 40, 3), (50, 64, 40, 8), (300, 96, 200, 16), (300, 96, 203, 1)):
        x, w, b, r = linear_inputs(T, K, N, torch.float16)
        want = S.linear(x, w, b, r, "gelu")
        room = torch.full((T, N + pad), 7.0, dtype=torch.float16, device="cuda")
        room[:, :N] = r
        out = room[:, :N]  # the residual itself
        a = abi.linear_args(T, K, N, abi.F16, "gelu", x=x, weight=w, residual=out, bias=b, out=out)
        scratch = torch.full((abi.ffn_workspace_size("linear", a) + 256,), 255, dtype=torch.uint8, device="cuda")
        scratch = scratch[-scratch.data_ptr() % 256:]
        abi.ffn_call("linear", a, scratch[:abi.ffn_workspace_size("linear", a)] if len(scratch) > 256 else None)
        R.check(out, R.linear(x, w, b, r, "gelu")[0])
        assert (out - want).abs().max() == 0 and (room[:, N:] == 7).all()


def test_scratch_of_a_caller(S):
    T, K, F = 700, 264, 504
    x, wg, wu, wd = gated_inputs(T, K, F, torch.bfloat16)
    h, g, u = S.gated_linear_save(x, wg, wu)
    dy = rand(T, K, dtype=torch.bfloat16, seed=3)
    want = S.gated_ffn_backward(dy, x, wg, wu, wd, g, u)
    out = [torch.empty_like(t) for t in want]
    a = abi.gated_args(T, K, F, abi.BF16, x=x, w_gate=wg, w_up=wu, w_down=wd, gate=g, up=u, grad=dy,
                       dx=out[0], dw_gate=out[1], dw_up=out[2], dw_down=out[3])
    need = abi.ffn_workspace_size("gated_ffn_bwd", a)
    assert need >= 3 * T * F * 2
    scratch = torch.full((need + 4096,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(2):  # with any contents, again and again
        abi.ffn_call("gated_ffn_bwd", a, scratch[:need])
        assert all(torch.equal(o, t) for o, t in zip(out, want))
    assert (scratch[need:] == 255).all()
    with pytest.raises(abi.FelixError, match="too small"):
        abi.ffn_call("gated_ffn_bwd", a, scratch[:need - 1])
    few = abi.linear_args(1, K, F, abi.BF16, x=x, weight=wg, out=h)
    assert abi.ffn_workspace_size("linear", few) == 0


def test_offsets_past_31_bits(S):
    # 2^31 elements and more in an output, a weight and a residual
    T, K, N = 66000, 64, 33000
    x, w = rand(T, K, dtype=torch.bfloat16, seed=1), rand(N, K, dtype=torch.bfloat16, seed=2, scale=0.1)
    y = S.linear(x, w, None, None, "silu")
    for rows in (slice(0, 40), slice(T // 2, T // 2 + 40), slice(T - 40, T)):
        R.check(y[rows], R.linear(x[rows], w, None, None, "silu")[0])
    z = S.linear(x, w, None, y)
    R.check(z[-40:], R.linear(x[-40:], w, None, y[-40:])[0])
    del z
    dx, dw, _ = S.linear_backward(y, x, w)
    R.check(dx[-40:], R.linear_backward(y[-40:], x[-40:], w)[0])
    del y, dx, dw
    N, K = 530000, 4096  # 2.2e9 weights, few tokens
    w = torch.empty(N, K, dtype=torch.float16, device="cuda").normal_(0, 0.02)
    for T in (1, 20):
        x = rand(T, K, dtype=torch.float16, seed=T)
        y = S.linear(x, w)
        for n in (0, N // 2, N - 64):
            R.check(y[:, n:n + 64], R.linear(x, w[n:n + 64])[0])


# ----------------------------------------------------------------- streams and graphs
def test_side_streams_and_threads(S):
    x, w, b, r = linear_inputs(900, 520, 1032, torch.float16)
    xg, wg, wu, wd = gated_inputs(900, 520, 1032, torch.float16)
    h, g, u = S.gated_linear_save(xg, wg, wu)
    dy = rand(900, 520, dtype=torch.float16, seed=4)
    want = S.linear(x, w, b, r, "gelu"), S.gated_ffn_backward(dy, xg, wg, wu, wd, g, u)
    torch.cuda.synchronize()
    errors = []

    def work():
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    y, d = S.linear(x, w, b, r, "gelu"), S.gated_ffn_backward(dy, xg, wg, wu, wd, g, u)
                s.synchronize()
            assert torch.equal(y, want[0]) and all(torch.equal(a, c) for a, c in zip(d, want[1]))
        except Exception as e:  # noqa: BLE001 (shown below)
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors


def capture(f):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = f()
    return g, out


def test_captured_and_replayed(S):
    T, K, F = 600, 264, 1000
    x, wg, wu, wd = gated_inputs(T, K, F, torch.bfloat16)
    static = x.clone()

    def step():
        y, g, u = S.gated_ffn_save(static, wg, wu, wd, static)
        return (y, *S.gated_ffn_backward(y, static, wg, wu, wd, g, u))

    graphs = [capture(step) for _ in range(2)]  # of two graphs each has scratch of its own
    for seed in (1, 2):
        static.copy_(rand(T, K, dtype=torch.bfloat16, seed=seed))
        want = step()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(5):
                    g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_a_backward_pass_is_captured_while_an_eager_graph_of_its_leaves_lives(S):
    x, w, b, r = linear_inputs(300, 128, 256, torch.float16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    eager = S.linear_autograd(*leaves, None, "gelu")
    grad = rand(300, 256, dtype=torch.float16, seed=6)

    def step():
        y, pre = S.linear_save(x, w, b, None, "gelu")
        return (y, *S.linear_backward(grad, x, w, pre, "gelu", bias=True))

    g, out = capture(step)
    g.replay()
    eager.backward(grad)
    torch.cuda.synchronize()
    assert torch.equal(out[0], eager)
    for leaf, d in zip(leaves, out[1:]):
        assert torch.equal(leaf.grad, d)


# --------------------------------------------------------------------------- autograd
@pytest.mark.parametrize("T", [6, 150])
def test_autograd(S, T):
    dtype = torch.bfloat16
    x, w, b, r = [t.requires_grad_() for t in linear_inputs(T, 72, 88, dtype)]
    grad = rand(T, 88, dtype=dtype, seed=6)
    y = S.linear_autograd(x, w, b, r, "silu")
    y.backward(grad)
    pre = S.linear_save(x.detach(), w.detach(), b.detach())[1]
    for t, want in zip((x, w, b), R.linear_backward(grad, x.detach(), w.detach(), pre, "silu")):
        R.check(t.grad, want)
    assert torch.equal(r.grad, grad)
    # only what is asked for, a gradient with stride 0, a plain layer
    y = S.linear_autograd(x.detach(), w, None, None)
    (dw,) = torch.autograd.grad(y.sum(), w)
    R.check(dw, R.linear_backward(torch.ones_like(y), x.detach(), w.detach())[1])
    x, wg, wu, wd = [t.requires_grad_() for t in gated_inputs(T, 72, 88, dtype)]
    dy = rand(T, 72, dtype=dtype, seed=7)
    y = S.gated_ffn_autograd(x, wg, wu, wd, x, "gelu")
    y.backward(dy)
    d = [t.detach() for t in (x, wg, wu, wd)]
    _, g, u = S.gated_linear_save(*d[:3], "gelu")
    want = S.gated_ffn_backward(dy, *d, g, u, "gelu")
    assert torch.equal(x.grad, want[0] + dy)  # through the block and the residual
    assert all(torch.equal(t.grad, v) for t, v in zip((wg, wu, wd), want[1:]))
    h = S.gated_linear_autograd(x, wg, wu)
    assert torch.autograd.grad(h.float().square().sum(), wg)[0].isfinite().all()
    with pytest.raises(RuntimeError, match="once_differentiable|twice|backward"):
        y = S.linear_autograd(x, wg)
        (dx,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        dx.float().sum().backward()


def test_arguments_of_the_binding_stay_as_they_are(S):
    # the C ABI reads its arguments before it returns: they may be reused at once
    x, w, b, r = linear_inputs(40, 64, 72, torch.float16)
    y = torch.empty(40, 72, dtype=torch.float16, device="cuda")
    a = abi.linear_args(40, 64, 72, abi.F16, x=x, weight=w, out=y)
    abi.ffn_call("linear", a)
    C.memset(C.byref(a), 255, C.sizeof(a))
    assert torch.equal(y, S.linear(x, w))


def test_calls_that_follow_one_another(S):
    """Each call reads what the one before wrote, into memory that earlier ones read: the same
    bits whether the calls are apart, follow at once, change streams or are replayed."""
    dtype = torch.bfloat16
    K, F = 512, 2304
    w = [rand(K, K, dtype=dtype, seed=i, scale=K ** -0.5) for i in range(4)]
    up = [rand(F, K, dtype=dtype, seed=i, scale=K ** -0.5) for i in range(2)]
    down = rand(K, F, dtype=dtype, seed=5, scale=F ** -0.5)
    odd = rand(K, K + 1, dtype=dtype, seed=6, scale=K ** -0.5)[:, 1:]  # copied for TMA
    start = rand(700, K, dtype=dtype, seed=7)
    other = torch.cuda.Stream()

    def chain(between):
        kept, a = [], start.clone()
        for i, n in enumerate([1, 7, 33, 64, 200, 700, 40, 3]):
            b = S.linear(a[:n], w[i % 4])
            between()
            b = S.linear(b, odd, residual=a[:n], activation="gelu")
            between()
            b = S.gated_ffn(b, *up, down, residual=b)
            between()
            if i % 2:
                b.mul_(0.5)
            y, pre = S.linear_save(b, w[1], activation="silu")
            between()
            grads = S.linear_backward(y, b, w[1], pre, "silu", bias=True)
            between()
            a[:n].copy_(S.linear(grads[0], w[2]))
            kept += [y, *grads]
        return [*kept, a]

    def move():
        here = torch.cuda.current_stream()
        other.wait_stream(here)
        with torch.cuda.stream(other):
            start.add_(0)
        here.wait_stream(other)

    want = chain(torch.cuda.synchronize)
    assert all(torch.isfinite(t).all() and t.abs().max() > 0 for t in want)
    for between in (lambda: None, move):
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(want, chain(between)))
    graph, out = capture(lambda: chain(lambda: None))
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.parametrize("T", [2, 40, 300])
def test_captured_with_branches(S, T):
    """Calls behind fills, copies, other kernels and joined streams, captured."""
    dtype, K = torch.bfloat16, 512
    x = rand(T, K, dtype=dtype, seed=1)
    w = [rand(K, K, dtype=dtype, seed=i, scale=K ** -0.5) for i in range(3)]
    side = torch.cuda.Stream()

    def f():
        here = torch.cuda.current_stream()
        a = S.linear(x, w[0], activation="silu")
        side.wait_stream(here)
        with torch.cuda.stream(side):
            b = torch.zeros_like(a)
            b = S.linear(b, w[1], residual=a)
            c = S.linear(b, w[2])
        d = S.gated_linear(a, w[1], w[2])
        here.wait_stream(side)
        e = S.linear(c, w[0], residual=d)
        y = e.clone()
        y.zero_()
        y.copy_(e)
        y = S.gated_ffn(y, w[0], w[1], w[2], residual=b)
        for t in (a, b, c):
            t.record_stream(here)
        return a, b, c, d, e, y

    want = f()
    torch.cuda.synchronize()
    graph, out = capture(f)
    for _ in range(5):
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


FIRST_CALL = """
import torch, sion_b200 as S
r = lambda *s: torch.randn(*s, device="cuda").bfloat16() / 16
x, wg, wu, wd, dy = r({T}, 512), r(1024, 512), r(1024, 512), r(512, 1024), r({T}, 512)
odd = r(1024, 513)[:, 1:]
def f():
    y, g, u = S.gated_ffn_save(x, wg, wu, wd, x)
    z, pre = S.linear_save(y, odd, activation="gelu")
    return (y, z, *S.gated_ffn_backward(dy, x, wg, wu, wd, g, u),
            *S.linear_backward(z, y, odd, pre, "gelu", True))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = f()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, f()))
"""


@pytest.mark.parametrize("T", [1, 300])
def test_the_first_call_of_a_process_is_captured(T):
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
    r = subprocess.run([sys.executable, "-c", FIRST_CALL.replace("{T}", str(T))], cwd=root,
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
