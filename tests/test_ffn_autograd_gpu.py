"""The feed-forward operators under torch.autograd keep and write only what a backward pass
will read: calls without a gradient are the plain ones, inputs whose partner is frozen may
be changed after the call."""
import pytest
import torch

import ffn_ref as R
from test_ffn_gpu import gated_inputs, linear_inputs, rand

pytestmark = pytest.mark.gpu
DT = torch.bfloat16


@pytest.fixture(scope="module")
def S():
    import sion_b200
    return sion_b200


def test_without_a_gradient_nothing_is_saved(S, monkeypatch):
    x, w, b, r = linear_inputs(70, 72, 88, DT)
    xg, wg, wu, wd = gated_inputs(70, 72, 88, DT)
    want = S.linear(x, w, b, r, "gelu"), S.gated_linear(xg, wg, wu), S.gated_ffn(xg, wg, wu, wd, xg)

    def never(*a, **k):
        raise AssertionError("saved for nobody")

    for name in ("linear_save", "gated_linear_save", "gated_ffn_save"):
        monkeypatch.setattr(S, name, never)

    def calls():
        return (S.linear_autograd(x, w, b, r, "gelu"), S.gated_linear_autograd(xg, wg, wu),
                S.gated_ffn_autograd(xg, wg, wu, wd, xg))

    for got in (calls(),):  # no input needs one
        assert all(torch.equal(a, c) and not a.requires_grad for a, c in zip(got, want))
    leaves = [t.requires_grad_() for t in (x, w, xg, wg)]
    with torch.no_grad():
        assert all(torch.equal(a, c) and not a.requires_grad for a, c in zip(calls(), want))
    [t.requires_grad_(False) for t in leaves]
    # the residual's gradient alone: the one that comes in
    for f, args in ((S.linear_autograd, (x, w, b)), (S.gated_ffn_autograd, (xg, wg, wu, wd))):
        res = rand(70, 88 if f is S.linear_autograd else 72, dtype=DT, seed=3).requires_grad_()
        y = f(*args, res, "gelu")
        grad = rand(*y.shape, dtype=DT, seed=4)
        y.backward(grad)
        assert torch.equal(res.grad, grad)


def held(y):
    return sum(t.numel() for t in y.grad_fn.saved_tensors if t is not None)


@pytest.mark.parametrize("T", [6, 150])
@pytest.mark.parametrize("shape", [(), (2,)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_linear_with_any_inputs_frozen(S, T, shape, act):
    K, N = 72, 88
    x, w, b, r = linear_inputs(T, K, N, DT)
    grad = rand(T, N, dtype=DT, seed=6)
    pre = S.linear_save(x, w, b)[1]
    want = R.linear_backward(grad, x, w, pre, act)
    lead = (*shape, T // 2) if shape else (T,)
    for choice in range(1, 8):
        leaves = [t.clone() for t in (x, w, b)]
        for i, t in enumerate(leaves):
            t.requires_grad_(bool(choice >> i & 1))
        lx, lw, lb = leaves
        y = S.linear_autograd(lx.view(*lead, K), lw, lb, r.view(*lead, N), act)
        size = (T * K if lw.requires_grad else 0) + (N * K if lx.requires_grad else 0)
        assert held(y) == size + (T * N if act != "none" else 0)
        with torch.no_grad():  # nobody reads these any more
            if not lw.requires_grad:
                lx.fill_(float("nan"))
            if not lx.requires_grad:
                lw.fill_(float("nan"))
        y.backward(grad.view(*lead, N))
        for t, v in zip(leaves, want):
            if t.requires_grad:
                R.check(t.grad, v)
            else:
                assert t.grad is None


@pytest.mark.parametrize("T", [6, 150])
def test_gated_with_any_inputs_frozen(S, T):
    K, F = 72, 88
    inputs = gated_inputs(T, K, F, DT)
    dy, dh = rand(T, K, dtype=DT, seed=6), rand(T, F, dtype=DT, seed=7)
    _, gate, up = S.gated_linear_save(*inputs[:3])
    for f, n, grad, want in (
            (S.gated_ffn_autograd, 4, dy, R.ffn_backward(dy, *inputs, gate, up)),
            (S.gated_linear_autograd, 3, dh,
             R.gated_backward(dh.double(), torch.zeros_like(dh).double(), *inputs[:3], gate, up, "silu")[0])):
        for choice in range(1, 1 << n):
            leaves = [t.clone() for t in inputs[:n]]
            for i, t in enumerate(leaves):
                t.requires_grad_(bool(choice >> i & 1))
            x, weights = leaves[0], leaves[1:]
            y = f(x.view(2, T // 2, K), *weights)
            any_weight = any(t.requires_grad for t in weights)
            size = 2 * T * F + (T * K if any_weight else 0) + \
                (2 * F * K if x.requires_grad else 0) + (K * F if n == 4 else 0)
            assert held(y) == size
            with torch.no_grad():
                if not any_weight:
                    x.fill_(float("nan"))
                if not x.requires_grad:
                    weights[0].fill_(float("nan")), weights[1].fill_(float("nan"))
            y.backward(grad.view_as(y))
            for t, v in zip(leaves, want):
                if t.requires_grad:
                    R.check(t.grad, v)
                else:
                    assert t.grad is None


def test_no_tokens(S):
    x, w, b, _ = linear_inputs(3, 40, 56, DT)
    for need in ((x,), (w, b), (x, w, b)):
        [t.requires_grad_(any(t is n for n in need)) for t in (x, w, b)]
        (S.linear_autograd(x[:0], w, b, None, "gelu").sum()).backward()
        for t in need:
            assert not t.grad.any()
            t.grad = None
