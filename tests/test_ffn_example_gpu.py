"""examples/ffn_block.py runs the feed-forward operators with attention, forward and
backward, as a training step does."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import ffn_block
    finally:
        sys.path.pop(0)
    return ffn_block


def test_example_runs_and_repeats():
    ex = _example()
    a, p = ex.train(steps=3, batch=2, tokens=70)
    b, _ = ex.train(steps=3, batch=2, tokens=70)
    assert len(a) == 3 and all(v == v and v < float("inf") for v in a)
    assert a[0] == b[0]  # (attention adds up dQ in no fixed order: later steps may differ)
    x = torch.randn(5, ex.WIDTH, device="cuda").half()
    with torch.no_grad():
        together = ex.feed_forward_token(p, x)
        for i in range(5):
            assert torch.equal(ex.feed_forward_token(p, x[i:i + 1])[0], together[i])


def test_gradients_against_elementary_operations():
    # The block's gradients against the same formulas in 64 bits. In 16 bits some 12 values in
    # a row are rounded on the way from an input through the block and back (norm, qkv, the
    # probabilities, attention, out, norm, gate, up, h, and their gradients), each by 2^-11
    # at most: 12 x 2^-11 = 0.6 % of the gradient's norm if all went one way.
    ex = _example()
    p = {k: v.requires_grad_() for k, v in ex.weights(5).items()}
    exact = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(2, 130, ex.WIDTH, device="cuda", generator=g).half().requires_grad_()
    x64 = x.detach().double().requires_grad_()
    dy = torch.randn(2, 130, ex.WIDTH, device="cuda", generator=g).half()
    y, y64 = ex.block(p, x), _in_64(ex, exact, x64)
    assert (y.double() - y64).norm() <= 12 * 2.0 ** -11 * y64.norm()
    y.backward(dy)
    y64.backward(dy.double())
    for a, b in [(x, x64)] + [(p[k], exact[k]) for k in p]:
        assert (a.grad.double() - b.grad).norm() <= 12 * 2.0 ** -11 * b.grad.norm()


def _in_64(ex, p, x):
    keep, ex.norm = ex.norm, lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)
    try:
        return ex.plain_block(p, x)
    finally:
        ex.norm = keep
