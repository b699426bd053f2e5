"""The counters at the head of the library's scratch stay zero between calls: calls that rely on
them (tiles from the queue: the last two; the bias gradient's sums: the first ones) give
the same bits after any call whose own data lie behind the counters."""
import pytest
import torch

from test_ffn_gpu import DTYPES, gated_inputs, linear_inputs, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    import sion_b200
    return sion_b200


@pytest.mark.parametrize("dtype", DTYPES)
def test_calls_in_turn_leave_the_counters_at_zero(S, dtype):
    # 8192 x 512 -> 5120: 320 tiles or more for 74 pairs, so that they come from the queue
    x, w, b, r = linear_inputs(8192, 512, 5120, dtype)
    grad = rand(8192, 5120, dtype=dtype, seed=9)
    xs, ws, _, _ = linear_inputs(700, 72, 4104, dtype)
    gs = rand(700, 4104, dtype=dtype, seed=8)

    def readers():
        return (S.linear(x, w, b, r, "relu"), S.linear(x, w, b, None, "gelu"),
                S.linear_backward(grad, x, w, bias=True)[2], *S.linear_backward(gs, xs, ws, bias=True))

    want = readers()
    # h of the block lies behind the counters: 7 x 11264 values are ten times as long as they
    xg, wg, wu, wd = gated_inputs(300, 512, 11264, dtype)
    odd = rand(300, 513, dtype=dtype, seed=7)[:, 1:]
    gate, up = (rand(300, 11264, dtype=dtype, seed=i) for i in (5, 6))
    for T in (1, 7, 20, 64, 300):
        for call in (lambda: S.gated_ffn(xg[:T], wg, wu, wd),
                     lambda: S.linear(odd[:T], wg),
                     lambda: S.gated_ffn_backward(xg[:T], xg[:T], wg, wu, wd, gate[:T], up[:T]),
                     lambda: S.gated_linear_backward(gate[:T], odd[:T], wg, wu, gate[:T], up[:T])):
            call()
            assert all(torch.equal(a, c) for a, c in zip(readers(), want)), T
