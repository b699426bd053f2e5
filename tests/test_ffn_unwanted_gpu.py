"""Backward passes of which not all gradients are wanted: the same bits for those that are, and
neither memory nor launches for what nobody reads."""
import pytest
import torch

from sion_b200 import abi
from test_ffn_gpu import DTYPES, gated_inputs, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def S():
    import sion_b200
    return sion_b200


@pytest.mark.parametrize("T,K,F", [(5, 64, 72), (70, 130, 127), (128, 4096, 256), (300, 4096, 512),
                                   (2100, 512, 5128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_any_choice_of_gradients(S, T, K, F, dtype):
    x, wg, wu, wd = gated_inputs(T, K, F, dtype)
    gate, up = (rand(T, F, dtype=dtype, seed=i) for i in (6, 7))
    dy, dh = rand(T, K, dtype=dtype, seed=8), rand(T, F, dtype=dtype, seed=9)
    names = ("dx", "dw_gate", "dw_up", "dw_down")
    shapes = (x, wg, wu, wd)
    code = abi.F16 if dtype == torch.float16 else abi.BF16
    for call, grad, want in (
            ("gated_ffn_bwd", dy, S.gated_ffn_backward(dy, x, wg, wu, wd, gate, up)),
            ("gated_linear_bwd", dh, S.gated_linear_backward(dh, x, wg, wu, gate, up))):
        for choice in range(1, 1 << len(want)):
            out = {n: torch.full_like(t, float("nan"))
                   for i, (n, t) in enumerate(zip(names, shapes)) if choice >> i & 1}
            a = abi.gated_args(T, K, F, code, x=x, w_gate=wg, w_up=wu, gate=gate, up=up, grad=grad,
                               **({"w_down": wd} if call == "gated_ffn_bwd" else {}), **out)
            abi.ffn_call(call, a)
            # (dx and a weight's gradient may be cut in depth otherwise in other company)
            for n, t in out.items():
                full = want[names.index(n)]
                assert (t.double() - full.double()).norm() <= 4 * torch.finfo(dtype).eps * full.double().norm()


def test_scratch_is_for_what_is_wanted():
    T, K, F = 512, 256, 1024
    t = torch.empty(1024, 1024, dtype=torch.float16, device="cuda")

    def size(call, *wanted):
        fields = {n: t for n in ("x", "w_gate", "w_up", "w_down", "gate", "up", "grad", *wanted)}
        if call == "gated_linear_bwd":
            del fields["w_down"]
        return abi.ffn_workspace_size(call, abi.gated_args(T, K, F, abi.F16, **fields))

    one = T * F * 2
    front = size("gated_linear_bwd", "dx") - 2 * one
    assert 0 < front <= 65536
    assert size("gated_ffn_bwd", "dx") == size("gated_ffn_bwd", "dw_up") == front + 2 * one
    assert size("gated_ffn_bwd", "dx", "dw_down") == front + 3 * one
    assert size("gated_ffn_bwd") == size("gated_linear_bwd") == 0


def test_no_gradient_needs_no_launch(S):
    x, wg, wu, wd = gated_inputs(300, 128, 256, torch.bfloat16)
    h, gate, up = S.gated_linear_save(x, wg, wu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.warns(UserWarning, match="empty"):  # nothing was recorded
        with torch.cuda.graph(graph):
            assert S.gated_ffn_backward(x, x, wg, wu, wd, gate, up, need_x=False,
                                        need_weights=False) == (None,) * 4
            assert S.gated_linear_backward(h, x, wg, wu, gate, up, need_x=False,
                                           need_weights=False) == (None,) * 3
            assert S.linear_backward(h, x, wg, gate, "silu", need_x=False,
                                     need_weight=False) == (None,) * 3
