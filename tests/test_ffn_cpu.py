"""Feed-forward operators: what is refused, before any device work, and the tests' own
formulas (their derivatives against differences)."""
import ctypes as C
import os
import re

import pytest
import torch

import ffn_ref as R
from sion_b200 import abi

CALLS = ("linear", "linear_bwd", "gated_linear", "gated_linear_bwd", "gated_ffn", "gated_ffn_bwd")
P = 0x10000  # an address that is never used


def args(call, **kw):
    linear = call.startswith("linear")
    a = (abi.LinearArgs if linear else abi.GatedArgs)(4, 16, 24, abi.F16, 4)
    names = [n for n, t in a._fields_ if t is abi.Matrix]
    for n in names:
        setattr(a, n, abi.Matrix(P, 64))
    if call == "gated_linear":
        a.residual = abi.Matrix(None, 0)
    if call == "gated_linear_bwd":
        a.dw_down = abi.Matrix(None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(call, text, workspace=None, **kw):
    L, a = abi.lib(), args(call, **kw)
    rc = getattr(L, "felix_" + call)(C.byref(a), workspace, 0, None)
    assert rc == abi.API_ERROR and text in L.felix_last_error_message().decode(), (call, text)


@pytest.mark.parametrize("call", CALLS)
def test_types_and_sizes(call):
    size = "in_features" if call.startswith("linear") else "features"
    other = "out_features" if call.startswith("linear") else "hidden"
    refused(call, "fp16 or bf16", dtype=abi.F32)
    refused(call, "fp16 or bf16", dtype=-1)
    refused(call, "activation", activation=6)
    refused(call, "activation", activation=-1)
    for f in (size, other):
        refused(call, "features must be", **{f: 0})
        refused(call, "features must be", **{f: (1 << 30) + 1})
    refused(call, "at most 2^30", tokens=(1 << 30) + 1)
    refused(call, "256-byte aligned", workspace=P + 16)
    rc = getattr(abi.lib(), "felix_" + call)(None, None, 0, None)
    assert rc == abi.API_ERROR


NEEDED = {"linear": ("x", "weight", "out"), "linear_bwd": ("grad", "x", "weight", "pre"),
          "gated_linear": ("x", "w_gate", "w_up", "out"),
          "gated_linear_bwd": ("grad", "gate", "up", "x", "w_gate", "w_up"),
          "gated_ffn": ("x", "w_gate", "w_up", "w_down", "out"),
          "gated_ffn_bwd": ("grad", "gate", "up", "x", "w_gate", "w_up", "w_down")}
OUTPUTS = {"linear": ("out", "pre"), "linear_bwd": ("dx", "dweight"),
           "gated_linear": ("out", "gate", "up"), "gated_linear_bwd": ("dx", "dw_gate", "dw_up"),
           "gated_ffn": ("out", "gate", "up"),
           "gated_ffn_bwd": ("dx", "dw_gate", "dw_up", "dw_down")}


@pytest.mark.parametrize("call", CALLS)
def test_matrices(call):
    for name in NEEDED[call]:
        text = "needs pre" if name == "pre" else "null pointer"
        refused(call, text, **{name: abi.Matrix(None, 0)})
        refused(call, "2-byte aligned", **{name: abi.Matrix(P + 1, 64)})
        refused(call, "not be negative", **{name: abi.Matrix(P, -64)})
    for name in OUTPUTS[call]:
        refused(call, "overlap", **{name: abi.Matrix(P, 15)})
    if call == "gated_linear":
        refused(call, "no residual", residual=abi.Matrix(P, 64))
    if call == "gated_linear_bwd":
        refused(call, "no down projection", dw_down=abi.Matrix(P, 64))
    if call == "linear":
        refused(call, "2-byte aligned", bias=P + 1)
    if call == "linear_bwd":
        refused(call, "2-byte aligned", dbias=P + 1)


def test_workspace_size_checks_the_same():
    n = C.c_size_t()
    for call in CALLS:
        a, back = args(call, dtype=9), int(call.endswith("_bwd"))
        if call.startswith("linear"):
            rc = abi.lib().felix_linear_workspace_size(C.byref(a), back, C.byref(n))
        else:
            rc = abi.lib().felix_gated_workspace_size(C.byref(a), int("ffn" in call), back, C.byref(n))
        assert rc == abi.API_ERROR


def test_the_header_and_the_binding_agree_on_the_structures():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(os.path.dirname(abi.__file__), "..", "include",
                                                      "felix_c.h")).read(), flags=re.S)
    for cls, name in ((abi.LinearArgs, "felix_linear_args"), (abi.GatedArgs, "felix_gated_args")):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        fields = []
        for line in body.split(";"):
            words = line.replace("const ", "").split(None, 1)
            if len(words) == 2:
                fields += [f.strip().lstrip("*") for f in words[1].split(",")]
        assert fields == [f for f, _ in cls._fields_]


@pytest.mark.parametrize("name", R.ACTS)
def test_derivatives_against_differences(name):
    z = torch.linspace(-6, 6, 481, dtype=torch.float64) + 1e-3
    h = 1e-6
    want = (R.act(name, z + h)[0] - R.act(name, z - h)[0]) / (2 * h)
    assert (R.act(name, z)[1] - want).abs().max() < 1e-8
    assert R.act(name, z)[1].abs().max() <= R.SLOPE


def central(f, t, grad, h=1e-6):
    """d sum(grad f) / dt by central differences, entry by entry."""
    out = torch.empty_like(t)
    for i in range(t.numel()):
        e = torch.zeros_like(t).flatten()
        e[i] = h
        e = e.view_as(t)
        out.view(-1)[i] = ((f(t + e) - f(t - e)) * grad).sum() / (2 * h)
    return out


@pytest.mark.parametrize("name", ["none", "gelu", "silu"])
def test_gradients_against_differences(name):
    # in 64 bits throughout: bfloat16's rounding is switched off by a type that has none here
    R.HALF[torch.float64], R.TINY[torch.float64] = 0.0, 0.0
    g = torch.Generator().manual_seed(3)

    def rand(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    x, w, b, dy = rand(3, 4), rand(5, 4), rand(5), rand(3, 5)
    pre = R.linear(x, w, b)[0][0]
    got = [v for v, _ in R.linear_backward(dy, x, w, pre, name)]
    f = lambda x, w, b: R.linear(x, w, b, None, name)[0][0]  # noqa: E731
    want = [central(lambda t: f(t, w, b), x, dy), central(lambda t: f(x, t, b), w, dy),
            central(lambda t: f(x, w, t), b, dy)]
    for a, c in zip(got, want):
        assert (a - c).abs().max() < 1e-7
    wg, wu, wd, dy = rand(6, 4), rand(6, 4), rand(4, 6), rand(3, 4)
    gate, up = x @ wg.t(), x @ wu.t()
    got = [v for v, _ in R.ffn_backward(dy, x, wg, wu, wd, gate, up, name)]
    f = lambda *t: R.ffn(*t, None, name)[0]  # noqa: E731
    want = [central(lambda t: f(t, wg, wu, wd), x, dy), central(lambda t: f(x, t, wu, wd), wg, dy),
            central(lambda t: f(x, wg, t, wd), wu, dy), central(lambda t: f(x, wg, wu, t), wd, dy)]
    for a, c in zip(got, want):
        assert (a - c).abs().max() < 1e-6
    del R.HALF[torch.float64], R.TINY[torch.float64]


def test_every_wait_of_a_warp_is_agreed_on():
    # a wait that gives up may do so in some lanes only: where a whole warp waits, its lanes
    # vote before they go on (the producers wait in one lane)
    csrc = os.path.join(os.path.dirname(abi.__file__), "csrc")
    for name in ("ffn_product_sm100.cu", "ffn_narrow_sm100.cu", "ffn_finish.cuh"):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(csrc, name)).read())
        for m in re.finditer(r"\bmbar_sleep_wait\(", text):
            before = text[max(0, m.start() - 60):m.start()]
            arguments = text[m.end():m.end() + 120]
            assert "__all_sync(~0u," in before or "kWdProducerEmpty" in arguments, (name, before)
