"""Feed-forward operators without a GPU: what the sources have to hold where it is not provoked
on a device, and calls that are neither refused for what they do not read nor end the
process."""
import os
import re
import subprocess

import pytest

from sion_b200 import abi
from test_ffn_cpu import P, args

CSRC = os.path.join(os.path.dirname(abi.__file__), "csrc")


def code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_a_cta_waits_for_what_the_others_send_even_after_it_gave_up():
    # Every CTA of a cluster sends its shares after the barrier, whatever happened before.
    # The wait for them is bounded by its own time alone: one that ended because of a flag set
    # earlier would let the CTA exit while copies into its memory are under way.
    text = code("ffn_finish.cuh")
    waits = re.findall(r"\bmbar_\w*wait\(([^;]*?)\)", text, re.S)
    assert len(waits) == 1 and waits[0].startswith("received, 0, &none,") and "abort" not in text
    assert "int none = 0;" in text


def test_refusals_without_memory(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = str(tmp_path / "no_memory_test")
    r = subprocess.run(["g++", "-std=c++20", "-O1", os.path.join(root, "tests", "cpp", "no_memory_test.cpp"),
                        f"-I{root}/include", f"-L{root}/sion_b200", "-lfelix_b200",
                        f"-Wl,-rpath,{root}/sion_b200", "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout + r.stderr


# Matrices that a call does not read: of the other direction, of the other operator, of a
# gradient that is not wanted.
UNREAD = [("linear", "grad dx dweight", {}),
          ("linear_bwd", "residual out", {}),
          ("linear_bwd", "pre", {"activation": 0}),
          ("linear_bwd", "x", {"dweight": abi.Matrix(None, 0)}),
          ("linear_bwd", "weight", {"dx": abi.Matrix(None, 0)}),
          ("gated_linear", "w_down grad dx dw_gate dw_up dw_down", {}),
          ("gated_linear_bwd", "w_down residual out", {}),
          ("gated_linear_bwd", "x", {"dw_gate": abi.Matrix(None, 0), "dw_up": abi.Matrix(None, 0)}),
          ("gated_linear_bwd", "w_gate w_up", {"dx": abi.Matrix(None, 0)}),
          ("gated_ffn", "grad dx dw_gate dw_up dw_down", {}),
          ("gated_ffn_bwd", "residual out", {}),
          ("gated_ffn_bwd", "x", {"dw_gate": abi.Matrix(None, 0), "dw_up": abi.Matrix(None, 0)}),
          ("gated_ffn_bwd", "w_gate w_up", {"dx": abi.Matrix(None, 0)})]


@pytest.mark.parametrize("call,names,fields", UNREAD)
def test_what_a_call_does_not_read_is_not_checked(call, names, fields):
    for name in names.split():
        for m in (abi.Matrix(P + 1, 64), abi.Matrix(P, -8)):
            a = args(call, **fields, **{name: m})
            try:
                abi.ffn_workspace_size(call, a)
            except abi.FelixError as e:  # without a device
                assert "no CUDA device" in str(e), (call, name)
    if call in ("linear", "linear_bwd"):
        other = {"bias": P + 1} if call == "linear_bwd" else {"dbias": P + 1}
        try:
            abi.ffn_workspace_size(call, args(call, **other))
        except abi.FelixError as e:
            assert "no CUDA device" in str(e), call
