"""Build-time check of the register count of the attention over the 4-bit cache (no
GPU): with eight consumer warps its setmaxnreg split assumes 168 at launch, and a build
with another count would refuse every call of more than eight rows."""
import os
import re

import pytest

from sion_b200 import build

_LOG = """ptxas info    : Compiling entry function '_ZN10felix_impl3kv415kv4_attn_kernelI6__halfLi128ELi2ELi4ELi8EEEvNS0_10AttnParamsE' for 'sm_100a'
ptxas info    : Function properties for _ZN10felix_impl3kv415kv4_attn_kernelI6__halfLi128ELi2ELi4ELi8EEEvNS0_10AttnParamsE
    24 bytes stack frame, 24 bytes spill stores, 40 bytes spill loads
ptxas info    : Used {n} registers, used 2 barriers, 24 bytes cumulative stack size
ptxas info    : Compiling entry function '_ZN10felix_impl3kv415kv4_attn_kernelI6__halfLi64ELi1ELi1ELi4EEEvNS0_10AttnParamsE' for 'sm_100a'
ptxas info    : Used 128 registers, used 2 barriers
"""


def test_the_assumed_count_passes_and_others_are_refused():
    build.check_kv4_registers(_LOG.format(n=168))
    for n in (160, 170, 128):
        with pytest.raises(RuntimeError, match="assumes 168"):
            build.check_kv4_registers(_LOG.format(n=n))


def test_a_log_without_the_kernels_is_refused():
    with pytest.raises(RuntimeError, match="no eight-warp"):
        build.check_kv4_registers(_LOG.split("ptxas info    : Compiling entry")[2])


def test_the_sources_assume_the_same_count():
    text = open(os.path.join(build.CSRC, "kv4_attn_sm100.cu")).read()
    assert int(re.search(r"kRegsLaunch = (\d+)", text).group(1)) == build.KV4_REGS_LAUNCH
