"""Build-time check of the register count of the feed-forward products' wide tiles (no
GPU): their setmaxnreg split assumes 168 at launch, and with another count the epilogue
would wait for registers that nobody gives up."""
import os
import re

import pytest

from sion_b200 import build

_LOG = """ptxas info    : Compiling entry function '_ZN9felix_ffn7product18ffn_product_kernelI6__halfLi0ELi2ELi2EEEvNS0_6ParamsE' for 'sm_100a'
    40 bytes stack frame, 96 bytes spill stores, 108 bytes spill loads
ptxas info    : Used {n} registers, used 2 barriers
ptxas info    : Compiling entry function '_ZN9felix_ffn7product18ffn_product_kernelI6__halfLi0ELi2ELi1EEEvNS0_6ParamsE' for 'sm_100a'
ptxas info    : Used 150 registers, used 2 barriers
"""


def test_the_assumed_count_passes_and_others_are_refused():
    build.check_ffn_registers(_LOG.format(n=168))
    for n in (160, 170, 128):
        with pytest.raises(RuntimeError, match="assumes 168"):
            build.check_ffn_registers(_LOG.format(n=n))


def test_a_log_without_the_kernels_is_refused():
    with pytest.raises(RuntimeError, match="no wide"):
        build.check_ffn_registers(_LOG.split("ptxas info    : Compiling entry")[2])


def test_the_sources_assume_the_same_count():
    text = open(os.path.join(build.CSRC, "ffn_product_sm100.cu")).read()
    m = re.search(r"kRegsLaunch = (\d+), kRegsFirst = (\d+), kRegsEpi = (\d+)", text)
    launch, first, epi = map(int, m.groups())
    assert launch == build.FFN_REGS_LAUNCH and 128 * first + 256 * epi <= 384 * launch


def test_kernels_that_start_early():
    """Every kernel waits for the launches before it; none has loads that may be moved in
    front of the wait, and none that allocates tensor memory lets the next launch in."""
    for name in ("ffn_sm100.cu", "ffn_product_sm100.cu", "ffn_few_sm100.cu",
                 "ffn_narrow_sm100.cu", "ffn_finish.cuh", "ffn_internal.h"):
        with open(os.path.join(build.CSRC, name)) as f:
            text = f.read()
        assert not re.search(r"__ldg\(|ld\.global\.nc|__restrict__|<<<", text), name
        for kernel in text.split("__global__")[1:]:
            body = kernel[:kernel.index("\n}\n")]
            assert "wait_for_earlier_launches();" in body, name
            if "tmem_alloc" in body:
                assert "launch_dependents" not in body, name
