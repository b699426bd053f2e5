"""The decode operators' sources define nothing that is not used."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sion_b200", "csrc")


def code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


@pytest.mark.parametrize("header,names", [("kv4_layout.cuh", r"\w+"), ("sm100_ptx.cuh", r"bulk_\w+")])
def test_what_a_header_defines_is_used(header, names):
    text = code(header)
    others = "".join(code(f) for f in sorted(os.listdir(CSRC)) if f != header)
    names = re.findall(r"(?:__forceinline__|constexpr)[^;={(]*?\b(%s)\s*\(" % names, text)
    assert names
    assert [n for n in names if not re.search(r"\b%s\b" % n, others) and
            len(re.findall(r"\b%s\b" % n, text)) == 1] == []


def test_the_units_share_no_namespace_for_what_is_their_own():
    # TokenParams and f2 mean different things in the cache's and in attention's file: in
    # one namespace that would break the one-definition rule
    inner = {}
    for f in ("kv4_attn_sm100.cu", "kv4_cache_sm100.cu", "sample_sm100.cu"):
        for name in re.findall(r"^namespace (\w+) \{", code(f), re.M):
            if name != "felix_impl":
                assert inner.setdefault(name, f) == f
    assert len(inner) == 3
