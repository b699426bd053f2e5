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
