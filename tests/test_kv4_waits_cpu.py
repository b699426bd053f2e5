"""A wait that gives up may do so in some lanes of a warp only. It is not provoked on a
GPU: what is checked is that the attention over the 4-bit cache waits in one place,
which brings the lanes together before they go on."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sion_b200", "csrc")


def test_every_wait_is_agreed_on_by_its_warp():
    text = open(os.path.join(CSRC, "kv4_attn_sm100.cu")).read()
    text = re.sub(r"//[^\n]*", "", text)
    assert len(re.findall(r"\bmbar_(?:try_)?wait\w*\(", text)) == 1
    helper = re.search(r"bool warp_wait\([^{]*\{(.*?)\n\}", text, re.S).group(1)
    assert re.search(r"__all_sync\(~0u,\s*felix_sm100::mbar_wait\(", helper)
    assert len(re.findall(r"(?<!bool )\bwarp_wait\(", text)) == 2


def test_whoever_leaves_after_a_wait_that_gave_up_lets_the_copies_land():
    text = open(os.path.join(CSRC, "kv4_attn_sm100.cu")).read()
    kernel = text[text.index("kv4_attn_kernel(const AttnParams P)"):]
    assert len(re.findall(r"if \((?:sm\.abort|gone)\) let_copies_land\(\);", kernel)) == 2
