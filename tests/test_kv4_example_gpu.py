"""examples/kv4_decode.py runs the decode operators together."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import kv4_decode
    finally:
        sys.path.pop(0)
    return kv4_decode


def test_example_runs_and_repeats():
    ex = _example()
    a, b = ex.decode(3, 4, 30), ex.decode(3, 4, 30)
    assert torch.equal(a["tokens"], b["tokens"]) and torch.equal(a["score"], b["score"])
    assert a["shared_pages"] == sum(n // ex.PAGE for n in a["prompt_lens"])
    assert a["highest_page"] < a["pages_in_use"]
    t = a["tokens"]
    assert t.shape[0] == 12 and int(t.max()) < ex.VOCAB and (a["score"] <= 0).all()
    live = (t[:, -1] >= 0).cpu() & (t[:, -1] != ex.END).cpu()
    want = torch.tensor([n for _ in range(4) for n in a["prompt_lens"]]) + t.shape[1] - 1
    assert (a["lens"].cpu()[live] == want[live]).all()


def test_example_greedy_answers_of_one_prompt_are_equal():
    # forked slots hold the same cache: without randomness they say the same
    ex = _example()
    t = ex.decode(2, 3, 40, temperature=0.0)["tokens"]
    for p in range(2):
        assert torch.equal(t[p], t[p + 2]) and torch.equal(t[p], t[p + 4])
