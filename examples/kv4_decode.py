"""Several sampled answers to several prompts, from a 4-bit paged cache.

A one-layer toy model with random weights shows the decode operators together,
as a serving loop uses them: the prompts' attention runs in fp16
(flash_attention), their keys and values enter the cache (kv4_reserve,
kv4_append); each prompt is forked into several answers that share its pages
(kv4_fork); every step projects (hgemm_nt), appends, attends over the cache
(kv4_attention) and samples (sample); answers that end leave (kv4_free), and the
pool is made dense (kv4_compact). No count goes through the host in the loop
except to see which answers have ended.

    python examples/kv4_decode.py [--prompts 3] [--answers 4] [--steps 40]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import sion_b200 as sion  # noqa: E402

HEADS, KV_HEADS, DIM, VOCAB, PAGE, END = 8, 2, 64, 1000, 16, 0
HIDDEN = HEADS * DIM


class Layer:
    """Embedding, one attention layer, logits; weights [out, in] in fp16."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g) * cols ** -0.5).half().cuda()

        self.embed = torch.randn(VOCAB, HIDDEN, generator=g).half().cuda()
        self.qkv = weight((HEADS + 2 * KV_HEADS) * DIM, HIDDEN)
        self.out = weight(HIDDEN, HIDDEN)
        self.logits = weight(VOCAB, HIDDEN)

    def project(self, tokens):
        """x, and views q, k, v [slots, heads, rows, D] of tokens [slots, rows]."""
        x = self.embed[tokens.clamp(min=0).long()]
        qkv = sion.hgemm_nt(x.view(-1, HIDDEN), self.qkv)
        qkv = qkv.view(*tokens.shape, HEADS + 2 * KV_HEADS, DIM).transpose(1, 2)
        return x, qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]

    def head(self, x, attended):
        """Logits [slots, vocab] of x [slots, 1, hidden] and its attention output."""
        y = attended.transpose(1, 2).reshape(-1, HIDDEN)
        y = x.view(-1, HIDDEN) + sion.hgemm_nt(y, self.out)
        return sion.hgemm_nt(y, self.logits)


def decode(prompts=3, answers=4, steps=40, seed=0, temperature=0.8, top_k=50, top_p=0.95):
    g = torch.Generator(device="cuda").manual_seed(seed)
    model, slots = Layer(seed), prompts * answers
    lens_host = [17 + 13 * i for i in range(prompts)]
    width = -(-(max(lens_host) + steps) // PAGE)
    pages = torch.zeros(slots * width, sion.kv4_page_bytes(KV_HEADS, DIM, PAGE), dtype=torch.uint8,
                        device="cuda")
    table = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(slots, dtype=torch.int32, device="cuda")
    refs = torch.zeros(len(pages), dtype=torch.int32, device="cuda")
    state = [table, lens, refs]  # updated in place

    # the prompts, padded to one length, in the first slots
    rows = max(lens_host)
    counts = torch.tensor(lens_host + [0] * (slots - prompts), dtype=torch.int32, device="cuda")
    tokens = torch.randint(1, VOCAB, (slots, rows), generator=g, device="cuda")
    x, q, k, v = model.project(tokens)
    group = HEADS // KV_HEADS
    o = sion.flash_attention(q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1), True)
    missing = sion.kv4_reserve(*state, counts, PAGE, out=state)[3]
    sion.kv4_append(pages, table, lens, k, v, counts=counts)
    last = (counts - 1).clamp(min=0).long()
    pick = torch.arange(slots, device="cuda")
    logits = model.head(x[pick, last], o[pick, :, last][:, :, None])

    # each prompt's other answers share its pages
    children = torch.arange(prompts, slots, dtype=torch.int32, device="cuda")
    missing = missing + sion.kv4_fork(pages, *state, children % prompts, children, PAGE, out=state)[3]
    shared = int((refs > 1).sum())
    logits = logits[pick % prompts]

    def draw(logits):
        return sion.sample(logits, torch.rand(slots, generator=g, device="cuda"),
                           temperature=temperature, top_k=top_k, top_p=top_p)

    token, logprob = draw(logits)
    live = torch.ones(slots, dtype=torch.bool, device="cuda")
    said, score = [token.clone()], logprob.clone()
    for _ in range(steps - 1):
        ended = live & (token == END)
        if ended.any():
            gone = ended.nonzero()[:, 0].to(torch.int32)
            sion.kv4_free(*state, gone, PAGE, out=state)
            live &= ~ended
            if not live.any():
                break
        one = live.to(torch.int32)
        missing = missing + sion.kv4_reserve(*state, one, PAGE, out=state)[3]
        x, q, k, v = model.project(token[:, None])
        sion.kv4_append(pages, table, lens, k, v, counts=one)
        token, logprob = draw(model.head(x, sion.kv4_attention(q, pages, table, lens, KV_HEADS,
                                                               counts=one)))
        token = torch.where(live, token, -1)
        score += torch.where(live, logprob, 0.0)
        said.append(token.clone())
    table_c, refs_c = sion.kv4_compact(pages, table, refs)
    in_use = int((refs_c > 0).sum())
    assert int(missing.sum()) == 0, "the pool was too small"
    return {"tokens": torch.stack(said, 1), "score": score, "lens": lens, "shared_pages": shared,
            "pages_in_use": in_use, "highest_page": int(table_c.max()), "prompt_lens": lens_host}


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompts", type=int, default=3)
    ap.add_argument("--answers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=40)
    a = ap.parse_args()
    r = decode(a.prompts, a.answers, a.steps)
    for i, (row, s) in enumerate(zip(r["tokens"].tolist(), r["score"].tolist())):
        print(f"prompt {i % a.prompts} answer {i // a.prompts} (log-probability {s:.1f}):",
              [t for t in row if t >= 0][:12], "...")
    print(f"{r['shared_pages']} pages were shared after the fork; {r['pages_in_use']} in use at the "
          f"end, the highest number {r['highest_page']}")


if __name__ == "__main__":
    main()
