"""A transformer block trained and then run one token at a time: causal flash attention
between linear layers, and a gated feed-forward block, with the residuals added in the
products' epilogues.

    python examples/ffn_block.py
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import sion_b200 as sion  # noqa: E402

HEADS, DIM = 4, 64
WIDTH, HIDDEN = HEADS * DIM, 704


def norm(x):
    x32 = x.float()
    return (x32 * torch.rsqrt(x32.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


def weights(seed: int, dtype=torch.float16) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def matrix(rows, cols):
        return (torch.randn(rows, cols, device="cuda", generator=g) * cols ** -0.5).to(dtype)

    return {"qkv": matrix(3 * WIDTH, WIDTH), "bias": torch.zeros(3 * WIDTH, device="cuda", dtype=dtype),
            "out": matrix(WIDTH, WIDTH), "gate": matrix(HIDDEN, WIDTH), "up": matrix(HIDDEN, WIDTH),
            "down": matrix(WIDTH, HIDDEN)}


def block(p: dict, x):
    """x [batch, tokens, WIDTH] through the block."""
    batch, tokens, _ = x.shape
    qkv = sion.linear_autograd(norm(x), p["qkv"], p["bias"])
    q, k, v = qkv.view(batch, tokens, 3, HEADS, DIM).permute(2, 0, 3, 1, 4)
    a = sion.flash_attention_autograd(q, k, v, causal=True)
    x = sion.linear_autograd(a.transpose(1, 2).reshape(batch, tokens, WIDTH), p["out"], None, x)
    return sion.gated_ffn_autograd(norm(x), p["gate"], p["up"], p["down"], x)


def plain_block(p: dict, x):
    """The same in elementary operations, in the type of its arguments."""
    batch, tokens, _ = x.shape
    qkv = norm(x) @ p["qkv"].t() + p["bias"]
    q, k, v = qkv.view(batch, tokens, 3, HEADS, DIM).permute(2, 0, 3, 1, 4)
    s = q @ k.transpose(-1, -2) * DIM ** -0.5
    s = s.masked_fill(torch.ones(tokens, tokens, device=x.device).triu(1).bool(), float("-inf"))
    a = torch.softmax(s, -1) @ v
    x = x + a.transpose(1, 2).reshape(batch, tokens, WIDTH) @ p["out"].t()
    h = norm(x)
    g = h @ p["gate"].t()
    return x + (g * torch.sigmoid(g) * (h @ p["up"].t())) @ p["down"].t()


def train(steps: int = 20, batch: int = 4, tokens: int = 192, rate: float = 0.002, seed: int = 0):
    """Fits the block to another one's answers; returns the losses."""
    target, p = weights(seed + 1), weights(seed)
    master = {k: v.float() for k, v in p.items()}
    p = {k: v.requires_grad_() for k, v in p.items()}
    g = torch.Generator(device="cuda").manual_seed(seed + 2)
    losses = []
    for _ in range(steps):
        x = torch.randn(batch, tokens, WIDTH, device="cuda", generator=g).half()
        with torch.no_grad():
            want = block(target, x)
        loss = (block(p, x) - want).float().square().sum(-1).mean()
        loss.backward()
        losses.append(loss.detach())
        with torch.no_grad():
            for k, t in p.items():
                master[k] -= rate * t.grad.float()
                t.copy_(master[k])
                t.grad = None
    return torch.stack(losses).tolist(), p


def feed_forward_token(p: dict, x):
    """The feed-forward half for the tokens of a decoding step, x [tokens, WIDTH]."""
    return sion.gated_ffn(norm(x), p["gate"], p["up"], p["down"], x)


if __name__ == "__main__":
    losses, params = train()
    print("loss", " ".join(f"{v:.4f}" for v in losses[::4]), f"{losses[-1]:.4f}")
    with torch.no_grad():
        tokens = torch.randn(5, WIDTH, device="cuda").half()
        print("five tokens at once and one by one differ by",
              float((feed_forward_token(params, tokens)
                     - torch.cat([feed_forward_token(params, t) for t in tokens.split(1)])).abs().max()))
