"""kv4_attention at the longest slot that a table can name: 2^31 - 16 tokens.

A thread adds some 150000 equal-sized terms one after another in fp32, a relative
150000 * 2^-24 = 0.9 % at worst, in the sum and in its divisor: 2 % of sum p |V| / S
is allowed, and 0.01 for the log of the divisor."""
import numpy as np
import pytest
import torch

import kv4_ref as R
from test_kv4_scales_gpu import i32, sion

pytestmark = pytest.mark.gpu


def test_the_longest_slot():
    rng = np.random.default_rng(1)
    D, page, pages, width = 64, 16, 4096, (2 ** 31 - 1) // 16
    pool = torch.zeros(pages, sion().kv4_page_bytes(1, D, page), dtype=torch.uint8, device="cuda")
    n = pages * page
    k = rng.standard_normal((1, 1, n, D))
    v = rng.standard_normal((1, 1, n, D)) + np.repeat([3.0, -1.0], n // 2)[:, None]
    sion().kv4_append(pool, torch.arange(pages, dtype=torch.int32, device="cuda")[None], i32([n]),
                      torch.from_numpy(k).half().cuda(), torch.from_numpy(v).half().cuda())
    table = (torch.arange(width, device="cuda", dtype=torch.int32) % pages)[None]
    K, V = (x[:, 0].reshape(n, D) for x in R.decode(pool.cpu().numpy(), page, 1, D))
    q = torch.from_numpy(rng.standard_normal((1, 2, 1, D))).half()
    for length in (page * width, page * width - 9, 2 ** 31 - 1):
        o, lse = sion().kv4_attention_lse(q.cuda(), pool, table, i32([length]), 1)
        o, lse = o.double().cpu().numpy()[0, :, 0], lse.cpu().numpy()[0, :, 0]
        times = np.repeat(np.bincount(np.arange(width) % pages, minlength=pages), page)
        for h in range(2):
            s = K @ q[0, h, 0].double().numpy() / np.sqrt(D)
            p = np.exp(s - s.max()) * times
            S = p.sum()
            assert (np.abs(o[h] - p @ V / S) <= 0.02 * (p @ np.abs(V)) / S).all()
            assert abs(lse[h] - (s.max() + np.log(S))) <= 0.01
