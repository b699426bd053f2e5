"""kv4_attention sees what the cache's bytes say, whoever wrote them: it agrees with
the format (and with kv4_read) for tokens inside `lens` that were never appended."""
import numpy as np
import pytest
import torch

import kv4_ref as R
from test_kv4_scales_gpu import TYPES, check, filled, i32, sion

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,rows,group", [(128, 1, 4), (64, 1, 1), (64, 5, 8), (128, 3, 4)])
def test_unwritten_tokens_of_a_zeroed_pool_are_zeros(dtype, D, rows, group):
    rng = np.random.default_rng(D + rows)
    page, n, wrote = 16, 90, 60
    pool = torch.zeros(6, sion().kv4_page_bytes(1, D, page), dtype=torch.uint8, device="cuda")
    table = np.array([[4, 0, 2, 5, 1, 3]], np.int32)
    k, v = (torch.from_numpy(rng.standard_normal((1, 1, wrote, D))).half().cuda() for _ in "kv")
    sion().kv4_append(pool, i32(table), i32([wrote]), k, v)
    _, got = sion().kv4_read(pool, i32(table), i32([n]), n, 1, D)
    assert (got[0, 0, wrote:] == 0).all()
    q = torch.from_numpy(rng.standard_normal((1, group, rows, D))).to(dtype)
    check(pool, table, n, q, 1, page)
    # nothing was written at all
    empty = torch.zeros_like(pool)
    o, lse = sion().kv4_attention_lse(q.cuda(), empty, i32(table), i32([n]), 1)
    assert (o.float().abs() < 1e-12).all()
    seen = torch.arange(n - rows + 1, n + 1, device="cuda", dtype=torch.float32)
    assert (lse[0] - seen.log()).abs().max() < 2e-5


@pytest.mark.parametrize("D", [64, 128])
def test_scale_zero_is_the_base_whatever_the_codes(D):
    rng = np.random.default_rng(D)
    page, n = 32, 70
    pool = rng.integers(0, 256, (3, sion().kv4_page_bytes(1, D, page))).astype(np.uint8)
    blocks = pool.reshape(3, page // 16, R.block_bytes(D))
    par = rng.uniform(-1, 1, (3, page // 16, 2, 16, 2)).astype(np.float16)
    par[..., 0] = np.abs(par[..., 0])
    par[:, :, 1, ::3, 0] = 0        # V scales of zero, of either sign
    par[:, :, 1, 1::6, 0] = -0.0
    blocks[..., 16 * D:] = par.reshape(3, page // 16, -1).view(np.uint8)
    table = np.array([[2, 0, 1]], np.int32)
    for rows, group in ((1, 4), (4, 8)):
        q = torch.from_numpy(rng.standard_normal((1, group, rows, D)) * 0.05).half()
        check(torch.from_numpy(pool).cuda(), table, n, q, 1, page)


def test_negative_scales_are_read_as_they_stand():
    rng = np.random.default_rng(7)
    D, page, n = 64, 16, 45
    pool = rng.integers(0, 256, (3, sion().kv4_page_bytes(1, D, page))).astype(np.uint8)
    par = rng.uniform(-1, 1, (3, 2, 16, 2)).astype(np.float16)
    par[:, 1, 5:9, 0] *= np.float16(1e-4)
    pool[:, 16 * D:] = par.reshape(3, -1).view(np.uint8)
    q = torch.from_numpy(rng.standard_normal((1, 8, 2, D)) * 0.05).half()
    check(torch.from_numpy(pool).cuda(), np.array([[1, 2, 0]], np.int32), n, q, 1, page)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 6])
def test_a_likely_token_of_zeros(dtype, rows):
    # the result is made by 4000 unlikely tokens
    rng = np.random.default_rng(3)
    n, D, page = 4001, 128, 64
    for where in (0, 2000, n - rows):
        for base in (0.0, 1e-4, 3.0):
            k, v = np.zeros((1, n, D)), rng.standard_normal((1, n, D)) * 0.006
            k[0, where] = 22 * np.log(2) / np.sqrt(D)
            v[0, where] = base
            pool, table = filled(k, v, page)
            q = torch.ones(1, 4, rows, D, dtype=TYPES[dtype][0])
            check(pool, table, n, q, 1, page)
