"""Sizes that the decode operators' 32-bit arguments or arithmetic do not hold are
refused, not cut off."""
import ctypes as C

import numpy as np
import pytest
import torch

from sion_b200 import abi

CACHE = dict(pages=0x1000, num_pages=4, page_size=16, kv_heads=2, head_dim=64, table=0x2000,
             lens=0x3000, slots=2, width=2)


def test_rows_past_31_bits_are_refused():
    L, st = abi.lib(), (C.c_int64 * 3)(0, 0, 0)
    c = abi.Kv4Cache(*[CACHE[f] for f, _ in abi.Kv4Cache._fields_])
    for rows in (1 << 31, (1 << 32) - 1):
        for rc in (L.felix_kv4_append(C.byref(c), 16, 16, abi.F16, rows, st, st, None, None),
                   L.felix_kv4_read(C.byref(c), rows, None, 16, 16, None)):
            assert rc == abi.API_ERROR and "rows" in L.felix_last_error_message().decode()


@pytest.mark.parametrize("heads", [0, 65536, (1 << 32) - 1])
def test_page_bytes_of_heads_that_no_cache_takes(heads):
    with pytest.raises(abi.FelixError, match="kv_heads must be 1..65535"):
        abi.kv4_page_bytes(heads, 64, 16)


@pytest.mark.gpu
def test_torch_sizes_past_32_bits_are_refused():
    import sion_b200 as S

    def i32(v):
        return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")

    pool = torch.full((2, S.kv4_page_bytes(1, 64, 16)), 5, dtype=torch.uint8, device="cuda")
    before = pool.clone()
    k = torch.ones(1, 1, 1, 64, device="cuda").half().expand(1, 1, (1 << 32) + 1, 64)
    x = torch.zeros(1, 1, device="cuda").expand(1, (1 << 32) + 5)
    u = torch.zeros(1, device="cuda")
    for text, call in [("rows", lambda: S.kv4_append(pool, i32([[0]]), i32([3]), k, k)),
                       ("rows", lambda: S.kv4_attention(k, pool, i32([[0]]), i32([3]), 1)),
                       ("kv_heads", lambda: S.kv4_page_bytes((1 << 32) + 2, 64, 16)),
                       ("kv_heads", lambda: S.kv4_read(pool, i32([[0]]), i32([3]), 1, (1 << 32) + 1, 64)),
                       ("vocab must be 1..524288", lambda: S.sample(x, u))]:
        with pytest.raises(RuntimeError, match=text):
            call()
    assert torch.equal(pool, before)


def test_pages_of_no_bytes_are_refused_before_any_change():
    # (the plan would be made, and the copies then fail to launch)
    L = abi.lib()
    assert L.felix_kv4_compact(16, 0, 16, 16, 2, 2, 4, 16, 16, None) == abi.API_ERROR
    assert "multiple of 16" in L.felix_last_error_message().decode()
    rc = L.felix_kv4_fork(16, 0, 16, 16, 16, 16, 16, 1, 2, 2, 4, 16, 16, 16, 16, 16, None)
    assert rc == abi.API_ERROR and "multiple of 16" in L.felix_last_error_message().decode()
