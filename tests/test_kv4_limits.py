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


@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_what_a_kernel_cannot_address_is_refused(off):
    # each of these would be a misaligned access on the device
    L, st = abi.lib(), (C.c_int64 * 3)(0, 0, 0)
    c = abi.Kv4Cache(*[CACHE[f] for f, _ in abi.Kv4Cache._fields_])

    def attend(q=64, out=64, ws=None):
        return L.felix_kv4_attention(C.byref(c), q, abi.F16, 4, 1, st, None, 0.0, out, None, ws,
                                     1 << 30, None)

    bad = [attend(ws=64 + off),
           L.felix_hgemm_ex(256, 256, 256, 1.0, 64, 64, 0.0, 64, 1, 0, 0, 0, 64 + off, 1 << 30, None),
           L.felix_hgemm_ex2(256, 256, 256, 1.0, 64, 64, 0.0, 64, 1, 0, 0, 0, 0, 64 + off, 1 << 30,
                             None),
           L.felix_sgemm_ex(256, 256, 256, 1.0, 64, 64, 0.0, 64, 4, 64 + off, 1 << 30, None)]
    if off < 2:
        bad += [attend(q=64 + off),
                L.felix_kv4_append(C.byref(c), 64 + off, 64, abi.F16, 1, st, st, None, None),
                L.felix_kv4_append(C.byref(c), 64, 64 + off, abi.BF16, 1, st, st, None, None),
                L.felix_sample(64 + off, abi.F16, 1, 5, 5, 64, None, None, None, None, 64, 64, None)]
    if off < 8:
        bad.append(attend(out=64 + off))
    if off < 4:
        bad.append(L.felix_sample(64 + off, abi.F32, 1, 5, 5, 64, None, None, None, None, 64, 64, None))
    for rc in bad:
        assert rc == abi.API_ERROR
        assert "aligned" in L.felix_last_error_message().decode()
