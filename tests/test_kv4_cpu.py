"""The 4-bit cache's and sampling's argument checks that need no GPU, and the
tests' own statement of the cache's layout."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R
from sion_b200 import abi


@pytest.mark.parametrize("D", [64, 128])
def test_page_bytes(D):
    for heads, page in ((1, 16), (8, 64), (3, 4096)):
        assert abi.kv4_page_bytes(heads, D, page) == page * heads * (D + 8)


@pytest.mark.parametrize("args", [(8, 96, 64), (8, 128, 24), (8, 128, 8), (8, 128, 8192)])
def test_page_bytes_refuses(args):
    with pytest.raises(abi.FelixError) as e:
        abi.kv4_page_bytes(*args)
    assert e.value.code == abi.API_ERROR


def cache(**kw):
    d = dict(pages=0x1000, num_pages=4, page_size=16, kv_heads=2, head_dim=64, table=0x2000,
             lens=0x3000, slots=2, width=2)
    d.update(kw)
    return abi.Kv4Cache(*[d[f] for f, _ in abi.Kv4Cache._fields_])


@pytest.mark.parametrize("kw,text", [({"pages": 0}, "null"), ({"table": 0}, "null"),
                                     ({"lens": 0}, "null"), ({"head_dim": 80}, "head_dim"),
                                     ({"page_size": 48}, "page_size"), ({"kv_heads": 0}, "kv_heads"),
                                     ({"num_pages": 0}, "num_pages"), ({"pages": 0x1008}, "aligned"),
                                     ({"width": 1 << 28}, "too many")])
def test_cache_arguments_are_checked_before_any_device_work(kw, text):
    L, c, st = abi.lib(), cache(**kw), (C.c_int64 * 3)(0, 0, 0)
    for rc in (L.felix_kv4_append(C.byref(c), 16, 16, abi.F16, 1, st, st, None, None),
               L.felix_kv4_read(C.byref(c), 1, None, 16, 16, None),
               L.felix_kv4_attention(C.byref(c), 16, abi.F16, 4, 1, st, None, 0.0, 16, None, None, 0,
                                     None)):
        assert rc == abi.API_ERROR and text in L.felix_last_error_message().decode()


def test_other_arguments_are_checked():
    L, c, st = abi.lib(), cache(), (C.c_int64 * 3)(0, 0, 0)
    att = L.felix_kv4_attention
    bad = [L.felix_kv4_append(C.byref(c), 16, 16, abi.F32, 1, st, st, None, None),
           L.felix_kv4_append(C.byref(c), None, 16, abi.F16, 1, st, st, None, None),
           att(C.byref(c), 16, abi.F32, 4, 1, st, None, 0.0, 16, None, None, 0, None),
           att(C.byref(c), 16, abi.F16, 3, 1, st, None, 0.0, 16, None, None, 0, None),
           att(C.byref(c), None, abi.F16, 4, 1, st, None, 0.0, 16, None, None, 0, None),
           L.felix_kv4_reserve(16, 16, 16, 16, 2, 2, 4, 17, 16, 16, 16, 16, None),
           L.felix_kv4_reserve(16, 16, 16, 16, 2, 2, 0, 16, 16, 16, 16, 16, None),
           L.felix_kv4_free(16, 16, None, 16, 1, 2, 2, 4, 16, 16, 16, 16, None),
           L.felix_kv4_fork(16, 2304, 16, 16, 16, None, 16, 1, 2, 2, 4, 16, 16, 16, 16, 16, None),
           L.felix_kv4_compact(16, 2300, 16, 16, 2, 2, 4, 16, 16, None),
           L.felix_kv4_copy_pages(16, 4, 16, 4, 100, 16, 16, 1, None),
           L.felix_sample(16, 3, 1, 5, 5, 16, None, None, None, None, 16, 16, None),
           L.felix_sample(16, abi.F32, 1, 0, 5, 16, None, None, None, None, 16, 16, None),
           L.felix_sample(16, abi.F32, 1, 5, 5, None, None, None, None, None, 16, 16, None)]
    assert bad == [abi.API_ERROR] * len(bad)
    assert att(C.byref(cache(slots=0)), None, abi.F16, 4, 1, None, None, 0.0, None, None, None, 0,
               None) == abi.SUCCESS


@pytest.mark.parametrize("D", [64, 128])
def test_reference_layout_places_every_code_once(D):
    # decode of a block whose nibbles are counted: each (token, dim) reads its own
    for part in (0, 1):
        seen = set()
        for nib in range(16 * D):
            block = np.zeros((1, R.block_bytes(D)), np.uint8)
            block[0, part * 8 * D + nib // 2] = 1 << 4 * (nib % 2)
            ones = np.full(64, 0, np.uint8).view(np.float16)
            ones[0::2] = 1.0
            block[0, 16 * D:16 * D + 64] = block[0, 16 * D + 64:] = ones.view(np.uint8)
            got = R.decode(block, 16, 1, D)[part][0, 0] + 8
            at = np.argwhere(got == 1)
            assert got.sum() == 1 and len(at) == 1
            seen.add(tuple(at[0]))
        assert len(seen) == 16 * D
