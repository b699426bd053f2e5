"""kv4_fork of a slot whose last page is not in the pool."""
import numpy as np
import pytest
import torch

from test_kv4_scales_gpu import i32, sion

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("missing", [-1, 6, 1 << 30])
def test_a_missing_last_page_stays_missing(missing, inplace):
    # a token without a page reads as zero and is not attended to; the copy of a
    # slot must not show in its place what a free page still holds
    page, D = 16, 64
    table = np.array([[0, missing], [-1, -1], [1, 2], [-1, -1]], np.int32)
    lens, refs = [20, 0, 20, 0], [1, 1, 1, 0, 0, 0]
    pool = torch.randint(0, 255, (6, sion().kv4_page_bytes(1, D, page)), dtype=torch.uint8,
                         device="cuda")
    before = pool.clone()
    t = [i32(table), i32(lens), i32(refs)]
    got = sion().kv4_fork(pool, *t, i32([0, 2]), i32([1, 3]), page, out=t if inplace else None)
    tab, n, r, status = (x.cpu().numpy() for x in got)
    assert status.tolist() == [0, 0] and n.tolist() == [20, 20, 20, 20]
    assert tab[1].tolist() == [0, -1] and tab[3].tolist() == [1, 3]
    assert r.tolist() == [2, 2, 1, 1, 0, 0]
    before[3] = before[2]
    assert torch.equal(pool, before)
    k, v = sion().kv4_read(pool, got[0], got[1], 20, 1, D)
    assert (k[1, 0, 16:] == 0).all() and (v[1, 0, 16:] == 0).all()
