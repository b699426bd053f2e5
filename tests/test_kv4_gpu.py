"""The 4-bit paged cache on the GPU: append, read, attention and the page
operations, through the Python module and the C ABI, against plain 64-bit
statements (kv4_ref.py).

Tolerances. Codes, scales and page numbers are exact. Attention: the scores
carry fp32 rounding (below 2e-5 in the exponent at these sizes), p * scale_v is
rounded once to fp16, a relative 2^-11 of terms p |V - base_v| <= 2 p max|V|, and
the result once to its type (fp16 2^-11, bf16 2^-8 relative; half of fp16's
smallest step at the bottom): |err| <= 2^-10 max|V| + 2e-5 max|V| + 2^-11 or 2^-8
|ref| + 2^-25. LSE: 2e-5 + 1e-6 |ref|."""
import numpy as np
import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def sion():
    import sion_b200
    return sion_b200


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def make_table(lens, page, pool_pages, rng, width=None):
    need = [R.pages_for(n, page) for n in lens]
    width = max(1, max(need)) if width is None else width
    order = rng.permutation(pool_pages)[:sum(need)]
    t, k = np.full((len(lens), width), -1, np.int32), 0
    for s, n in enumerate(need):
        t[s, :n] = order[k:k + n]
        k += n
    return t


def build(lens, kvh, D, page, rng, dtype=torch.float16, spare=2, amp_k=1.0, amp_v=1.0):
    """A pool whose unused bytes read as NaN, filled through kv4_append."""
    total = sum(R.pages_for(n, page) for n in lens) + spare
    pool = torch.full((total, sion().kv4_page_bytes(kvh, D, page)), 0xFF, dtype=torch.uint8,
                      device="cuda")
    table = make_table(lens, page, total, rng)
    rows = max(1, max(lens))
    k = torch.from_numpy(rng.standard_normal((len(lens), kvh, rows, D)) * amp_k).to(dtype)
    v = torch.from_numpy(rng.standard_normal((len(lens), kvh, rows, D)) * amp_v).to(dtype)
    sion().kv4_append(pool, i32(table), i32(lens), k.cuda(), v.cuda(), counts=i32(lens))
    return pool, table, k, v


def check_attention(pool, table, lens, q, kvh, page, counts=None, scale=0.0):
    D, rows = q.shape[3], q.shape[2]
    o, lse = sion().kv4_attention_lse(q, pool, i32(table), i32(lens), kvh,
                                      counts=None if counts is None else i32(counts), scale=scale)
    o2 = sion().kv4_attention(q, pool, i32(table), i32(lens), kvh,
                              counts=None if counts is None else i32(counts), scale=scale)
    torch.cuda.synchronize()
    assert o.dtype == q.dtype and torch.equal(o, o2)
    K, V = R.decode(pool.cpu().numpy(), page, kvh, D)
    n = [rows] * len(lens) if counts is None else [min(max(c, 0), rows) for c in counts]
    ref, L, M = R.attention(q.double().cpu().numpy(), K, V, table, lens, page, n,
                            scale or 1 / np.sqrt(D))
    got, gl = o.double().cpu().numpy(), lse.double().cpu().numpy()
    eps = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    tol = (2.0 ** -10 + 2e-5) * M[..., None] + eps * np.abs(ref) + 2.0 ** -25
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= tol).all(), np.abs(got - ref).max()
    empty = np.isinf(L)
    assert (gl[empty] == -np.inf).all() and (got[empty] == 0).all()
    assert (np.abs(gl[~empty] - L[~empty]) <= 2e-5 + 1e-6 * np.abs(L[~empty])).all()
    return o, lse


# ------------------------------------------------------------- append and read
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,page,kvh", [(64, 16, 1), (128, 64, 3), (64, 128, 8), (128, 16, 2)])
def test_append_and_read(dtype, D, page, kvh):
    rng = np.random.default_rng(D + page)
    lens = [0, 1, 15, 16, 17, 31, 33, 64, 100, page + 1]
    pool, table, k, v = build(lens, kvh, D, page, rng, TYPES[dtype])
    K, V = R.decode(pool.cpu().numpy(), page, kvh, D)
    wk, wv = R.quantised(k.double().numpy()), R.quantised(v.double().numpy())
    for s, n in enumerate(lens):
        for t in range(n):
            np.testing.assert_array_equal(K[table[s, t // page], :, t % page], wk[s, :, t])
            np.testing.assert_array_equal(V[table[s, t // page], :, t % page], wv[s, :, t])
    # the last 20 tokens, right-aligned: row i is token len - count + i
    counts = [min(n, 20) for n in lens]
    rk, rv = sion().kv4_read(pool, i32(table), i32(lens), 20, kvh, D, counts=i32(counts))
    for got, want in ((rk, wk), (rv, wv)):
        got = got.cpu().numpy()
        for s, (n, c) in enumerate(zip(lens, counts)):
            np.testing.assert_array_equal(got[s, :, :c],
                                          want[s, :, n - c:n].astype(np.float16))
            assert (got[s, :, c:] == 0).all()
    # without counts all rows are tokens; those before the first read as zero
    rk, _ = sion().kv4_read(pool, i32(table), i32(lens), 18, kvh, D)
    rk = rk.cpu().numpy()
    for s, n in enumerate(lens):
        assert (rk[s, :, :max(18 - n, 0)] == 0).all()
        if n >= 18:
            np.testing.assert_array_equal(rk[s], wk[s, :, n - 18:n].astype(np.float16))


def test_append_one_token_at_a_time_equals_all_at_once():
    rng = np.random.default_rng(3)
    lens, kvh, D, page = [37, 5, 64], 2, 128, 32
    pool, table, k, v = build(lens, kvh, D, page, rng)
    step = torch.full_like(pool, 0xFF)
    # K and V as views of one projection [slots, rows, 2, heads, D]
    kv = torch.stack([k, v], 0).permute(1, 3, 0, 2, 4).contiguous().cuda()
    for t in range(max(lens)):
        now = [min(t + 1, n) for n in lens]
        counts = [1 if t < n else 0 for n in lens]
        part = kv[:, t:t + 1]
        sion().kv4_append(step, i32(table), i32(now), part[:, :, 0].transpose(1, 2),
                          part[:, :, 1].transpose(1, 2), counts=i32(counts))
    torch.cuda.synchronize()
    assert torch.equal(step, pool)


def test_append_special_values():
    D, page = 64, 16
    x = torch.zeros(1, 1, 8, D)
    x[0, 0, 0] = 3.25                       # all equal
    x[0, 0, 1, 5] = float("inf")
    x[0, 0, 2, 7] = float("nan")
    x[0, 0, 3] = torch.linspace(-65504, 65504, D)
    x[0, 0, 4] = torch.linspace(0, 1e-7, D)  # below fp16's steps
    x[0, 0, 5, 0], x[0, 0, 5, 1] = 1e30, -1e38  # past fp16 (bf16 only)
    x[0, 0, 6, ::2] = -0.0
    x[0, 0, 7] = torch.linspace(100, 100.5, D)
    pool = torch.zeros(1, sion().kv4_page_bytes(1, D, page), dtype=torch.uint8, device="cuda")
    for dtype in TYPES.values():
        y = x.clone()
        if dtype == torch.float16:
            y[0, 0, 5] = 0
        y = y.to(dtype)
        sion().kv4_append(pool, i32([[0]]), i32([8]), y.cuda(), y.cuda())
        K, V = R.decode(pool.cpu().numpy(), page, 1, D)
        want = R.quantised(y.double().numpy())
        np.testing.assert_array_equal(K[0, :, :8], want[0])
        np.testing.assert_array_equal(V[0, :, :8], want[0])
        assert np.isnan(K[0, 0, 1]).all() and np.isnan(K[0, 0, 2]).all()


def test_append_leaves_out_what_has_no_place():
    # no page in the table, past the table's width, before the first token
    D, page, kvh = 64, 16, 1
    pool = torch.full((3, sion().kv4_page_bytes(kvh, D, page)), 7, dtype=torch.uint8, device="cuda")
    before = pool.clone()
    k = torch.randn(1, kvh, 4, D, device="cuda").half()
    for table, n in (([[-1]], 4), ([[3]], 4), ([[1 << 30]], 4), ([[1]], 20)):
        sion().kv4_append(pool, i32(table), i32([n]), k, k)
        assert torch.equal(pool, before)
    sion().kv4_append(pool, i32([[1]]), i32([2]), k, k)  # rows 2 and 3 are tokens 0 and 1
    K, _ = R.decode(pool.cpu().numpy(), page, kvh, D)
    np.testing.assert_array_equal(K[1, :, :2], R.quantised(k.double().cpu().numpy())[0, :, 2:])
    assert torch.equal(pool[0], before[0]) and torch.equal(pool[2], before[2])


# ------------------------------------------------------------------- attention
LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 130, 333]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,page,kvh,group", [(64, 16, 2, 4), (128, 64, 1, 8), (128, 16, 3, 1),
                                              (64, 128, 2, 3), (128, 32, 1, 13)])
def test_attention_single_tokens(dtype, D, page, kvh, group):
    rng = np.random.default_rng(D + page + group)
    pool, table, _, _ = build(LENS, kvh, D, page, rng)
    q = torch.from_numpy(rng.standard_normal((len(LENS), kvh * group, 1, D)) * 2)
    check_attention(pool, table, LENS, q.to(TYPES[dtype]).cuda(), kvh, page)


@pytest.mark.parametrize("D,rows,group", [(128, 2, 4), (64, 5, 8), (64, 3, 3), (128, 19, 2),
                                          (64, 70, 1), (128, 1, 40)])
def test_attention_several_rows(D, rows, group):
    rng = np.random.default_rng(rows + group)
    pool, table, _, _ = build(LENS, 2, D, 32, rng)
    # q as a transposed view [slots, rows, heads, D], its batch stride padded
    q = torch.from_numpy(rng.standard_normal((len(LENS), rows + 1, 2 * group, D))).half().cuda()
    q = q[:, :rows].transpose(1, 2)
    check_attention(pool, table, LENS, q, 2, 32)  # rows > len: the early rows see nothing
    counts = [rng.integers(-1, rows + 3) for _ in LENS]
    check_attention(pool, table, LENS, q, 2, 32, counts=counts, scale=0.37)


def test_attention_many_slots_and_a_long_one():
    rng = np.random.default_rng(8)
    lens = [int(n) for n in rng.integers(0, 40, 700)]
    lens[650] = 9001
    pool, table, _, _ = build(lens, 1, 64, 16, rng)
    q = torch.from_numpy(rng.standard_normal((700, 4, 1, 64))).half().cuda()
    check_attention(pool, table, lens, q, 1, 16)


def test_attention_of_few_long_slots_is_split_and_repeatable():
    rng = np.random.default_rng(9)
    lens = [30011, 7]
    pool, table, _, _ = build(lens, 2, 128, 64, rng)
    q = torch.from_numpy(rng.standard_normal((2, 16, 1, 128))).to(torch.bfloat16).cuda()
    o, lse = check_attention(pool, table, lens, q, 2, 64)
    for _ in range(5):
        o2, lse2 = sion().kv4_attention_lse(q, pool, i32(table), i32(lens), 2)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_attention_uniform_over_many_tokens_keeps_the_mean():
    # equal scores over many tokens: the result is a small mean of large terms;
    # the codes' offset must not show. Per term 2^-11 relative and of either
    # sign, so the sum is off by about 2^-11 sqrt(n) |V|: five times that is allowed.
    rng = np.random.default_rng(10)
    n, D = 60000, 64
    pool, table, _, _ = build([n], 1, D, 128, rng, amp_k=0.0)
    q = torch.zeros(1, 8, 1, D, device="cuda").half()
    o, _ = sion().kv4_attention_lse(q, pool, i32(table), i32([n]), 1)
    _, V = R.decode(pool.cpu().numpy(), 128, 1, D)
    v = V[table[0]].transpose(0, 2, 1, 3).reshape(-1, 1, D)[:n, 0]
    ref = v.mean(0)
    err = np.abs(o.double().cpu().numpy()[0, 0, 0] - ref)
    assert (err <= 2.0 ** -11 * np.abs(ref) + 5 * 2.0 ** -11 * np.abs(v).std() / np.sqrt(n)
            + 2.0 ** -25).all(), err.max()


@pytest.mark.parametrize("amp_k,amp_v,amp_q", [(1.0, 1e-6, 1.0), (1.0, 6000.0, 1.0),
                                               (1e-5, 1.0, 1.0), (200.0, 1.0, 0.01),
                                               (1e-3, 1.0, 1e6), (3.0, 1.0, 1e-30)])
def test_attention_magnitudes(amp_k, amp_v, amp_q):
    rng = np.random.default_rng(11)
    lens = [100, 3, 70]
    pool, table, _, _ = build(lens, 2, 128, 16, rng, amp_k=amp_k, amp_v=amp_v)
    q = torch.from_numpy(rng.standard_normal((3, 8, 1, 128)) * amp_q).to(torch.bfloat16).cuda()
    # scores of up to |q . k| / sqrt(D); where they are large their own fp32
    # rounding (2^-22 of the terms' sum) leads: keep to a scale that bounds them
    check_attention(pool, table, lens, q, 2, 16,
                    scale=1 / np.sqrt(128) / max(1.0, amp_q * amp_k / 2))


def test_attention_values_of_mixed_scales():
    # one token's values a million times another's: neither may be lost
    rng = np.random.default_rng(12)
    lens, kvh, D, page = [64], 1, 64, 16
    pool, table, k, v = build(lens, kvh, D, page, rng)
    for big in (0, 40):
        v2 = v.clone() * 1e-4
        v2[0, 0, big] *= 3e6
        sion().kv4_append(pool, i32(table), i32(lens), k.cuda(), v2.cuda())
        q = torch.zeros(1, 4, 1, D).half()
        q[0, 1:] = torch.from_numpy(rng.standard_normal((3, 1, D))).half()
        check_attention(pool, table, lens, q.cuda(), kvh, page)
        # without the large one in sight (row 0 of a prefix), the small ones count
        if big == 40:
            check_attention(pool, table, [30], q.cuda(), kvh, page)


def test_attention_pages_that_are_not_there():
    rng = np.random.default_rng(13)
    lens = [100, 60, 40]
    pool, table, _, _ = build(lens, 1, 64, 16, rng)
    table[0, 2], table[0, 5] = -1, pool.shape[0]
    table[1] = -1                 # nothing to see at all
    q = torch.from_numpy(rng.standard_normal((3, 8, 1, 64))).half().cuda()
    check_attention(pool, table, lens, q, 1, 16)
    check_attention(pool, table[:, :1].copy(), lens, q, 1, 16)  # lens past the table


def test_attention_nan_stays_with_its_slot_and_head():
    rng = np.random.default_rng(14)
    lens, kvh, D, page = [50, 50], 2, 64, 16
    pool, table, k, v = build(lens, kvh, D, page, rng)
    clean = pool.clone()
    q = torch.from_numpy(rng.standard_normal((2, 8, 1, D))).half().cuda()
    good = sion().kv4_attention(q, clean, i32(table), i32(lens), kvh)
    for which in (0, 1):
        kk, vv = k.clone(), v.clone()
        (kk, vv)[which][0, 1, 20, 3] = float("nan")
        sion().kv4_append(pool, i32(table), i32(lens), kk.cuda(), vv.cuda())
        o = sion().kv4_attention(q, pool, i32(table), i32(lens), kvh)
        assert torch.isnan(o[0, 4:]).all()
        assert torch.equal(o[0, :4], good[0, :4]) and torch.equal(o[1], good[1])
    bad = q.clone()
    bad[0, 2, 0, 1] = float("nan")
    bad[1, 5, 0, 1] = float("inf")
    o = sion().kv4_attention(bad, clean, i32(table), i32(lens), kvh)
    assert torch.isnan(o[0, 2]).all() and torch.isnan(o[1, 5]).all()
    o[0, 2], o[1, 5] = good[0, 2], good[1, 5]
    assert torch.equal(o, good)


def test_attention_pool_past_four_gigabytes():
    rng = np.random.default_rng(15)
    kvh, D, page = 8, 128, 128
    size = sion().kv4_page_bytes(kvh, D, page)
    pages = (5 << 30) // size
    pool = torch.empty(pages, size, dtype=torch.uint8, device="cuda")
    lens = [200, 129]
    table = np.array([[pages - 1, pages - 3], [pages - 2, 0]], np.int32)
    k = torch.from_numpy(rng.standard_normal((2, kvh, 200, D))).half()
    v = torch.from_numpy(rng.standard_normal((2, kvh, 200, D))).half()
    sion().kv4_append(pool, i32(table), i32(lens), k.cuda(), v.cuda(), counts=i32(lens))
    q = torch.from_numpy(rng.standard_normal((2, 8, 1, D))).half().cuda()
    o = sion().kv4_attention(q, pool, i32(table), i32(lens), kvh)
    sion().kv4_copy_pages(pool, pool, i32([pages - 1, pages - 3, pages - 2, 0]), i32([5, 6, 7, 8]))
    o2 = sion().kv4_attention(q, pool, i32([[5, 6], [7, 8]]), i32(lens), kvh)
    assert torch.equal(o, o2)
    small = pool[5:9].contiguous()
    check_attention(small, np.array([[0, 1], [2, 3]], np.int32), lens, q, kvh, page)
    assert torch.equal(sion().kv4_attention(q, small, i32([[0, 1], [2, 3]]), i32(lens), kvh), o)


def test_attention_on_another_stream_and_with_a_workspace(felix):
    rng = np.random.default_rng(16)
    lens = [5000, 3]
    pool, table, _, _ = build(lens, 1, 64, 64, rng)
    q = torch.from_numpy(rng.standard_normal((2, 8, 1, 64))).half().cuda()
    want = sion().kv4_attention(q, pool, i32(table), i32(lens), 1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = sion().kv4_attention(q, pool, i32(table), i32(lens), 1)
    side.synchronize()
    assert torch.equal(got, want)
    t, n = i32(table), i32(lens)
    cache = felix.kv4_cache(pool, t, n, 64, 1, 64)
    ws = torch.zeros(felix.kv4_attention_workspace_size(64), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        out = torch.empty_like(q)
        felix.kv4_attention(cache, q, out, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    with pytest.raises(felix.FelixError) as e:
        felix.kv4_attention(cache, q, out, workspace=ws[:1024])
    assert e.value.code == felix.API_ERROR


def test_attention_empty_calls():
    pool = torch.zeros(1, sion().kv4_page_bytes(1, 64, 16), dtype=torch.uint8, device="cuda")
    q = torch.zeros(0, 2, 1, 64, device="cuda").half()
    assert sion().kv4_attention(q, pool, i32(np.zeros((0, 3))), i32(np.zeros(0)), 1).numel() == 0
    q = torch.zeros(2, 2, 0, 64, device="cuda").half()
    assert sion().kv4_attention(q, pool, i32([[0], [0]]), i32([3, 3]), 1).numel() == 0
    q = torch.ones(2, 2, 1, 64, device="cuda").half()
    assert (sion().kv4_attention(q, pool, i32(np.zeros((2, 0))), i32([3, 3]), 1) == 0).all()


# ------------------------------------------------------------- page operations
def state(rng, slots, pages, width, page, kvh=1, D=64, share=True):
    lens = rng.integers(0, width * page // 2, slots).astype(np.int32)
    lens[rng.random(slots) < 0.25] = 0
    if slots > 4:
        lens[1], lens[2] = page, 2 * page  # whole pages
    while sum(R.pages_for(n, page) for n in lens) > pages * 3 // 4:
        lens //= 2
    table = make_table([int(n) for n in lens], page, pages, rng, width)
    if share:
        for s in range(1, slots, 3):
            n = min(lens[s - 1], lens[s]) // page
            table[s, :n] = table[s - 1, :n]
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    pool = rng.integers(0, 256, (pages, sion().kv4_page_bytes(kvh, D, page))).astype(np.uint8)
    return pool, table, lens, refs


def same(got, want):
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g.cpu().numpy(), np.asarray(w))


SIZES = [(1, 1, 1, 16), (7, 40, 9, 16), (40, 700, 30, 32), (1500, 9000, 11, 16), (33, 20011, 900, 16)]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("slots,pages,width,page", SIZES)
def test_reserve(slots, pages, width, page, inplace):
    rng = np.random.default_rng(slots + pages)
    _, table, lens, refs = state(rng, slots, pages, width, page)
    for counts in (np.ones(slots, int), rng.integers(0, 2 * page, slots), np.zeros(slots, int),
                   rng.integers(-3, 3, slots), np.full(slots, pages * page)):
        want = R.reserve(table, lens, refs, counts, page)
        t = [i32(table), i32(lens), i32(refs)]
        got = sion().kv4_reserve(*t, i32(counts), page, out=t if inplace else None)
        same(got, want)
        if not inplace:
            same(t, (table, lens, refs))
        elif want[3][0] == 0:
            assert got[0].data_ptr() == t[0].data_ptr()


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("slots,pages,width,page", SIZES)
def test_fork(slots, pages, width, page, inplace):
    rng = np.random.default_rng(slots + pages + 1)
    pool, table, lens, refs = state(rng, slots, pages, width, page)
    n = min(2 * slots, 1400)
    for k in range(3):
        parents, children = rng.integers(0, slots, n), rng.integers(0, slots, n)
        if k == 1:  # only empty children, and bad numbers
            empty = np.flatnonzero(lens == 0)
            children = empty[rng.integers(0, len(empty), n)] if len(empty) else children
            children[::7], parents[::5] = -1, slots
        if k == 2:
            parents, children = parents[:0], children[:0]
        want = R.fork(pool, table, lens, refs, parents, children, page)
        p, t = torch.from_numpy(pool).cuda(), [i32(table), i32(lens), i32(refs)]
        got = sion().kv4_fork(p, *t, i32(parents), i32(children), page, out=t if inplace else None)
        same([p, *got], want)
        if not inplace:
            same(t, (table, lens, refs))


def test_fork_without_room_changes_nothing():
    rng = np.random.default_rng(5)
    page, pages = 16, 6
    table = np.array([[0, 1, -1], [2, 3, 4], [-1] * 3, [-1] * 3], np.int32)
    lens = np.array([20, 40, 0, 0], np.int32)
    refs = np.array([1, 1, 1, 1, 1, 0], np.int32)
    pool = rng.integers(0, 256, (pages, sion().kv4_page_bytes(1, 64, page))).astype(np.uint8)
    for parents in ([0, 1], [0, 9]):
        p, t = torch.from_numpy(pool).cuda(), [i32(table), i32(lens), i32(refs)]
        got = sion().kv4_fork(p, *t, i32(parents), i32([2, 3]), page)
        want = R.fork(pool, table, lens, refs, parents, [2, 3], page)
        same([p, *got], want)
    assert want[4] == [0, 1]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("slots,pages,width,page", SIZES)
def test_free(slots, pages, width, page, inplace):
    rng = np.random.default_rng(slots + pages + 2)
    _, table, lens, refs = state(rng, slots, pages, width, page)
    for gone in (rng.integers(-2, slots + 2, slots), [], [0, 0, 0], list(range(slots))):
        want = R.free(table, lens, refs, gone, page)
        t = [i32(table), i32(lens), i32(refs)]
        got = sion().kv4_free(*t, i32(np.asarray(gone, np.int32)), page, out=t if inplace else None)
        same(got, want)
    assert (want[2] == 0).all()


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("slots,pages,width,page", SIZES)
def test_compact(slots, pages, width, page, inplace):
    rng = np.random.default_rng(slots + pages + 3)
    pool, table, lens, refs = state(rng, slots, pages, width, page)
    want = R.compact(pool, table, refs)
    p, t = torch.from_numpy(pool).cuda(), [i32(table), i32(refs)]
    got = sion().kv4_compact(p, *t, out=t if inplace else None)
    same([p, *got], want)
    # what each slot holds is unchanged
    for s in range(0, slots, 1 + slots // 50):
        n = R.pages_for(lens[s], page)
        np.testing.assert_array_equal(p.cpu().numpy()[got[0].cpu().numpy()[s, :n]],
                                      pool[table[s, :n]])
    live = int((refs > 0).sum())
    assert (got[1].cpu().numpy()[:live] > 0).all() and (got[1].cpu().numpy()[live:] == 0).all()


@pytest.mark.parametrize("fill", [0, 1])
def test_compact_empty_and_full(fill):
    refs = np.full(3000, fill, np.int32)
    table = (np.arange(3000, dtype=np.int32) if fill else np.full(3000, -1, np.int32)).reshape(30, 100)
    pool = np.random.default_rng(1).integers(0, 256, (3000, 16 * 72)).astype(np.uint8)
    p = torch.from_numpy(pool).cuda()
    t, r = sion().kv4_compact(p, i32(table), i32(refs))
    same((p, t, r), (pool, table, refs))


def test_copy_pages():
    rng = np.random.default_rng(6)
    for kvh, D, page in ((1, 64, 16), (8, 128, 64), (3, 64, 16)):
        size = sion().kv4_page_bytes(kvh, D, page)
        a = torch.randint(0, 256, (40, size), dtype=torch.uint8, device="cuda")
        b = torch.zeros(31, size, dtype=torch.uint8, device="cuda")
        src, dst = rng.permutation(40)[:20], rng.permutation(31)[:20]
        src[3], dst[4], src[5], dst[6] = -1, -5, 40, 31
        want = b.clone()
        for s, d in zip(src, dst):
            if 0 <= s < 40 and 0 <= d < 31:
                want[d] = a[s]
        sion().kv4_copy_pages(a, b, i32(src), i32(dst))
        assert torch.equal(b, want)
    sion().kv4_copy_pages(a, b, i32(np.zeros(0)), i32(np.zeros(0)))


def test_decode_steps_in_a_graph_equal_the_steps():
    # reserve in place, append, attention, sample: one captured step replayed
    rng = np.random.default_rng(7)
    S, kvh, H, D, page, width = 5, 2, 8, 64, 16, 6
    size = sion().kv4_page_bytes(kvh, D, page)

    def fresh():
        lens = i32([0, 3, 15, 16, 40])
        table, refs = i32(np.full((S, width), -1)), i32(np.zeros(40))
        pool = torch.zeros(40, size, dtype=torch.uint8, device="cuda")
        zero = torch.zeros_like(lens)
        sion().kv4_reserve(table, zero, refs, lens, page, out=[table, zero, refs])
        k = torch.from_numpy(np.random.default_rng(1).standard_normal((S, kvh, 40, D))).half().cuda()
        sion().kv4_append(pool, table, zero, k, k, counts=lens)
        return pool, table, zero, refs

    x = torch.zeros(S, H, 1, D, device="cuda").half()
    kv = torch.zeros(S, kvh, 1, D, device="cuda").half()
    u = torch.zeros(S, device="cuda")
    one = i32([1, 1, 0, 1, 1])

    def step(st):
        pool, table, lens, refs = st
        sion().kv4_reserve(table, lens, refs, one, page, out=[table, lens, refs])
        sion().kv4_append(pool, table, lens, kv, kv, counts=one)
        o = sion().kv4_attention(x, pool, table, lens, kvh, counts=one)
        return o, sion().sample(o[:, :, 0].reshape(S, H * D), u, top_k=5)

    inputs = [(torch.from_numpy(rng.standard_normal((S, H, 1, D))).half().cuda(),
               torch.from_numpy(rng.standard_normal((S, kvh, 1, D))).half().cuda(),
               torch.rand(S, device="cuda")) for _ in range(20)]
    eager, want = fresh(), []
    for a, b, c in inputs:
        x.copy_(a), kv.copy_(b), u.copy_(c)
        o, (t, lp) = step(eager)
        want.append((o.clone(), t.clone(), lp.clone()))
    st = fresh()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step(fresh())  # the library's scratch for this stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=warm):
            o, (t, lp) = step(st)
    torch.cuda.synchronize()
    for (a, b, c), w in zip(inputs, want):
        x.copy_(a), kv.copy_(b), u.copy_(c)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, w[0]) and torch.equal(t, w[1]) and torch.equal(lp, w[2])
    assert (st[2].cpu() == eager[2].cpu()).all() and torch.equal(st[0], eager[0])


# -------------------------------------------------------------------- refusals
def test_refusals():
    S = sion()
    pool = torch.zeros(4, S.kv4_page_bytes(2, 64, 16), dtype=torch.uint8, device="cuda")
    table, lens, refs = i32([[0, 1], [2, -1]]), i32([20, 3]), i32([1, 1, 1, 0])
    k = torch.zeros(2, 2, 1, 64, device="cuda").half()
    q = torch.zeros(2, 4, 1, 64, device="cuda").half()
    bad = [
        ("unsupported head dimension", lambda: S.kv4_page_bytes(2, 96, 16)),
        ("power of two", lambda: S.kv4_page_bytes(2, 64, 24)),
        ("power of two", lambda: S.kv4_page_bytes(2, 64, 8)),
        ("kv_heads must be positive", lambda: S.kv4_page_bytes(0, 64, 16)),
        ("must be float16 or bfloat16", lambda: S.kv4_append(pool, table, lens, k.float(), k.float())),
        ("same shape", lambda: S.kv4_append(pool, table, lens, k, k[:, :1])),
        ("page's bytes", lambda: S.kv4_append(pool[:, :-16].contiguous(), table, lens, k, k)),
        ("one entry per slot", lambda: S.kv4_append(pool, table, lens, k[:1], k[:1])),
        ("same slots", lambda: S.kv4_append(pool, table, lens[:1], k, k)),
        ("table must be int32", lambda: S.kv4_append(pool, table.long(), lens, k, k)),
        ("counts must", lambda: S.kv4_append(pool, table, lens, k, k, counts=i32([1]))),
        ("pages must be contiguous uint8", lambda: S.kv4_read(pool.float(), table, lens, 1, 2, 64)),
        ("multiple of kv_heads", lambda: S.kv4_attention(q[:, :3], pool, table, lens, 2)),
        ("4D", lambda: S.kv4_attention(q[0], pool, table, lens, 2)),
        ("one entry per slot", lambda: S.kv4_attention(q[:1], pool, table, lens, 2)),
        ("must be on", lambda: S.kv4_attention(q, pool, table.cpu(), lens, 2)),
        ("must be CUDA", lambda: S.kv4_attention(q.cpu(), pool, table, lens, 2)),
        ("page_size must be", lambda: S.kv4_reserve(table, lens, refs, i32([1, 1]), 20)),
        ("out must have 3", lambda: S.kv4_reserve(table, lens, refs, i32([1, 1]), 16, out=[table])),
        ("same length", lambda: S.kv4_fork(pool, table, lens, refs, i32([0]), i32([1, 0]), 16)),
        ("one entry per page", lambda: S.kv4_compact(pool, table, refs[:3])),
        ("same bytes", lambda: S.kv4_copy_pages(pool, pool[:, :16].contiguous(), i32([0]), i32([1]))),
        ("contiguous", lambda: S.kv4_free(table.t(), lens, refs, i32([0]), 16)),
    ]
    for text, call in bad:
        with pytest.raises(RuntimeError, match=text):
            call()
