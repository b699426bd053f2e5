"""Token sampling on the GPU against a plain 64-bit statement (kv4_ref.kept).

A row's kept tokens are exact. The token drawn for u is the one whose interval
of the running sum holds u; the kernel's weights are fp32 exponentials held to
2^-32, so an interval's ends may lie off the 64-bit ones by the weights' relative
2^-22 and V * 2^-32 of the total: tokens within that of u's place are allowed.
Log-probabilities: 1e-6 * (1 + |z|)."""
import numpy as np
import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu


def sample(*a, **k):
    import sion_b200
    return sion_b200.sample(*a, **k)


def check_row(x, u, tok, lp, temp, k, p, mp):
    order, n, w = R.kept(x, temp, k, p, mp)
    keep = np.zeros(len(x), bool)
    keep[order[:n]] = True
    # top-p and min-p cut at a running sum or a weight: where the next (or the
    # last) one is within rounding of the cut, either is right
    choices = {n}
    tol = 2.0 ** -20
    if p is not None and p < 1:
        m = len(x) if not k or k <= 0 else min(k, len(x))
        upto = np.cumsum(w[order[:m]])
        before = np.concatenate([[0.0], upto[:-1]])
        lo = int(np.sum(before < p * upto[-1] * (1 - tol)))
        hi = int(np.sum(before < p * upto[-1] * (1 + tol)))
        if n in range(lo, hi + 1):
            choices |= set(range(max(lo, 1), hi + 1))
    if mp:
        lo, hi = int(np.sum(w[order] >= mp * (1 + tol))), int(np.sum(w[order] >= mp * (1 - tol)))
        if n in range(lo, hi + 1):
            choices |= set(range(max(lo, 1), hi + 1))
    for n in sorted(choices)[:64]:
        keep = np.zeros(len(x), bool)
        keep[order[:n]] = True
        c = np.cumsum(np.where(keep, w, 0.0))
        eps = c[-1] * 2.0 ** -21 + len(x) * 2.0 ** -32
        if keep[tok] and c[tok] - w[tok] - eps <= u * c[-1] <= c[tok] + eps:
            xf = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
            z = 0.0 if xf[tok] == xf.max() else (xf[tok] - xf.max()) / temp
            want = z - np.log(c[-1])
            if abs(lp - want) <= 1e-6 * (1 + abs(z)) + 2.0 ** -20:
                return
    raise AssertionError((tok, u, lp, keep[tok], n, len(choices)))


DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (5, 31), (7, 1000), (4, 1025), (6, 32000),
                                    (3, 50021), (2, 131072), (2, 200003)])
def test_sample(dtype, rows, V):
    rng = np.random.default_rng(rows + V)
    x = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 3)
    x[:, V // 3] += 9
    if V > 30:
        x[:, 3::7] = -float("inf")
        x[0, 5] = float("nan")
    x = x.to(DT[dtype])
    xs = x.float().numpy()
    sets = [(None, None, None, None), (0.7, 5, None, None), (1.3, None, 0.9, None),
            (1.0, None, None, 0.05), (0.9, 50, 0.8, 0.01), (2.5, 1000, 0.99, None),
            (1.0, 1, None, None), (1.0, V + 5, 1.0, 0.0), (1.0, 0, 0.0, None),
            (1.0, None, None, 2.0), (1.0, 7, 1e-9, None), (40.0, None, 0.5, None)]
    for temp, k, p, mp in sets:
        u = rng.random(rows).astype(np.float32)
        tok, lp = sample(x.cuda(), torch.from_numpy(u).cuda(), temperature=temp, top_k=k, top_p=p,
                         min_p=mp)
        assert tok.dtype == torch.int32 and lp.dtype == torch.float32
        tok, lp = tok.cpu().numpy(), lp.cpu().numpy()
        for i in range(rows):
            t = float(np.float32(temp)) if temp else 1.0
            check_row(xs[i], float(u[i]), int(tok[i]), float(lp[i]), t, k,
                      None if p is None else float(np.float32(p)),
                      None if mp is None else float(np.float32(mp)))


@pytest.mark.parametrize("V", [300, 5000, 140000])
def test_sample_ties_go_to_the_lowest_index(V):
    # three values only: top-k and top-p cut inside runs of equal ones
    rng = np.random.default_rng(V)
    x = rng.integers(0, 3, V).astype(np.float32)
    big = np.flatnonzero(x == 2)
    N = 400
    u = (np.arange(N) + 0.5) / N
    xs = torch.from_numpy(np.tile(x, (N, 1))).cuda()
    k = min(len(big) - 1, 37)
    tok, lp = sample(xs, torch.from_numpy(u.astype(np.float32)).cuda(), top_k=k)
    np.testing.assert_array_equal(tok.cpu().numpy(), big[(u * k).astype(int)])
    np.testing.assert_allclose(lp.cpu().numpy(), -np.log(k), atol=2e-6)
    # the largest ones and ten of the next
    mid = np.flatnonzero(x == 1)[:10]
    tok, _ = sample(xs, torch.from_numpy(u.astype(np.float32)).cuda(), top_k=len(big) + 10)
    got = tok.cpu().numpy()
    assert np.isin(got, np.concatenate([big, mid])).all()
    # top_p: of n equal ones those with less than p of the mass before them
    y = torch.zeros(N, V, device="cuda")
    tok, _ = sample(y, torch.from_numpy(u.astype(np.float32)).cuda(), top_p=0.25)
    n = int(np.ceil(0.25 * V))
    np.testing.assert_array_equal(tok.cpu().numpy(), (u.astype(np.float32).astype(float) * n).astype(int))


def test_sample_does_not_depend_on_the_batch():
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.standard_normal((300, 40000)).astype(np.float32) * 2).half().cuda()
    u = torch.rand(300, device="cuda")
    kw = dict(temperature=0.8, top_p=0.9)
    tok, lp = sample(x, u, **kw)
    for i in (0, 17, 299):
        a, b = sample(x[i:i + 1], u[i:i + 1], **kw)
        assert a[0] == tok[i] and b[0] == lp[i]
    a, b = sample(x[::3], u[::3].contiguous(), **kw)  # rows apart
    assert torch.equal(a, tok[::3]) and torch.equal(b, lp[::3])
    wide = torch.full((300, 40007), 50.0, device="cuda").half()  # an odd row stride
    wide[:, :40000] = x
    a, b = sample(wide[:, :40000], u, **kw)
    assert torch.equal(a, tok) and torch.equal(b, lp)


@pytest.mark.parametrize("V", [9, 4099, 150001])
def test_sample_special_rows(V):
    ninf = float("-inf")
    x = torch.full((9, V), ninf)
    x[1] = torch.finfo(torch.float32).min       # a mask of the lowest value everywhere
    x[2, 4] = 1.0                               # one token left
    x[3, 2] = x[3, 7] = float("inf")            # two infinities share
    x[4] = float("nan")
    x[5] = 0.0
    x[5, V - 1] = -0.0                          # equal to +0
    x[6] = torch.arange(V).float() % 5          # greedy: the first 4
    x[7, 3] = -1e30
    x[8] = 3.0
    u = torch.tensor([0.5, 0.5, 0.5, 0.75, 0.5, 1 - 2.0 ** -24, 0.5, 0.0, float("nan")])
    t = torch.tensor([1, 1, 1, 1, 1, 1, 0.0, 1e-3, 1.0])
    for kw in ({}, {"top_k": V // 2 + 5}, {"min_p": 0.5}):
        tok, lp = sample(x.cuda(), u.cuda(), temperature=t.cuda(), **kw)
        tok, lp = tok.cpu().numpy(), lp.cpu().numpy()
        n = V if "top_k" not in kw else min(V, kw["top_k"])
        assert tok[0] == -1 and lp[0] == -np.inf and tok[4] == -1
        assert tok[1] == int(0.5 * n) and abs(lp[1] + np.log(n)) < 1e-5
        assert tok[2] == 4 and lp[2] == 0
        assert tok[3] == 7 and abs(lp[3] + np.log(2)) < 1e-6
        assert tok[5] == n - 1
        assert tok[6] == 4 and lp[6] == 0
        assert tok[7] == 3 and lp[7] == 0
        assert tok[8] == 0


def test_sample_frequencies():
    # the inverse of the distribution function over an even grid of u: each kept
    # token is drawn its share of the grid, within two points of it
    rng = np.random.default_rng(4)
    V, N = 700, 20000
    x = rng.standard_normal(V).astype(np.float32)
    u = (np.arange(N) + 0.5) / N
    xs = torch.from_numpy(x).cuda().expand(N, V)
    tok, _ = sample(xs, torch.from_numpy(u.astype(np.float32)).cuda(), temperature=0.7, top_k=100,
                    top_p=0.8)
    order, n, w = R.kept(x, float(np.float32(0.7)), 100, float(np.float32(0.8)), None)
    w = np.where(np.isin(np.arange(V), order[:n]), w, 0)
    got = np.bincount(tok.cpu().numpy(), minlength=V)
    assert (np.abs(got - N * w / w.sum()) <= 2).all()


def test_sample_largest_vocabularies():
    # fp32 rows that do not fit a cluster's shared memory, up to the limit
    rng = np.random.default_rng(5)
    for V in (400000, 524288):
        x = (rng.standard_normal((2, V)) * 3).astype(np.float32)
        u = rng.random(2).astype(np.float32)
        for temp, k, p, mp in ((1.0, 300000, 0.99, None), (0.5, 40, 0.9, 0.01), (1.0, None, None, None)):
            tok, lp = sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(),
                             temperature=temp, top_k=k, top_p=p, min_p=mp)
            for i in range(2):
                check_row(x[i], float(u[i]), int(tok[i]), float(lp[i]), temp, k,
                          None if p is None else float(np.float32(p)),
                          None if mp is None else float(np.float32(mp)))


def test_sample_quotients_are_correctly_rounded():
    # two tokens, the second drawn (its mass is over 2^-24 of the total): its
    # log-probability is q = (x1 - x0) / T less log(1 + exp(q)). q is in (8, 16),
    # where a unit in the last place is 9.5e-7: with the last rounding of half of
    # that, a quotient that is one unit off is seen
    rng = np.random.default_rng(6)
    n = 100000
    t = np.exp(rng.uniform(-3, 3, n)).astype(np.float32)
    z = rng.uniform(-15.9, -8.1, n)
    x = np.stack([np.zeros(n), z * t], 1).astype(np.float32)
    u = np.full(n, 1 - 2.0 ** -24, np.float32)
    tok, lp = sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(),
                     temperature=torch.from_numpy(t).cuda())
    drawn = tok.cpu().numpy() == 1
    q = x[:, 1] / t
    assert drawn.all()
    q = q.astype(np.float64)
    np.testing.assert_allclose(lp.cpu().numpy(), q - np.log1p(np.exp(q)), rtol=0, atol=5.5e-7)


@pytest.mark.parametrize("V", [1500, 30000, 131072])
@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 1023, 1024, 1025, 5000])
def test_sample_top_k_around_the_limits(V, k):
    rng = np.random.default_rng(V + k)
    for x in (rng.standard_normal((2, V)), np.round(rng.standard_normal((2, V)) * 2),
              np.repeat([[0.0], [-np.inf]], V, 1) + (np.arange(V) == 7)):
        x = x.astype(np.float32)
        x[1, 7] = 1.0
        u = rng.random(2).astype(np.float32)
        for p, mp in ((None, None), (0.7, None), (0.9, 0.1)):
            tok, lp = sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(),
                             temperature=0.9, top_k=k, top_p=p, min_p=mp)
            for i in range(2):
                check_row(x[i], float(u[i]), int(tok[i]), float(lp[i]), float(np.float32(0.9)), k,
                          None if p is None else float(np.float32(p)),
                          None if mp is None else float(np.float32(mp)))


def test_sample_refusals(felix):
    x, u = torch.zeros(2, 5, device="cuda"), torch.zeros(2, device="cuda")
    for text, call in [
            ("must be CUDA", lambda: sample(x.cpu(), u)),
            ("2D", lambda: sample(x[0], u)),
            ("float32, float16 or bfloat16", lambda: sample(x.double(), u)),
            ("one entry per row", lambda: sample(x, u[:1])),
            ("top_k must be", lambda: sample(x, u, top_k=torch.ones(2, device="cuda"))),
            ("vocab", lambda: sample(x[:, :0], u)),
            ("vocab must be 1..524288", lambda: sample(torch.zeros(2, 524289, device="cuda"), u)),
            ("temperature must be on", lambda: sample(x, u, temperature=torch.ones(2)))]:
        with pytest.raises(RuntimeError, match=text):
            call()
    tok, lp = sample(x[:0], u[:0])
    assert tok.numel() == 0 and lp.numel() == 0
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(felix.FelixError):
        felix.check(felix.lib().felix_sample(None, 0, 2, 5, 5, u.data_ptr(), None, None, None, None,
                                             i.data_ptr(), u.data_ptr(), None))
    with pytest.raises(felix.FelixError):
        felix.check(felix.lib().felix_sample(x.data_ptr(), 7, 2, 5, 5, u.data_ptr(), None, None,
                                             None, None, i.data_ptr(), u.data_ptr(), None))
