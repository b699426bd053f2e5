"""Calls from several host threads, on one stream and on each thread's own: the
library's scratch, and threads that have not used CUDA before."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

import kv4_ref as R

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # cudaStreamPerThread


def sion():
    import sion_b200
    return sion_b200


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def in_threads(works):
    """Runs the functions in threads of their own, let off together."""
    gate, errors = threading.Barrier(len(works)), []

    def run(f):
        try:
            gate.wait()
            f()
        except Exception as e:  # noqa: BLE001 (shown by the assertion below)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(f,)) for f in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


class Fork:
    """A pool whose odd slots become copies of its even ones, again and again from the
    same state: after any number of calls its bytes are those after one."""
    page, slots, pages = 16, 400, 1500

    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        self.size = 16 * 72
        order = rng.permutation(self.pages).astype(np.int32)
        table = np.full((self.slots, 2), -1, np.int32)
        table[::2] = order[:self.slots].reshape(-1, 2)
        lens = np.where(np.arange(self.slots) % 2 == 0, rng.integers(17, 32, self.slots), 0)
        refs = np.zeros(self.pages, np.int32)
        refs[order[:self.slots]] = 1
        pool = rng.integers(0, 256, (self.pages, self.size)).astype(np.uint8)
        parents = rng.permutation(np.arange(0, self.slots, 2))
        children = np.arange(1, self.slots, 2)
        self.want = R.fork(pool, table, lens.astype(np.int32), refs, parents, children, self.page)
        self.pool = torch.from_numpy(pool).cuda()
        self.dev = [i32(x) for x in (table, lens, refs, parents, children)]
        self.out = [torch.empty_like(x) for x in self.dev[:3]] + [i32([7, 7])]

    def call(self, lib, stream):
        ptr = [x.data_ptr() for x in self.dev]
        out = [x.data_ptr() for x in self.out]
        return lib.felix_kv4_fork(self.pool.data_ptr(), self.size, *ptr, self.slots // 2, self.slots,
                                  2, self.pages, self.page, *out, C.c_void_p(stream))

    def check(self):
        for got, want in zip([self.pool, *self.out], self.want):
            np.testing.assert_array_equal(got.cpu().numpy(), np.asarray(want))


@pytest.mark.parametrize("own_streams", [False, True])
def test_forks_of_two_host_threads(felix, own_streams):
    # a fork is a plan and then the copies that it lists: between the two no other
    # thread's plan may take its place
    forks = [Fork(1), Fork(2)]
    torch.cuda.synchronize()
    stream = PER_THREAD if own_streams else torch.cuda.Stream().cuda_stream
    lib, bad = felix.lib(), []

    def work(f):
        return lambda: bad.extend(rc for rc in (f.call(lib, stream) for _ in range(1500)) if rc)

    in_threads([work(f) for f in forks])
    torch.cuda.synchronize()
    assert not bad
    for f in forks:
        f.check()


def attend_case(seed, tokens=20000):
    """Few long slots, whose parts are joined through the scratch."""
    rng = np.random.default_rng(seed)
    pool = torch.randint(0, 256, (tokens // 64 + 1, sion().kv4_page_bytes(2, 64, 64)),
                         dtype=torch.uint8, device="cuda")
    blocks = pool.view(pool.shape[0], -1, R.block_bytes(64))
    par = rng.uniform(0, 1, (*blocks.shape[:2], 64)).astype(np.float16)
    blocks[..., 16 * 64:] = torch.from_numpy(par.view(np.uint8)).cuda()
    table = i32(rng.permutation(pool.shape[0])[None])
    q = torch.from_numpy(rng.standard_normal((1, 16, 1, 64))).half().cuda()
    return pool, table, i32([tokens]), q


def test_attention_of_host_threads_on_their_own_streams(felix):
    cases = [attend_case(s) for s in range(3)]
    want = [sion().kv4_attention(q, pool, table, lens, 2) for pool, table, lens, q in cases]
    outs = [[torch.zeros_like(c[3]) for _ in range(200)] for c in cases]
    torch.cuda.synchronize()

    def work(case, out):
        pool, table, lens, q = case
        cache = felix.kv4_cache(pool, table, lens, 64, 2, 64)

        def run():
            for o in out:
                felix.kv4_attention(cache, q, o, stream=PER_THREAD)
        return run

    in_threads([work(c, o) for c, o in zip(cases, outs)])
    torch.cuda.synchronize()
    for w, out in zip(want, outs):
        for o in out:
            assert torch.equal(o, w)


@pytest.mark.parametrize("op", ["hgemm", "sgemm", "flash_attn_fwd"])
def test_the_first_call_of_a_new_host_thread(felix, op):
    # nothing has made the device's context current there
    x = torch.randn(2, 2, 128, 128, device="cuda").to(torch.float32 if op == "sgemm" else torch.float16)
    out = [torch.zeros_like(x) for _ in range(2)]
    stream = torch.cuda.current_stream().cuda_stream

    def call(o):
        if op == "flash_attn_fwd":
            felix.flash_attn_fwd(x, x, x, o, stream=stream)
        else:
            getattr(felix, op)(x[0, 0], x[0, 1], o[0, 0], stream=stream)

    call(out[0])
    in_threads([lambda: call(out[1])])
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[1]) and out[0].abs().sum() > 0


def test_hgemm_of_host_threads_while_the_scratch_grows(felix):
    # each thread asks for more and more scratch on one stream
    stream = torch.cuda.Stream().cuda_stream
    sizes = [(256, 256, 4096), (512, 384, 4096), (1100, 1100, 4096), (2200, 2200, 2048)]
    g = torch.Generator().manual_seed(1)
    cases = []
    for m, n, k in sizes:
        a = torch.randn(m, k, generator=g).half().cuda()
        b = torch.randn(n, k, generator=g).half().cuda()
        cases.append((a, b, sion().hgemm_nt(a, b)))
    outs = [[torch.zeros_like(c[2]) for c in cases] for _ in range(4)]
    torch.cuda.synchronize()

    def work(out):
        def run():
            for (a, b, _), o in zip(cases, out):
                for _ in range(20):
                    felix.hgemm(a, b, o, b_layout=felix.B_NK, stream=stream)
        return run

    in_threads([work(o) for o in outs])
    torch.cuda.synchronize()
    for out in outs:
        for o, c in zip(out, cases):
            # the order in which parts are added may differ: fp32 sums, fp16 results
            assert (o.float() - c[2].float()).abs().max() <= 2.0 ** -10 * c[2].float().abs().max()


# ----------------------------------------------------------------------- graphs
def capture(f, stream=None):
    """f's work as a graph, with no call of it before."""
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        f()
    return g


def test_a_graph_keeps_its_scratch_while_the_stream_goes_on():
    # a reserve alone is captured; then the same stream asks for far more scratch
    rng = np.random.default_rng(5)
    slots, width, pages, page = 50, 40, 1500, 16
    lens0 = rng.integers(0, 100, slots).astype(np.int32)
    empty = np.full((slots, width), -1, np.int32)
    table0, _, refs0, status = R.reserve(empty, np.zeros(slots, np.int32), np.zeros(pages, np.int32),
                                         lens0, page)
    assert status == [0, 0]
    counts = rng.integers(0, 60, slots).astype(np.int32)
    want = R.reserve(table0, lens0, refs0, counts, page)
    dev = [i32(x) for x in (table0, lens0, refs0, counts)]
    side, got = torch.cuda.Stream(), []
    g = capture(lambda: got.extend(sion().kv4_reserve(*dev, page)), side)
    pool, table, lens, q = attend_case(4)
    a = torch.randn(1100, 4096, device="cuda").half()
    b = torch.randn(1100, 4096, device="cuda").half()
    with torch.cuda.stream(side):
        first = sion().kv4_attention(q, pool, table, lens, 2)
        for _ in range(3):
            sion().hgemm_nt(a, b)
            g.replay()
            o = sion().kv4_attention(q, pool, table, lens, 2)
        junk = [torch.full((1 << 20,), -1, dtype=torch.int32, device="cuda") for _ in range(30)]
        for x in got:
            x.fill_(99)
        g.replay()
    torch.cuda.synchronize()
    for x, w in zip(got, want):
        np.testing.assert_array_equal(x.cpu().numpy(), np.asarray(w))
    assert torch.equal(o, first) and all(int(j[0]) == -1 for j in junk[:2])


def test_graphs_of_one_stream_run_at_once():
    # two graphs captured one after the other, replayed on two streams, and eager calls
    # on the stream of the captures beside them
    cases = [attend_case(s) for s in (6, 7, 8)]
    want = [sion().kv4_attention(q, pool, table, lens, 2) for pool, table, lens, q in cases]
    side = torch.cuda.Stream()
    outs, graphs = [], []
    for pool, table, lens, q in cases[:2]:
        o = []
        graphs.append(capture(lambda: o.extend(sion().kv4_attention(q, pool, table, lens, 2)
                                               for _ in range(20)), side))
        outs.append(o)
    streams = [torch.cuda.Stream() for _ in graphs]
    pool, table, lens, q = cases[2]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side):
            eager = [sion().kv4_attention(q, pool, table, lens, 2) for _ in range(20)]
        torch.cuda.synchronize()
        for w, out in zip(want, [*outs, eager]):
            assert all(torch.equal(o, w) for o in out)


def test_branches_of_one_graph_have_their_own_scratch():
    cases = [attend_case(s) for s in (9, 10)]
    want = [sion().kv4_attention(q, pool, table, lens, 2) for pool, table, lens, q in cases]
    main, other, outs = torch.cuda.Stream(), torch.cuda.Stream(), [[], []]

    def run():
        other.wait_stream(main)
        for (pool, table, lens, q), out, s in zip(cases, outs, (main, other)):
            with torch.cuda.stream(s):
                out.extend(sion().kv4_attention(q, pool, table, lens, 2) for _ in range(20))
        main.wait_stream(other)

    g = capture(run, main)
    for _ in range(10):
        g.replay()
        torch.cuda.synchronize()
        for w, out in zip(want, outs):
            assert all(torch.equal(o, w) for o in out)


@pytest.mark.parametrize("op", ["hgemm", "sgemm", "topk", "fork", "backward"])
def test_capture_without_a_call_before(felix, op):
    gen = torch.Generator().manual_seed(3)

    def rand(*shape):
        return torch.randn(*shape, generator=gen).cuda()

    if op in ("hgemm", "sgemm"):  # stream-K: parts and counters
        a, b = rand(1100, 4096), rand(1100, 4096)
        if op == "hgemm":
            a, b = a.half(), b.half()
            f = lambda o: o.append(sion().hgemm_nt(a, b))  # noqa: E731
        else:
            b = b.t().contiguous()
            f = lambda o: o.append(sion().sgemm(a, b))  # noqa: E731
    elif op == "topk":
        x, out = rand(2, 3000001), torch.zeros(2, device="cuda")
        f = lambda o: o.append(topk(felix, x, out).clone())  # noqa: E731
    elif op == "fork":
        s = Fork(11)
        f = lambda o: o.extend(sion().kv4_fork(s.pool, *s.dev, s.page))  # noqa: E731
    else:
        q, k, v, do = (rand(1, 2, 300, 64).half() for _ in range(4))
        out, lse = sion().flash_attention_lse(q, k, v)
        f = lambda o: o.extend(sion().flash_attention_backward(q, k, v, out, lse, do))  # noqa: E731
    got, want = [], []
    g = capture(lambda: f(got), torch.cuda.Stream())
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    f(want)
    torch.cuda.synchronize()
    assert len(got) == len(want) > 0
    for a, b in zip(got, want):
        # sums of several CTAs may be added in another order
        assert (a.double() - b.double()).abs().max() <= 2e-3 * max(b.double().abs().max(), 1e-30)


def topk(felix, x, out):
    felix.check(felix.lib().felix_topk_select(x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1], 5,
                                              1, torch.cuda.current_stream().cuda_stream))
    return out


def test_graphs_that_are_gone_give_their_scratch_back():
    pool, table, lens, q = attend_case(12)
    out = []

    def once():
        out.clear()
        g = capture(lambda: out.append(sion().kv4_attention(q, pool, table, lens, 2)))
        g.replay()
        torch.cuda.synchronize()
        del g

    for _ in range(3):
        once()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(30):  # 10 MB each
        once()
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] < 100 << 20
