"""The library's scratch: calls from several host threads, on one stream and on each
thread's own."""
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
