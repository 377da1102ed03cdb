"""fork_pages, reserve_pages, release_pages, compact_pages and copy_pages against the oracle.

Whole numbers and copied bytes: everything is compared exactly."""

import numpy as np
import pytest
import torch

import gemma4_fa4_amd as g4
from oracle import paged_cache as pc
from paged_testutil import DEV, E4M3, cu_of, empty_cache, ints

pytestmark = pytest.mark.gpu


class Pool:
    """The same pool twice: lists for the oracle, device tensors for the calls."""

    def __init__(self, seed, batch, width, pages, page):
        rng = self.rng = np.random.default_rng(seed)
        self.page = page
        lens = [int(x) for x in rng.integers(0, (width - 1) * page + 1, batch)]
        ids = [int(x) for x in rng.permutation(pages)]
        self.table, self.lens, self.refs = [], [], [0] * pages
        for n in lens:
            used = pc.pages_of(n, page)
            if used > len(ids):
                n = used = 0
            row, ids = ids[:used], ids[used:]
            for p in row:
                self.refs[p] = 1
            self.table.append(row + [-1] * (width - used))
            self.lens.append(n)
        self.upload()

    def upload(self):
        self.t, self.l, self.r = ints(self.table), ints(self.lens), ints(self.refs)

    def same(self):
        assert self.t.tolist() == self.table
        assert self.l.tolist() == self.lens
        assert self.r.tolist() == self.refs
        for p, n in enumerate(self.refs):  # every reference is a row's
            assert n >= 0

    def fork(self, parents):
        pc.fork(self.table, self.lens, self.refs, parents, self.page)
        g4.fork_pages(self.t, self.l, self.r, ints(parents), page_size=self.page)
        self.same()

    def reserve(self, new_lens):
        want = pc.reserve(self.table, self.lens, self.refs, new_lens, self.page)
        got = g4.reserve_pages(self.t, self.l, self.r, ints(new_lens), page_size=self.page)
        assert [x.tolist() for x in got] == [list(x) for x in want]
        self.same()
        return want

    def release(self, keep, window=None, sinks=0):
        pc.release(self.table, self.lens, self.refs, keep, self.page, window or 0, sinks)
        g4.release_pages(self.t, self.l, self.r, ints(keep), page_size=self.page,
                         sliding_window=window, num_sinks=sinks)
        self.same()

    def compact(self):
        want = pc.compact(self.table, self.refs)
        got = g4.compact_pages(self.t, self.r)
        assert [x.tolist() for x in got] == [list(x) for x in want]
        self.same()
        return got


SHAPES = [  # seed, batch, width, pages, page size
    (1, 1, 1, 1, 32),
    (2, 1, 5, 3, 64),
    (3, 7, 6, 50, 32),
    (4, 70, 4, 200, 128),
    (5, 33, 40, 9000, 32),  # several rounds of the ordering workgroup's scans
    (6, 1500, 3, 5000, 256),  # more rows than its threads
    (7, 300, 60, 40000, 32),  # more entries than one workgroup forks; scans of several steps
]


@pytest.mark.parametrize("seed,batch,width,pages,page", SHAPES)
def test_a_life_of_random_calls(seed, batch, width, pages, page):
    pool = Pool(seed, batch, width, pages, page)
    rng = pool.rng
    for _ in range(4):
        parents = rng.integers(-1, batch + 1, batch)
        parents = np.where(rng.random(batch) < 0.6, np.arange(batch), parents)
        pool.fork([int(x) for x in parents])
        pool.reserve([n + int(x) for n, x in zip(pool.lens, rng.integers(0, 3, batch))])
        pool.reserve([n + int(x) for n, x in zip(pool.lens, rng.integers(-5, 3 * page, batch))])
        keep = [n - int(x) for n, x in zip(pool.lens, rng.integers(-2, page + 2, batch))]
        pool.release(keep, *((page + 9, 3) if rng.random() < 0.5 else ()))
        pool.compact()


def test_a_pool_that_runs_out():
    pool = Pool(7, 4, 6, 40, 32)
    pool.release([0] * 4)
    src, dst, granted = pool.reserve([6 * 32, 7 * 32, 6 * 32, 1])  # row 1 is wider than the table
    assert granted == [1, 0, 1, 1]
    pool = Pool(8, 3, 4, 5, 32)
    pool.release([0] * 3)
    assert pool.reserve([64, 128, 32])[2] == [1, 0, 0]  # 2, then 4 of 3 left; ranks are not reused
    assert pool.reserve([64, 96, 32])[2] == [1, 1, 0]


def test_nothing_free_and_nothing_asked():
    pool = Pool(9, 2, 3, 6, 32)
    pool.release([0, 0])
    pool.reserve([96, 96])
    assert pool.reserve([96, 96])[2] == [1, 1]
    assert pool.reserve([97, 97])[2] == [0, 0]
    pool.compact()


@pytest.mark.parametrize("entry", [-7, -2])
def test_entries_that_are_no_pages(entry):
    # tables with IDs out of range: counts of pages are left alone, nothing else is touched
    table, lens, refs = [[9, entry, 1], [2147483647, 0, -1]], [96, 64], [1, 1, 0, 0]
    t, l, r = ints(table), ints(lens), ints(refs)
    guard = torch.full((8,), 7, dtype=torch.int32, device=DEV)
    g4.fork_pages(t, l, r, ints([0, 0]), page_size=32)
    pc.fork(table, lens, refs, [0, 0], 32)
    assert (t.tolist(), l.tolist(), r.tolist()) == (table, lens, refs)
    g4.release_pages(t, l, r, ints([0, 33]), page_size=32)
    pc.release(table, lens, refs, [0, 33], 32)
    assert (t.tolist(), l.tolist(), r.tolist()) == (table, lens, refs)
    g4.compact_pages(t, r)
    assert guard.eq(7).all()


@pytest.mark.parametrize("d,heads,page", [(256, 3, 32), (512, 4, 64), (256, 16, 256), (512, 1, 32)])
def test_copies(d, heads, page):
    cache = empty_cache(20, heads, page, d)
    g = torch.Generator().manual_seed(d + page)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.randn(t.shape, generator=g))
    was = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    src, dst = [3, -1, 19, 5, 3, 20, 4, 7], [0, 1, 2, 5, 8, 9, -1, 2147483647]
    g4.copy_pages(cache, ints(src), ints(dst))
    for t, x in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), was):
        want = x.clone()
        for s, e in ((3, 0), (19, 2), (3, 8)):
            want[e] = x[s]
        as_bytes = (lambda y: y.view(torch.uint8)) if t.dtype == E4M3 else (lambda y: y)
        assert torch.equal(as_bytes(t), as_bytes(want))
    g4.copy_pages(cache, ints([]), ints([]))


def test_a_graph_and_another_stream():
    # a captured serving step (lengths + 1, reserve, copy) against eager calls of the oracle
    page, batch = 32, 5
    pool = Pool(11, batch, 8, 60, page)
    pool.release([40, 40, 31, 32, 1])
    pool.fork([0, 0, 2, 2, 4])
    cache = empty_cache(60, 2, page, 256)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(1)
    cache.k_scale.copy_(torch.arange(60.0)[:, None, None].expand_as(cache.k_scale))
    cache.v_scale.fill_(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        new = pool.l + 1  # (allocated before the capture)
        with torch.cuda.graph(graph, stream=side):
            torch.add(pool.l, 1, out=new)
            src, dst, granted = g4.reserve_pages(pool.t, pool.l, pool.r, new, page_size=page)
            g4.copy_pages(cache, src, dst)
    torch.cuda.synchronize()
    for _ in range(40):
        want = pc.reserve(pool.table, pool.lens, pool.refs, [n + 1 for n in pool.lens], page)
        before = cache.k_scale.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert [src.tolist(), dst.tolist(), granted.tolist()] == [list(x) for x in want]
        pool.same()
        for s, d in zip(*want[:2]):
            if d >= 0:
                before[d] = before[s]
        assert torch.equal(cache.k_scale, before)


def test_append_after_a_fork_leaves_the_parent():
    page = 32
    table, lens, refs = ints([[2, 0, -1], [-1, -1, -1]]), ints([40, 0]), ints([1, 0, 1, 0, 0])
    cache = empty_cache(5, 2, page, 256)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(41, 2, 256, generator=g).to(torch.bfloat16).to(DEV)
    g4.paged_cache_append(cache, x[:40], x[:40], table, lens, ints([0, 40, 40]))
    before = g4.paged_cache_gather(cache, table, lens, ints([0, 40, 40]), 40)
    g4.fork_pages(table, lens, refs, ints([0, 0]), page_size=page)
    src, dst, granted = g4.reserve_pages(table, lens, refs, ints([40, 41]), page_size=page)
    g4.copy_pages(cache, src, dst)
    big = 100 * x[40:]  # raises the scale of the copied block
    g4.paged_cache_append(cache, big, big, table, lens, ints([0, 0, 1]))
    after = g4.paged_cache_gather(cache, table, lens, ints(cu_of([40, 41])), 81)
    for a, b in zip(before, after):
        assert torch.equal(a, b[:40])
        assert torch.equal(b[:32], b[40:72]) and not torch.equal(b[32:40], b[72:80])
