"""Pages that several sequences hold, on the GPU (qvx_kv_fork, qvx_kv_free, qvx_kv_compact, qvx_kv_copy), against the same
bookkeeping in plain Python: whole numbers, so equal."""
from __future__ import annotations

import numpy as np
import pytest

import qorvix_amd as qvx

pytestmark = pytest.mark.gpu


class Pool:
    """Rows of a page table and their pages, on the host."""

    def __init__(self, rows, width, page, n_pages, seed=0):
        self.r = np.random.default_rng(seed)
        self.page, self.n_pages = page, n_pages
        self.table = np.full((rows, width), -1, np.int32)
        self.lens = np.zeros(rows, np.int32)
        self.extra = np.zeros(n_pages, np.int32)
        self.free = self.r.permutation(n_pages).astype(np.int32)
        self.taken = 0

    def fill(self, lens):
        for b, n in enumerate(lens):
            k = -(-n // self.page)
            self.table[b, :k] = self.free[self.taken: self.taken + k]
            self.taken += k
            self.lens[b] = n

    def fork(self, pairs):
        out, extra = [], self.extra.copy()
        for a, b in pairs:
            n = int(self.lens[a])
            full, left = divmod(n, self.page)
            self.table[b] = -1
            self.table[b, :full] = self.table[a, :full]
            for p in self.table[a, :full]:
                if 0 <= p < self.n_pages:
                    extra[p] += 1
            if left:
                fresh = self.free[self.taken]
                self.taken += 1
                self.table[b, full] = fresh
                out.append((self.table[a, full], fresh))
            self.lens[b] = n
        self.extra = extra
        return out

    def release(self, rows, begin=None, end=None):
        gone = set()
        for i, b in enumerate(rows):
            lo, hi = (0, self.table.shape[1]) if begin is None else (max(begin[i], 0), min(end[i], self.table.shape[1]))
            for c in range(lo, hi):
                p = self.table[b, c]
                if p < 0:
                    continue
                self.table[b, c] = -1
                if p >= self.n_pages:
                    continue
                if self.extra[p]:
                    self.extra[p] -= 1
                else:
                    assert p not in gone
                    gone.add(int(p))
            if begin is None:
                self.lens[b] = 0
        self.taken -= len(gone)
        self.free[self.taken: self.taken + len(gone)] = sorted(gone)

    def compact(self):
        names = set(self.free[self.taken:].tolist())
        used = [p for p in range(self.n_pages) if p not in names]
        u = len(used)
        src, dst = [p for p in used if p >= u], sorted(p for p in names if p < u)
        to = dict(zip(src, dst))
        self.table = np.vectorize(lambda p: to.get(p, p), otypes=[np.int32])(self.table)
        for a, b in to.items():
            self.extra[b], self.extra[a] = self.extra[a], 0
        self.free[self.taken:] = np.arange(u, u + len(self.free) - self.taken)
        return list(zip(src, dst)), u


class Dev:
    def __init__(self, torch, p):
        self.torch = torch
        self.page = p.page
        self.table, self.lens, self.extra, self.free = (torch.from_numpy(x.copy()).cuda() for x in (p.table, p.lens, p.extra, p.free))
        self.taken = torch.tensor([p.taken, 0], dtype=torch.int32, device="cuda")

    def ints(self, v):
        return self.torch.tensor(list(v), dtype=self.torch.int32, device="cuda")

    def fork(self, pairs):
        return qvx.kv_fork_t(self.ints(a for a, _ in pairs), self.ints(b for _, b in pairs), self.table, self.page, self.lens,
                             self.extra, self.free, self.taken)

    def release(self, rows, begin=None, end=None):
        qvx.kv_free_t(self.ints(rows), self.table, self.lens, self.extra, self.free, self.taken,
                      None if begin is None else self.ints(begin), None if end is None else self.ints(end))

    def same(self, p, status=0):
        assert self.taken.tolist() == [p.taken, status]
        for x, y in ((self.table, p.table), (self.lens, p.lens), (self.extra, p.extra), (self.free, p.free)):
            assert np.array_equal(x.cpu().numpy(), y)


@pytest.mark.parametrize("page,n_pages,longest,rows", [(16, 300, 200, 12), (1, 5000, 150, 20), (24, 20000, 4000, 60),
                                                       (8, 70000, 9000, 24), (128, 1, 100, 1)])
def test_forks_and_releases(cuda, page, n_pages, longest, rows):
    r = np.random.default_rng(page)
    p = Pool(2 * rows, -(-longest // page) + 1, page, n_pages, seed=page)
    lens = r.integers(0, longest + 1, rows)
    lens[0] = longest if n_pages > 1 else 0
    if rows > 2:
        lens[1], lens[2] = 0, longest // page * page
    p.fill(lens)
    d = Dev(cuda, p)
    live, spare = list(range(rows)), list(range(rows, 2 * rows))
    for step in range(4):
        n = int(r.integers(1, len(spare) + 1))
        to = [int(x) for x in r.permutation(spare)[:n]]
        pairs = [(int(r.choice(live)), b) for b in to]
        want = p.fork(pairs)
        got, count = d.fork(pairs)
        assert count.tolist() == [len(want)] and got.cpu().numpy()[: len(want)].tolist() == [list(map(int, x)) for x in want]
        d.same(p)
        live += to
        spare = [x for x in spare if x not in to]
        gone = [int(x) for x in r.permutation(live)[: rows]] if len(live) > rows else live[:1]
        p.release(gone)
        d.release(gone)
        d.same(p)
        live = [x for x in live if x not in gone]
        spare += gone
    rest = live[: max(1, len(live))] or spare[:1]
    p.release(rest)
    d.release(rest)
    d.same(p)


def test_release_behind_a_window(cuda):
    p = Pool(8, 40, 16, 400, seed=4)
    p.fill([600, 640, 33, 0, 17])
    p.fork([(0, 5), (1, 6)])
    d = Dev(cuda, p)
    begin, end = [1, 3, 0, -5, 2 ** 31 - 1, 10], [30, 60, 0, 9, 2 ** 31 - 1, 3]
    p.release([0, 1, 2, 3, 4, 5], begin, end)
    d.release([0, 1, 2, 3, 4, 5], begin, end)
    d.same(p)
    p.release([0, 1, 5, 6])
    d.release([0, 1, 5, 6])
    d.same(p)


def test_one_row_twice_is_released_once(cuda):
    for n_pages in (60, 40000):
        p = Pool(3, 8, 4, n_pages, seed=1)
        p.fill([30, 9])
        d = Dev(cuda, p)
        p.release([0])
        d.release([0, 0, 0])
        d.same(p)


def test_statuses(cuda):
    torch = cuda
    p = Pool(6, 4, 8, 9, seed=2)
    p.fill([30, 20])  # seven pages of nine
    d = Dev(torch, p)
    pairs, count = d.fork([(0, 2), (1, 3), (0, 4)])  # three fresh pages, two left
    d.same(p, qvx.MAP_PAGES)
    assert count.tolist() == [0] and (pairs == -1).all()
    for bad in ([(0, 6)], [(0, -1)], [(7, 2)], [(0, 0)], [(0, 2), (-1, 3)]):
        d.fork(bad)
        d.same(p, qvx.MAP_SEQUENCE)
    d.lens[1] = -3
    d.fork([(1, 2)])
    assert d.taken.tolist() == [7, qvx.MAP_NEGATIVE]
    d.lens[1] = 33
    d.fork([(1, 2)])
    assert d.taken.tolist() == [7, qvx.MAP_COLUMNS]
    d.lens[1] = 20
    p.fork([(0, 2), (1, 3)])
    d.fork([(0, 2), (1, 3)])
    d.same(p)
    p.release([2])
    d.release([2, 9])  # a row that is not there is passed over
    d.same(p, qvx.MAP_SEQUENCE)
    d.taken[0] = 2  # fewer than come back: five of row 0 and 2's pages, three lost
    d.release([0, 1, 3])
    assert d.taken.tolist() == [0, qvx.MAP_PAGES]
    assert (d.table == -1).all() and (d.extra == 0).all()


def test_fork_with_totals_elsewhere(cuda):
    torch = cuda
    p = Pool(4, 5, 16, 30, seed=3)
    p.fill([70, 16])
    d = Dev(torch, p)
    out, n_pairs = d.ints([-9, -9]), d.ints([0])
    pairs = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    a, b = d.ints([0, 1]), d.ints([2, 3])
    rc = qvx.kv_fork(a.data_ptr(), b.data_ptr(), 2, d.table.data_ptr(), 4, 5, 16, d.lens.data_ptr(), d.extra.data_ptr(), 30,
                     d.free.data_ptr(), 30, d.taken.data_ptr(), out.data_ptr(), pairs.data_ptr(), n_pairs.data_ptr(),
                     torch.cuda.current_stream().cuda_stream)
    assert rc == qvx.OK
    before = p.taken
    p.fork([(0, 2), (1, 3)])
    assert d.taken.tolist() == [before, 0] and out.tolist() == [p.taken, 0] and n_pairs.tolist() == [1]


@pytest.mark.parametrize("n_pages,share", [(1, 0.0), (2, 0.5), (31, 0.4), (256, 0.5), (257, 0.9), (4500, 0.6), (70000, 0.3)])
def test_compaction(cuda, n_pages, share):
    p = Pool(9, max(n_pages // 6, 1), 4, n_pages, seed=n_pages)
    each = int(share * n_pages) // 8
    p.fill([each * 4] * 8)
    if each:
        p.fork([(3, 8)])
    d = Dev(cuda, p)
    pairs, u = p.compact()
    got, moved = qvx.kv_compact_t(d.table, d.extra, d.free, d.taken)
    assert moved.tolist() == [len(pairs), u]
    assert got.cpu().numpy()[: len(pairs)].tolist() == [list(x) for x in pairs]
    d.same(p)
    again, moved = qvx.kv_compact_t(d.table, d.extra, d.free, d.taken)
    assert moved.tolist() == [0, u]
    d.same(p)


def test_compaction_elsewhere_keeps_its_inputs(cuda):
    torch = cuda
    p = Pool(5, 60, 4, 300, seed=8)
    p.fill([100, 37, 0, 200, 5])
    d = Dev(torch, p)
    outs = [torch.zeros_like(x) for x in (d.table, d.extra, d.free)]
    pairs, moved = torch.zeros((150, 2), dtype=torch.int32, device="cuda"), d.ints([0, 0])
    rc = qvx.kv_compact(d.table.data_ptr(), outs[0].data_ptr(), 5, 60, d.extra.data_ptr(), outs[1].data_ptr(), 300,
                        d.free.data_ptr(), outs[2].data_ptr(), 300, d.taken.data_ptr(), pairs.data_ptr(), moved.data_ptr(),
                        torch.cuda.current_stream().cuda_stream)
    assert rc == qvx.OK
    d.same(p)
    p.compact()
    d.table, d.extra, d.free = outs
    d.same(p)


@pytest.mark.parametrize("t,page,hk,d,pad", [(qvx.F16, 16, 8, 128, 0), (qvx.F32, 3, 1, 8, 16), (qvx.Q8_0, 7, 3, 32, 48),
                                             (qvx.BF16, 128, 4, 64, 0)])
@pytest.mark.parametrize("layers", [1, 3, 70])
def test_copies(cuda, t, page, hk, d, pad, layers):
    torch = cuda
    size, n = qvx.kv_page_bytes(t, hk, page, d), 23
    g = torch.Generator(device="cuda").manual_seed(5)
    pool = torch.randint(0, 256, (layers, n, 2 * (size + pad)), generator=g, device="cuda", dtype=torch.uint8)
    caches = [qvx.KvCache.of(x[:, :size], x[:, size + pad: 2 * size + pad], t, page, hk, d) for x in pool]
    want = pool.clone()
    pairs = [(3, 7), (0, 22), (22, 1), (5, 5), (-1, 4), (6, 23), (11, 2), (12, 8), (13, 9)]
    keep = torch.zeros(2 * (size + pad), dtype=torch.bool, device="cuda")
    keep[:size] = keep[size + pad: 2 * size + pad] = True
    pairs[2] = (10, 1)  # no page read that is written
    for a, b in [x for i, x in enumerate(pairs[:7]) if 0 <= x[0] < n and 0 <= x[1] < n]:
        want[:, b] = torch.where(keep, pool[:, a], pool[:, b])
    dev = torch.tensor(pairs, dtype=torch.int32, device="cuda")
    qvx.kv_copy_t(caches, dev, torch.tensor([7], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool, want)
    for a, b in pairs[7:]:
        want[:, b] = torch.where(keep, want[:, a], want[:, b])
    qvx.kv_copy_t(caches, dev)
    assert torch.equal(pool, want)
    qvx.kv_copy_t(caches, dev, torch.tensor([-4], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool, want)


def test_a_beam_step_captured(cuda):
    """Forks, copies and releases in one graph, against the same calls one by one."""
    torch = cuda
    p = Pool(8, 12, 8, 80, seed=9)
    p.fill([40, 37, 50, 61])
    p.fork([(0, 4)])
    p.release([4])
    d, e = Dev(torch, p), Dev(torch, p)
    size = qvx.kv_page_bytes(qvx.F16, 2, 8, 64)
    pools = [torch.randint(0, 255, (80, 2 * size), device="cuda", dtype=torch.uint8)]
    pools.append(pools[0].clone())
    caches = [[qvx.KvCache.of(x[:, :size], x[:, size:], qvx.F16, 8, 2, 64)] for x in pools]
    rows = [x.ints([0, 1, 2, 3]) for x in (d, d)]
    source, to = d.ints([0, 0, 2, 3]), d.ints([4, 5, 6, 7])

    def step(x, pool):
        pairs, count = qvx.kv_fork_t(source, to, x.table, 8, x.lens, x.extra, x.free, x.taken)
        qvx.kv_copy_t(caches[pool], pairs, count)
        qvx.kv_free_t(rows[0], x.table, x.lens, x.extra, x.free, x.taken)

    warm = Dev(torch, p)
    step(warm, 1)
    torch.cuda.synchronize()
    pools[1].copy_(pools[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(d, 0)
    for i, (a, b, gone) in enumerate([([0, 0, 2, 3], [4, 5, 6, 7], [0, 1, 2, 3]), ([4, 6, 6, 7], [0, 1, 2, 3], [4, 5, 6, 7]),
                                      ([1, 1, 1, 1], [4, 5, 6, 7], [0, 1, 2, 3])]):
        source.copy_(d.ints(a))
        to.copy_(d.ints(b))
        rows[0].copy_(d.ints(gone))
        graph.replay()
        torch.cuda.synchronize()
        step(e, 1)
        p.fork(list(zip(a, b)))
        p.release(gone)
        d.same(p)
        e.same(p)
        assert torch.equal(pools[0], pools[1]), i
