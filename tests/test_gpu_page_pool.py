"""Page pool: reserve, release, fork and compact against a plain Python model of
the table, the counts and the cache. Everything here is copied or counted, so
results are compared bit for bit."""
import numpy as np
import pytest

import gemma_kv as gk

pytestmark = pytest.mark.gpu

EVERYTHING = 2**31 - 1


class Pool:
    """The model: page table, counts, lengths and caches as numpy arrays."""

    def __init__(self, layers, pages, page, max_pages, batch, heads, dim, window, seed=0):
        self.shape = (layers, pages, page, max_pages, batch, heads, dim, window)
        self.layers, self.pages, self.page, self.max_pages = layers, pages, page, max_pages
        self.batch, self.window = batch, window
        self.table = np.full((batch, max_pages), -1, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.lens = np.zeros(batch, np.int32)
        rng = np.random.default_rng(seed)
        self.k, self.v = (rng.integers(-2**15, 2**15, (layers, pages, page, heads * dim)).astype(np.int16)
                          for _ in range(2))

    def config(self):
        return gk.make_config(*self.shape)

    def slots(self, lo, hi):
        """Table slots of logical pages lo .. hi - 1."""
        if hi <= lo:
            return []
        if self.window == 0:
            return list(range(lo, hi))
        return [(lo + i) % self.max_pages for i in range(min(hi - lo, self.max_pages))]

    def release(self, first, end):
        for b in range(self.batch):
            f, e = max(int(first[b]), 0), max(int(end[b]), 0)
            last = e // self.page if self.window else min(e // self.page, self.max_pages)
            for s in self.slots(-(-f // self.page), last):
                if self.table[b, s] >= 0:
                    self.refs[self.table[b, s]] -= 1
                    self.table[b, s] = -1

    def reserve(self, first, end):
        wanted = []
        for b in range(self.batch):
            f, e = int(first[b]), int(end[b])
            if e <= f:
                continue
            if f < 0 or (self.window == 0 and -(-e // self.page) > self.max_pages):
                return 2
            wanted += [(b, s) for s in self.slots(f // self.page, -(-e // self.page)) if self.table[b, s] < 0]
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        if len(free) < len(wanted):
            return 1
        for (b, s), p in zip(wanted, free):
            self.table[b, s], self.refs[p] = p, 1
        return 0

    def fork(self, parents, children):
        for p, c in zip(parents, children):
            ok = 0 <= p < self.batch and 0 <= c < self.batch and c not in parents
            if not ok or list(children).count(c) > 1 or (self.table[c] >= 0).any() or self.lens[p] < 0 or \
                    (self.window == 0 and self.lens[p] > self.max_pages * self.page):
                return 2
        free = [p for p in range(self.pages) if self.refs[p] == 0]
        todo = []
        for p, c in zip(parents, children):
            n = int(self.lens[p])
            for s in range(self.max_pages):
                if self.table[p, s] >= 0:
                    if self.window > 0 or (s == n // self.page and n % self.page):
                        todo.append((p, c, s, self.page if self.window > 0 else n % self.page))
        if len(free) < len(todo):
            return 1
        for p, c in zip(parents, children):
            n = int(self.lens[p])
            if self.window == 0:
                for s in range(n // self.page):
                    if self.table[p, s] >= 0:
                        self.table[c, s] = self.table[p, s]
                        self.refs[self.table[p, s]] += 1
            self.lens[c] = n
        for (p, c, s, rows), page in zip(todo, free):
            self.table[c, s], self.refs[page] = page, 1
            for x in (self.k, self.v):
                x[:, page, :rows] = x[:, self.table[p, s], :rows]
        return 0

    def compact(self, sequences, first, kept, refs=True):
        status = []
        for i, (b, f, ks) in enumerate(zip(sequences, first, kept)):
            cap = self.max_pages * self.page
            bad = not 0 <= b < self.batch or f < 0 or list(sequences).count(b) > 1
            bad = bad or any(p < f + j for j, p in enumerate(ks)) or any(x >= y for x, y in zip(ks, ks[1:]))
            bad = bad or any((p - f >= cap if self.window else p >= cap) for p in ks)
            if bad:
                status.append(1)
                continue
            def where(p):
                return self.table[b, (p // self.page) % self.max_pages], p % self.page
            pairs = [(where(p), where(f + j)) for j, p in enumerate(ks)]
            if any(s[0] < 0 or d[0] < 0 for s, d in pairs):
                status.append(2)
            elif refs and any(s != d and self.refs[d[0]] > 1 for s, d in pairs):
                status.append(3)
            else:
                status.append(0)
                for (sp, so), (dp, do) in pairs:
                    for x in (self.k, self.v):
                        x[:, dp, do] = x[:, sp, so]
        return status


class OnDevice:
    def __init__(self, pool, dev):
        import torch
        self.t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        self.config, self.pool = pool.config(), pool
        self.table, self.refs, self.lens = self.t(pool.table), self.t(pool.refs), self.t(pool.lens)
        self.k, self.v = self.t(pool.k), self.t(pool.v)

    def i32(self, x):
        return self.t(np.asarray(x, np.int32))

    def release(self, first, end, **kw):
        gk.check(gk.kv_cache_release_pages(self.table, self.refs, self.config, self.i32(first), self.i32(end), **kw))

    def reserve(self, first, end):
        status = self.i32([77])
        gk.check(gk.kv_cache_reserve_pages(self.table, self.refs, self.config, self.i32(first), self.i32(end), status))
        return int(status)

    def fork(self, parents, children):
        status = self.i32([77])
        gk.check(gk.kv_cache_fork_bf16(self.k, self.v, self.config, self.table, self.refs, self.lens,
                                       self.i32(parents), self.i32(children), len(parents), status))
        return int(status)

    def compact(self, sequences, first, kept, refs=True):
        n = len(sequences)
        off = np.cumsum([0] + [len(k) for k in kept])
        flat = [p for k in kept for p in k]
        status = self.i32([77] * n)
        gk.check(gk.kv_cache_compact_bf16(
            self.k, self.v, self.config, self.table, self.refs if refs else None, self.i32(sequences), self.i32(first),
            self.i32(off), self.i32(flat) if flat else None, n, len(flat), status))
        return status.tolist()

    def check(self, what=""):
        p = self.pool
        for name, want in (("table", p.table), ("refs", p.refs), ("lens", p.lens), ("k", p.k), ("v", p.v)):
            assert np.array_equal(getattr(self, name).cpu().numpy(), want), (what, name)


def make(dev, layers=2, pages=40, page=4, max_pages=8, batch=5, heads=1, dim=64, window=0, seed=0):
    p = Pool(layers, pages, page, max_pages, batch, heads, dim, window, seed)
    return p, OnDevice(p, dev)


@pytest.mark.parametrize("page", [1, 4, 7, 64])
@pytest.mark.parametrize("window", [0, 20])
def test_turnover(dev, page, window):
    """Ranges of every kind, call after call: empty, within a page, past the
    table, wrapped around the ring; pages shared or not."""
    p, d = make(dev, layers=1, page=page, max_pages=8 if window == 0 else 9, batch=6, pages=45, dim=8, window=window)
    rng = np.random.default_rng(page + window)
    for step in range(30):
        room = p.max_pages * page
        first = rng.integers(0, room, 6)
        end = first + rng.integers(-3, room // 2 + 2, 6)
        if window == 0 and step % 5:
            end = np.minimum(end, room)
        if window:
            first, end = first + 1000, end + 1000
        assert d.reserve(first, end) == p.reserve(first, end), step
        d.check((step, "reserve"))
        kind = step % 4
        if kind == 0:
            first, end = first, np.full(6, EVERYTHING)
        elif kind == 1:
            first, end = np.where(rng.random(6) < 0.5, 0, EVERYTHING), np.full(6, EVERYTHING)
        elif kind == 2:
            first, end = rng.integers(-5, room, 6), rng.integers(-5, room + 9, 6)
        d.release(first, end)
        p.release(first, end)
        d.check((step, "release"))


def test_reserve_refusals(dev):
    """Too few pages, a position past the table, a negative one: nothing changes."""
    p, d = make(dev, pages=10)
    assert p.reserve([0] * 5, [8] * 5) == d.reserve([0] * 5, [8] * 5) == 0
    for first, end in (([8] * 5, [9] * 4 + [8]), ([0] * 5, [33] + [0] * 4), ([-1] + [0] * 4, [1] + [0] * 4),
                       ([EVERYTHING - 1] + [0] * 4, [EVERYTHING] + [0] * 4)):
        assert d.reserve(first, end) == p.reserve(first, end) != 0
        d.check((first, end))
    assert d.reserve([5] * 5, [-7] * 5) == 0
    d.check()


def test_release_underflow(dev):
    """A count that is zero already stays zero, whoever else maps the page."""
    p, d = make(dev)
    p.table[0, 0] = p.table[1, 0] = 3
    p.refs[3] = 1
    d = OnDevice(p, dev)
    d.release([0] * 5, [EVERYTHING] * 5)
    assert d.refs.tolist() == [0] * 40 and (d.table == -1).all()


@pytest.mark.parametrize("batch,max_pages,pages", [(64, 700, 44000), (1, 20000, 20001), (4096, 5, 20480)])
def test_reserve_many(dev, batch, max_pages, pages):
    """More pages at once than one list of the kernel's, taken from a pool with holes."""
    p, _ = make(dev, layers=1, batch=batch, max_pages=max_pages, pages=pages, page=1, dim=8)
    rng = np.random.default_rng(1)
    for s in rng.permutation(pages)[:pages // 50]:
        p.refs[s] = 2
    d = OnDevice(p, dev)
    first = rng.integers(0, 3, batch)
    end = np.minimum(max_pages, first + max(1, int(max_pages * 0.9)))
    want = p.reserve(first, end)
    assert d.reserve(first, end) == want == 0
    d.check()
    assert d.reserve([0] * batch, [max_pages] * batch) == p.reserve([0] * batch, [max_pages] * batch)
    d.check()


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512), (1, 8), (2, 24)])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_fork_full(dev, heads, dim, page):
    """Lengths at and around page borders, a hole in a parent's table, two
    children of one parent, grandchildren, pages ahead of the length."""
    p, _ = make(dev, batch=9, max_pages=6, pages=60, page=page, heads=heads, dim=dim)
    p.lens[:4] = [0, 2 * page, min(3 * page + 1, 6 * page), 6 * page]
    assert p.reserve([0] * 9, [0, 3 * page, 5 * page, 6 * page] + [0] * 5) == 0
    p.table[3, 1] = -1  # released in the middle
    p.refs[:] = 0
    for s in p.table[p.table >= 0]:
        p.refs[s] += 1
    d = OnDevice(p, dev)
    for parents, children in (([0, 1, 2, 2], [4, 5, 6, 7]), ([6], [8])):
        assert d.fork(parents, children) == p.fork(parents, children) == 0
        d.check((parents, children))


@pytest.mark.parametrize("page", [1, 16, 64])
def test_fork_ring(dev, page):
    window = 100
    pages = (window + 2 * page - 2) // page
    p, _ = make(dev, batch=4, max_pages=pages, pages=4 * pages, page=page, heads=8, dim=256, window=window)
    p.lens[:2] = [1234, 40]
    assert p.reserve([1100, 0, 0, 0], [1234, 40, 0, 0]) == 0
    d = OnDevice(p, dev)
    assert d.fork([0, 1], [3, 2]) == p.fork([0, 1], [3, 2]) == 0
    d.check()


def test_fork_refusals(dev):
    p, _ = make(dev, pages=12)
    p.lens[:3] = [9, 32, 40]
    assert p.reserve([0] * 5, [9, 32, 0, 0, 0]) == 0
    d = OnDevice(p, dev)
    for parents, children in (([0], [1]), ([0, 0], [3, 3]), ([0, 3], [3, 4]), ([0], [0]), ([5], [3]), ([-1], [3]),
                              ([0], [5]), ([0], [-1]), ([2], [3]), ([0, 0], [2, 3])):
        want = p.fork(parents, children)
        assert d.fork(parents, children) == want != 0, (parents, children)
        d.check((parents, children))


def test_fork_of_a_large_ring_by_windows(dev):
    """More copied pages than one list of the kernel's."""
    p, _ = make(dev, layers=1, batch=40, max_pages=1024, pages=40 * 1024, page=1, dim=8, window=1024)
    p.lens[:20] = 5000
    assert p.reserve([3976] * 20 + [0] * 20, [5000] * 20 + [0] * 20) == 0
    d = OnDevice(p, dev)
    parents, children = list(range(20)), list(range(20, 40))
    assert d.fork(parents, children) == p.fork(parents, children) == 0
    d.check()


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512), (1, 8), (3, 40)])
@pytest.mark.parametrize("page", [1, 5, 64])
def test_compact(dev, heads, dim, page):
    """Lists of every length: none, one, all, every second, tokens that stay."""
    n = 300
    mp = -(-n // page)
    p, _ = make(dev, layers=3, batch=6, max_pages=mp, pages=6 * mp, page=page, heads=heads, dim=dim)
    assert p.reserve([0] * 6, [n] * 6) == 0
    rng = np.random.default_rng(page)
    perm = rng.permutation(6 * mp).astype(np.int32)
    p.table = perm[p.table]
    d = OnDevice(p, dev)
    kept = [[], [n - 1], list(range(1, n)), list(range(50, n, 2)), [3, 4, 5, 9, 200],
            sorted(rng.choice(n, 77, replace=False).tolist())]
    first = [0, 17, 0, 50, 3, 0]
    assert d.compact([3, 0, 1, 2, 5, 4], first, kept) == p.compact([3, 0, 1, 2, 5, 4], first, kept) == [0] * 6
    d.check()


@pytest.mark.parametrize("rows", [4095, 4096, 4097, 9000])
def test_compact_long(dev, rows):
    """More rows than one list of the kernel's."""
    page = 16
    n = rows + 700
    mp = -(-n // page)
    p, _ = make(dev, layers=1, batch=2, max_pages=mp, pages=2 * mp, page=page, heads=1, dim=64)
    assert p.reserve([0, 0], [n, n]) == 0
    d = OnDevice(p, dev)
    rng = np.random.default_rng(rows)
    kept = [sorted(rng.choice(n, rows, replace=False).tolist()), list(range(700, n))]
    assert d.compact([1, 0], [0, 1], kept) == p.compact([1, 0], [0, 1], kept) == [0, 0]
    d.check()


def test_compact_ring(dev):
    p, _ = make(dev, layers=2, batch=2, max_pages=5, pages=10, page=8, window=30)
    assert p.reserve([460, 470], [500, 500]) == 0
    d = OnDevice(p, dev)
    kept = [[490, 491, 495, 499], [471, 480, 499]]
    assert d.compact([0, 1], [489, 470], kept) == p.compact([0, 1], [489, 470], kept) == [0, 0]
    d.check()
    # A list that reaches around the whole ring would meet its own rows.
    assert d.compact([0], [460], [[461, 500]]) == p.compact([0], [460], [[461, 500]]) == [1]
    d.check()


def test_compact_refusals(dev):
    """Each bad request leaves its sequence as it was; the good one beside it is served."""
    p, _ = make(dev, batch=8, pages=64, max_pages=8)
    assert p.reserve([0] * 8, [32, 32, 32, 32, 20, 32, 32, 32]) == 0
    p.refs[p.table[5, 1]] = 2
    d = OnDevice(p, dev)
    seqs = [0, 1, 2, 3, 4, 5, 6, 7]
    first = [4, 4, 0, -1, 0, 4, 0, 3]
    kept = [[6, 5], [3, 9], [8, 8], [5], [3, 21], [9], [40], [7, 9, 31]]
    want = p.compact(seqs, first, kept)
    assert d.compact(seqs, first, kept) == want == [1, 1, 1, 1, 2, 3, 1, 0]
    d.check()
    # Without counts no page is taken to be shared; tokens in place need no page of their own.
    assert d.compact([5], [4], [[9]], refs=False) == p.compact([5], [4], [[9]], refs=False) == [0]
    assert d.compact([5], [4], [[4, 5, 6]]) == p.compact([5], [4], [[4, 5, 6]]) == [0]
    d.check()
    assert d.compact([1, 1, 2], [0, 0, 0], [[5], [9], [9]]) == p.compact([1, 1, 2], [0, 0, 0], [[5], [9], [9]]) == [1, 1, 0]
    assert d.compact([8, -1], [0, 0], [[5], [9]]) == [1, 1]
    d.check()


def test_compact_bad_offsets(dev):
    """Offsets that descend or pass the list are refused without reading past it."""
    import torch
    p, d = make(dev, batch=4)
    assert p.reserve([0] * 4, [32] * 4) == 0
    d = OnDevice(p, dev)
    status = d.i32([77] * 3)
    gk.check(gk.kv_cache_compact_bf16(d.k, d.v, d.config, d.table, d.refs, d.i32([0, 1, 2]), d.i32([0, 0, 0]),
                                      d.i32([0, 3, 2, 9]), d.i32([4, 5, 6]), 3, 3, status))
    torch.cuda.synchronize()
    p.compact([0], [0], [[4, 5, 6]])
    assert status.tolist() == [0, 1, 1]
    d.check()


def test_a_branch_and_its_parent_go_on_apart(dev):
    """Fork, append to both, drop the parent: neither sees the other's tokens."""
    p, _ = make(dev, batch=3, max_pages=6, pages=18, page=4)
    p.lens[0] = 10
    assert p.reserve([0] * 3, [10, 0, 0]) == 0
    d = OnDevice(p, dev)
    assert d.fork([0], [2]) == p.fork([0], [2]) == 0
    rng = np.random.default_rng(5)
    for at in range(10, 15):
        first, end = [at, 0, at], [at + 1, 0, at + 1]
        assert d.reserve(first, end) == p.reserve(first, end) == 0
        row = rng.integers(-2**15, 2**15, (2, 2, 64)).astype(np.int16)
        for layer in range(2):
            gk.check(gk.kv_cache_write_bf16(d.k, d.v, d.config, d.table, d.i32([0, 2]), d.i32([at, at]), 2, layer,
                                            d.t(row[0]), d.t(row[1])))
            for j, b in enumerate((0, 2)):
                p.k[layer, p.table[b, at // 4], at % 4] = row[0, j]
                p.v[layer, p.table[b, at // 4], at % 4] = row[1, j]
        d.check(at)
    for b in (0, 2):
        first = [EVERYTHING] * 3
        first[b] = 0
        d.release(first, [EVERYTHING] * 3)
        p.release(first, [EVERYTHING] * 3)
        d.check(b)
    assert (p.refs == 0).all()


def test_captured_turnover_and_fork(dev):
    """A beam step in a graph: drop the branches, fork anew; replayed with other
    lengths and parents, eager work between."""
    import torch
    p, _ = make(dev, batch=6, max_pages=8, pages=48, page=4)
    p.lens[:3] = [9, 17, 32]
    assert p.reserve([0] * 6, [9, 17, 32, 0, 0, 0]) == 0
    d = OnDevice(p, dev)
    first, end = d.i32([EVERYTHING] * 3 + [0] * 3), d.i32([EVERYTHING] * 6)
    parents, children, status = d.i32([0, 0, 2]), d.i32([3, 4, 5]), d.i32([77])

    def step():
        gk.check(gk.kv_cache_release_pages(d.table, d.refs, d.config, first, end))
        gk.check(gk.kv_cache_fork_bf16(d.k, d.v, d.config, d.table, d.refs, d.lens, parents, children, 3, status))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    rng = np.random.default_rng(0)
    for replay in range(4):
        of = rng.integers(0, 3, 3)
        parents.copy_(d.i32(of))
        graph.replay()
        torch.cuda.synchronize()
        p.release([EVERYTHING] * 3 + [0] * 3, [EVERYTHING] * 6)
        assert p.fork(of.tolist(), [3, 4, 5]) == int(status) == 0
        d.check(replay)
        add = (d.k.float().sum() * 0).item()  # the program's own work between replays
        assert add == 0.0


def test_other_stream(dev):
    import torch
    p, _ = make(dev)
    assert p.reserve([0] * 5, [32] * 5) == 0
    d = OnDevice(p, dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        d.release([9] * 5, [EVERYTHING] * 5)
    d.release([5] * 5, [EVERYTHING] * 5, stream=s)
    s.synchronize()
    p.release([9] * 5, [EVERYTHING] * 5)
    p.release([5] * 5, [EVERYTHING] * 5)
    d.check()


@pytest.mark.parametrize("heads,dim,pages", [(8, 256, 21000), (1, 512, 84000)])
def test_a_cache_of_more_than_four_gigabytes(dev, heads, dim, pages):
    """Fork and compact at the far end of a cache past 2^32 bytes."""
    import torch
    page, layers = 64, 2
    cfg = gk.make_config(layers, pages, page, 4, 2, heads, dim, 0)
    k, v = (torch.empty((layers, pages, page, heads * dim), dtype=torch.int16, device=dev) for _ in range(2))
    assert k[0].numel() * 2 > 2**32
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    refs = torch.ones(pages, dtype=torch.int32, device=dev)
    refs[pages - 2:] = 0
    table = i32([[pages - 3, pages - 5, -1, -1], [-1] * 4])
    gen = torch.Generator(device="cpu").manual_seed(1)
    rows = [torch.randint(-2**15, 2**15, (layers, 2, page, heads * dim), generator=gen).to(torch.int16).to(dev) for _ in range(2)]
    for x, r in zip((k, v), rows):
        x[:, pages - 3], x[:, pages - 5] = r[:, 0], r[:, 1]
    lens, status = i32([100, 0]), i32([77])
    gk.check(gk.kv_cache_fork_bf16(k, v, cfg, table, refs, lens, i32([0]), i32([1]), 1, status))
    assert int(status) == 0 and lens.tolist() == [100, 100]
    assert table[1].tolist() == [pages - 3, pages - 2, -1, -1]
    assert refs[pages - 5:].tolist() == [1, 1, 2, 1, 0]
    for x, r in zip((k, v), rows):
        assert torch.equal(x[:, pages - 2, :36], r[:, 1, :36])
    kept = [66, 70, 71, 99]
    st = i32([77])
    gk.check(gk.kv_cache_compact_bf16(k, v, cfg, table, refs, i32([1]), i32([65]), i32([0, 4]), i32(kept), 1, 4, st))
    assert int(st) == 0
    for x, r in zip((k, v), rows):
        assert torch.equal(x[:, pages - 2, 1:5], r[:, 1, [p - 64 for p in kept]])
        assert torch.equal(x[:, pages - 5], r[:, 1]) and torch.equal(x[:, pages - 3], r[:, 0])


@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("seed", range(10))
def test_random_walk(dev, window, seed):
    """Any of the operators in any order, refused calls among them, over many sequences
    and a pool that runs short; table, counts, lengths and rows after every one."""
    rng = np.random.default_rng(seed)
    page = int(rng.choice([1, 3, 8, 16]))
    max_pages = (window + 2 * page - 2) // page if window else int(rng.integers(1, 70))
    batch = int(rng.integers(2, 60))
    pages = int(rng.integers(max_pages, batch * max_pages + 2))
    heads, dim = [(1, 8), (2, 24), (8, 256)][int(rng.integers(3))]
    p, d = make(dev, layers=2, pages=pages, page=page, max_pages=max_pages, batch=batch, heads=heads, dim=dim,
                window=window, seed=seed)
    cap = max_pages * page
    seen = set()
    for turn in range(30):
        kind = ["reserve", "release", "fork", "compact"][int(rng.integers(4))]
        if kind == "reserve":
            some = rng.random(batch) < 0.2
            end = np.where(some, rng.integers(0, cap + (3 if rng.random() < 0.1 else 1), batch), p.lens)
            first = np.minimum(p.lens, end) if window else np.zeros(batch, int)
            got = d.reserve(first, end)
            assert got == p.reserve(first, end), (turn, kind)
            if got == 0:
                p.lens[:] = np.maximum(p.lens, end)
                d.lens.copy_(d.i32(p.lens))
        elif kind == "release":
            gone = rng.random(batch) < 0.3
            first = np.where(gone, 0, p.lens)
            d.release(first, [EVERYTHING] * batch)
            p.release(first, [EVERYTHING] * batch)
            p.lens[gone] = 0
            d.lens.copy_(d.i32(p.lens))
            got = 0
        elif kind == "fork":
            empty = [b for b in range(batch) if (p.table[b] < 0).all()]
            n = int(rng.integers(1, 6))
            held = [b for b in range(batch) if b not in empty] or [0]
            children = [int(c) for c in rng.permutation(empty if empty and rng.random() < 0.9 else batch)[:n]]
            parents = [int(x) for x in rng.choice(held, len(children))]
            got = d.fork(parents, children)
            assert got == p.fork(parents, children), (turn, kind)
        else:
            who = [int(b) for b in rng.permutation(batch)[:int(rng.integers(1, 5))]]
            first = [int(rng.integers(0, max(int(p.lens[b]), 1))) for b in who]
            kept = [sorted(int(x) for x in rng.choice(np.arange(f, max(int(p.lens[b]), f + 1)),
                                                      int(rng.integers(0, max(int(p.lens[b]) - f, 1))), replace=False))
                    for b, f in zip(who, first)]
            got = d.compact(who, first, kept)
            assert got == p.compact(who, first, kept), (turn, kind)
            got = max(got)
        seen.add((kind, got))
        d.check((turn, kind))
    assert len({kind for kind, _ in seen}) == 4, seen


def test_compact_requests_that_break_several_rules(dev):
    """The lowest code, on every run, wherever in a long list the rules are broken."""
    n, page = 4500, 4
    mp = n // page
    p, _ = make(dev, layers=1, pages=6 * mp, max_pages=mp, batch=6, dim=8, page=page)
    assert p.reserve([0] * 6, [n] * 6) == 0
    for b in range(6):
        p.refs[p.table[b, 30]] = 2            # positions 120 .. 123
    for b in (0, 1, 2, 4):
        p.refs[p.table[b, 700]] = 0
        p.table[b, 700] = -1                  # positions 2800 .. 2803
    kept = [list(range(1, n)) for _ in range(6)]
    kept[1][4000] = 4000                      # not behind the one before
    kept[3][0] = -1
    kept[4] = [2800, 2801] + list(range(4000, 4400))
    d = OnDevice(p, dev)
    seqs, first = [0, 1, 2, 3, 4, 5], [0, 0, 0, 0, 100, 0]
    for turn in range(20):
        assert d.compact(seqs, first, kept) == p.compact(seqs, first, kept) == [2, 1, 2, 1, 2, 3]
    assert d.compact([2, 5, 2], [0, 0, 0], [kept[2], kept[5], [5]]) == [1, 3, 1]
    d.check()


def test_reserve_refuses_shared_pages_that_will_be_written(dev):
    """A branch, or its parent, that was shortened into their shared pages."""
    p, _ = make(dev, batch=6, max_pages=6, pages=14, page=4)
    p.lens[0] = 18
    assert p.reserve([0] * 6, [18] + [0] * 5) == 0
    d = OnDevice(p, dev)
    assert d.fork([0, 0], [1, 2]) == p.fork([0, 0], [1, 2]) == 0
    d.release([EVERYTHING, 10] + [EVERYTHING] * 4, [EVERYTHING] * 6)
    p.release([EVERYTHING, 10] + [EVERYTHING] * 4, [EVERYTHING] * 6)
    p.lens[1] = 10
    d.lens.copy_(d.i32(p.lens))
    d.check()
    nothing, one = [0] * 6, lambda b, x: [x if i == b else 0 for i in range(6)]  # noqa: E731
    for b, at in ((1, 10), (1, 11), (1, 8), (0, 15), (2, 1)):
        assert d.reserve(one(b, at), one(b, at + 1)) == 3, (b, at)
        d.check((b, at))
    # Before too few pages, behind bad ranges; from 0 on nothing is taken to be written.
    assert d.reserve([0, 10, 0, 0, 0, 0], [0, 11, 0, 24, 24, 24]) == 3
    assert d.reserve([0, 10, 0, -1, 0, 0], [0, 11, 0, 4, 0, 0]) == 2
    assert d.reserve(nothing, [18, 10, 18, 0, 0, 0]) == 0
    assert d.reserve([18, 0, 18, 0, 0, 0], [20, 0, 19, 0, 0, 0]) == 0  # pages of their own
    d.check()
    # The way on: a branch of the shortened branch has the begun page as its own.
    assert d.fork([1], [3]) == p.fork([1], [3]) == 0
    d.release([EVERYTHING, 0] + [EVERYTHING] * 4, [EVERYTHING] * 6)
    p.release([EVERYTHING, 0] + [EVERYTHING] * 4, [EVERYTHING] * 6)
    assert d.reserve(one(3, 10), one(3, 14)) == p.reserve(one(3, 10), one(3, 14)) == 0
    d.check()
    # Shared no more, the pages may be written again.
    d.release([EVERYTHING, 0, 0, 0, 0, 0], [EVERYTHING] * 6)
    p.release([EVERYTHING, 0, 0, 0, 0, 0], [EVERYTHING] * 6)
    assert d.reserve(one(0, 15), one(0, 16)) == 0
    d.check()


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("seed", range(4))
def test_appends_never_reach_another_sequence(dev, page, seed):
    """Branches that grow, shrink to anywhere and branch again: after every step each
    sequence's rows in the cache are its own tokens."""
    import torch
    rng = np.random.default_rng(seed)
    batch, max_pages = 7, 40 // page + 1
    pages, dim, cap = 5 * max_pages, 8, max_pages * page
    cfg = gk.make_config(1, pages, page, max_pages, batch, 1, dim, 0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, refs = torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev), i32([0] * pages)
    k, v = (torch.zeros((pages, page, dim), dtype=torch.int16, device=dev) for _ in range(2))
    lengths, status = i32([0] * batch), i32([77])
    tokens, count, codes = [[] for _ in range(batch)], 0, set()

    def release(first):
        gk.check(gk.kv_cache_release_pages(table, refs, cfg, i32(first), i32([EVERYTHING] * batch)))

    def fork(parent, child):
        lengths.copy_(i32([len(x) for x in tokens]))
        gk.check(gk.kv_cache_fork_bf16(k, v, cfg, table, refs, lengths, i32([parent]), i32([child]), 1, status))
        if int(status) == 0:
            tokens[child] = list(tokens[parent])
        return int(status)

    for turn in range(300):
        b = int(rng.integers(batch))
        kind = ["append", "append", "fork", "shorten", "drop"][int(rng.integers(5))]
        if kind == "append":
            n = int(rng.integers(1, 2 * page + 3))
            if len(tokens[b]) + n > cap:
                continue
            first = [len(x) for x in tokens]
            end = [f + n if i == b else f for i, f in enumerate(first)]
            for attempt in range(2):
                gk.check(gk.kv_cache_reserve_pages(table, refs, cfg, i32(first), i32(end), status))
                codes.add(int(status))
                empty = [c for c in range(batch) if not tokens[c]]
                if int(status) != 3 or not empty or attempt:
                    break
                if fork(b, empty[0]) != 0:
                    break
                release([0 if i == b else EVERYTHING for i in range(batch)])
                tokens[b], b = [], empty[0]
                first = [len(x) for x in tokens]
                end = [f + n if i == b else f for i, f in enumerate(first)]
            if int(status) == 0:
                new = list(range(count + 1, count + 1 + n))
                count += n
                rows = i32(new).to(torch.int16)[:, None].expand(n, dim).contiguous()
                at = [len(tokens[b]) + j for j in range(n)]
                gk.check(gk.kv_cache_write_bf16(k, v, cfg, table, i32([b] * n), i32(at), n, 0, rows, -rows))
                tokens[b] += new
        elif kind == "fork":
            empty = [c for c in range(batch) if not tokens[c] and c != b]
            if empty and tokens[b]:
                release([0 if i == empty[0] else EVERYTHING for i in range(batch)])
                fork(b, empty[0])
        else:
            tokens[b] = tokens[b][:int(rng.integers(0, len(tokens[b]) + 1))] if kind == "shorten" else []
            release([len(x) for x in tokens])
        held = table.cpu().numpy()
        for c in range(batch):
            if tokens[c]:
                at = np.arange(len(tokens[c]))
                rows = torch.from_numpy(held[c, at // page].astype(np.int64)).to(dev)
                offset = torch.from_numpy(at % page).to(dev)
                want = i32(tokens[c]).to(torch.int16)[:, None].expand(-1, dim)
                assert torch.equal(k[rows, offset], want) and torch.equal(v[rows, offset], -want), (turn, kind, c)
        mapped = np.bincount(held[held >= 0], minlength=pages)
        assert np.array_equal(refs.cpu().numpy(), mapped), (turn, kind)
    assert 0 in codes and (3 in codes) == (page > 1)  # whole pages are never gone on in
