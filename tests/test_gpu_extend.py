"""Attention of ragged new tokens over the paged cache against its definition in
64 bits.

Tolerance, before any run: the output is rounded once to bf16 (2^-8 |o|). Each
weight is rounded to bf16 before it meets V (2^-8 of sum w|v|). A score is a
fp32 sum of D products, off by at most D 2^-24 sum |q k| scale, which shifts its
weight by that factor, in the numerator and, at most as much, in the sum; sums
over n keys in fp32 add n 2^-24 of sum w|v| each."""
import math

import numpy as np
import pytest

import gemma_kv as gk

pytestmark = pytest.mark.gpu

NAN = float("nan")


class Batch:
    """A ragged batch, its cache and table. What no row sees is NaN: slots
    behind the prior keys, unmapped and unused pages."""

    def __init__(self, dev, heads, dim, rows, prior, page=16, window=0, sinks=0, ring=False, layers=1, seed=0,
                 spread=1.0, spare=3, max_pages=None, released=True, extra_rows=0, holes=()):
        import torch
        self.dev, self.heads, self.dim, self.rows, self.prior = dev, heads, dim, rows, prior
        self.page, self.window, self.sinks, self.ring, self.layers = page, window, sinks, ring, layers
        self.batch, self.total = len(rows), sum(rows) + extra_rows
        gen = torch.Generator(device="cpu").manual_seed(seed + 1)
        normal = lambda *s: torch.randn(s, generator=gen, dtype=torch.float32).mul_(spread).bfloat16()  # noqa: E731
        longest = max(n + p for n, p in zip(rows, prior))
        if max_pages is None:
            max_pages = (window + 2 * page - 2) // page if ring else max(1, -(-longest // page))
        self.max_pages = max_pages
        used = []
        for b, (n, p) in enumerate(zip(rows, prior)):
            lo = max(0, p - window + 1) if window else 0
            for j in range(-(-p // page)):
                if ring and j < -(-p // page) - max_pages:
                    continue
                if not ring and released and window and (j + 1) * page <= lo and j * page >= sinks:
                    continue
                if (b, j) not in holes:
                    used.append((b, j))
        self.pages = len(used) + spare
        order = torch.randperm(self.pages, generator=gen)
        table = torch.full((self.batch, max_pages), -1, dtype=torch.int32)
        ck, cv = (torch.full((layers, self.pages, page, heads, dim), NAN, dtype=torch.bfloat16) for _ in range(2))
        for (b, j), physical in zip(used, order):
            table[b, j % max_pages] = int(physical)
        for (b, j), physical in zip(used, order):  # a ring's slot holds its newest page
            live = min(page, prior[b] - j * page)
            if ring and j * page + page <= prior[b] - max_pages * page:
                continue
            ck[:, physical, :live], cv[:, physical, :live] = normal(layers, live, heads, dim), normal(layers, live, heads, dim)
            if ring and live < page and j >= max_pages:
                # Behind the newest token the ring still holds the page of a turn before.
                ck[:, physical, live:], cv[:, physical, live:] = (normal(layers, page - live, heads, dim) for _ in range(2))
        self.q = normal(self.total, 16, dim).to(dev)
        self.k, self.v = normal(self.total, heads, dim).to(dev), normal(self.total, heads, dim).to(dev)
        self.ck, self.cv, self.table = ck.to(dev), cv.to(dev), table.to(dev)
        self.config = gk.make_config(layers, self.pages, page, max_pages, self.batch, heads, dim, window if ring else 0)
        self.offsets = torch.tensor(np.cumsum([0] + rows), dtype=torch.int32, device=dev)
        self.lengths = torch.tensor(prior, dtype=torch.int32, device=dev)
        self.scale = 1.0 / math.sqrt(dim)
        self.buffers()

    def buffers(self):
        import torch
        shape = (self.config, self.batch, self.total)
        self.plan_bytes = gk.flash_attention_extend_plan_bytes(*shape)
        self.ws_bytes = gk.flash_attention_extend_workspace_bytes(*shape)
        # Neither needs initialisation: start from the worst.
        self.plan = torch.full((self.plan_bytes,), 0xFF, dtype=torch.uint8, device=self.dev)
        self.ws = torch.full((self.ws_bytes,), 0xFF, dtype=torch.uint8, device=self.dev)

    def make_plan(self, **kw):
        gk.check(gk.flash_attention_extend_plan(self.plan, self.plan_bytes, self.offsets, self.lengths, self.config,
                                                self.batch, self.total, self.window, self.sinks, **kw))

    def attend(self, out, layer=0, q=None, k=None, v=None, **kw):
        gk.check(gk.flash_attention_extend_paged_bf16(
            out, self.q if q is None else q, self.k if k is None else k, self.v if v is None else v, self.ck, self.cv,
            self.table, self.plan, self.plan_bytes, self.config, layer, self.batch, self.total, self.scale, self.ws,
            self.ws_bytes, **kw))

    def run(self, layer=0, **kw):
        import torch
        out = torch.full((self.total, 16, self.dim), 7.0, dtype=torch.bfloat16, device=self.dev)
        self.make_plan()
        self.attend(out, layer, **kw)
        torch.cuda.synchronize()
        return out

    def expected(self, layer=0):
        """(o, sum of w|v|, the largest sum of |q k| scale, keys) in 64 bits."""
        import torch
        o = torch.zeros(self.total, 16, self.dim, dtype=torch.float64, device=self.dev)
        a, s, most = torch.zeros_like(o), 0.0, 0
        start = 0
        for b, (n, p) in enumerate(zip(self.rows, self.prior)):
            if n == 0:
                continue
            keys = torch.arange(p, device=self.dev)
            if self.window:
                keys = keys[(keys > p - self.window) | (keys < self.sinks)]
            logical = keys // self.page
            if not self.ring:
                keys, logical = keys[logical < self.max_pages], logical[logical < self.max_pages]
            held = self.table[b].long()[logical % self.max_pages]
            keys, held = keys[held >= 0], held[held >= 0]
            new = slice(start, start + n)
            k = torch.cat([self.ck[layer, held, keys % self.page], self.k[new]]).double()
            v = torch.cat([self.cv[layer, held, keys % self.page], self.v[new]]).double()
            positions = torch.cat([keys, p + torch.arange(n, device=self.dev)])
            at = p + torch.arange(n, device=self.dev)[:, None]
            seen = positions <= at
            if self.window:
                seen &= (positions > at - self.window) | (positions < self.sinks)
            for h in range(16):
                kv = h * self.heads // 16
                q = self.q[new, h].double()
                x = (q @ k[:, kv].t() * self.scale).masked_fill(~seen, -math.inf)
                w = torch.softmax(x, -1)
                o[new, h] = w @ v[:, kv]
                a[new, h] = w @ v[:, kv].abs()
                s = max(s, float((q.abs() @ k[:, kv].abs().t()).max()) * self.scale)
            most = max(most, len(positions))
            start += n
        return o, a, s, most

    def check(self, out, layer=0, what=""):
        o, a, s, n = self.expected(layer)
        held = sum(self.rows)
        bound = 2.0**-8 * o.abs() + a * (2.0**-8 + 2 * self.dim * 2.0**-24 * s + 2 * n * 2.0**-24) * (1 + 2.0**-7)
        off = (out[:held].double() - o[:held]).abs()
        assert bool((off <= bound[:held] + 1e-30).all()), (
            what, float(off.max()), float((off / (bound[:held] + 1e-30)).max()))
        assert bool((out[held:] == 7.0).all()), "rows that no sequence holds"


GEOMETRIES = [(8, 256), (1, 512)]


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("page", [1, 7, 16, 64, 100])
@pytest.mark.parametrize("prior", [0, 1, 31, 32, 33, 63, 64, 65, 500])
def test_one_token(dev, heads, dim, page, prior):
    b = Batch(dev, heads, dim, [1], [prior], page=page, seed=prior)
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("rows", [2, 3, 7, 8, 9, 16, 17, 33, 63, 64, 65, 128, 130, 257])
@pytest.mark.parametrize("prior", [0, 95])
def test_one_sequence(dev, heads, dim, rows, prior):
    b = Batch(dev, heads, dim, [rows], [prior], seed=rows)
    b.check(b.run())


RAGGED = [([1, 0, 5, 1, 130, 0, 33, 2], [700, 40, 0, 64, 129, 0, 1000, 31]), ([0, 0, 3], [5, 6, 7]),
          ([1] * 40, [3 * i for i in range(40)]), ([300, 1, 1, 1], [0, 3000, 17, 1025])]


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("case", range(len(RAGGED)))
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 0), (64, 4), (129, 70), (1000, 1), (1, 1), (40, 5000)])
def test_ragged(dev, heads, dim, case, window, sinks):
    rows, prior = RAGGED[case]
    b = Batch(dev, heads, dim, rows, prior, window=window, sinks=sinks, seed=case, extra_rows=2)
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("page", [1, 16, 48])
@pytest.mark.parametrize("window", [1, 100, 129])
def test_ring(dev, heads, dim, page, window):
    rows, prior = [1, 77, 1, 300, 4, 0, 140], [5000, 333, 0, 128, 99, 10, 0]
    b = Batch(dev, heads, dim, rows, prior, page=page, window=window, ring=True, seed=page)
    b.check(b.run())


def test_a_window_narrower_than_the_ring(dev):
    b = Batch(dev, 8, 256, [3, 90], [700, 64], page=16, window=128, ring=True)
    b.window = 37
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_holes_in_the_table(dev, heads, dim):
    """Unmapped pages that the rows would see are skipped, whole tiles too."""
    holes = [(0, j) for j in range(0, 9)] + [(1, 3), (1, 4), (1, 11)] + [(2, j) for j in range(40)]
    b = Batch(dev, heads, dim, [1, 20, 2], [300, 200, 640], holes=holes)
    b.check(b.run())
    b.table[1, 2] = b.pages + 5  # out of the cache: as good as unmapped
    out = b.run()
    b.table[1, 2] = -1
    b.check(out)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_longer_than_the_table(dev, heads, dim):
    """New tokens may lie behind the table's last page: they come from k and v."""
    b = Batch(dev, heads, dim, [50, 1], [64, 60], max_pages=4)
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("prior", [4000, 20011])
def test_long_context_is_shared_out(dev, heads, dim, prior):
    b = Batch(dev, heads, dim, [1, 2, 9], [prior, 50, prior // 2], page=64)
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_many_sequences(dev, heads, dim):
    rng = np.random.default_rng(0)
    rows = [int(x) for x in rng.integers(0, 4, 700)]
    prior = [int(x) for x in rng.integers(0, 60, 700)]
    b = Batch(dev, heads, dim, rows, prior, seed=5)
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("spread", [1e-3, 8.0, 60.0])
def test_small_and_large_values(dev, heads, dim, spread):
    """From even weights to weights on one key (scores of thousands)."""
    b = Batch(dev, heads, dim, [40, 1, 3], [100, 333, 0], spread=spread)
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("rows,prior", [([40], [0]), ([2], [3000]), ([12, 30, 1], [3000, 40, 7]), ([300], [100])])
@pytest.mark.parametrize("window", [0, 9])
def test_what_a_row_does_not_see_is_not_in_it(dev, heads, dim, rows, prior, window):
    """Infinities and NaN in keys and values of new tokens, and of cached ones that the
    window has passed for some rows: in the rows that see them, and nowhere else."""
    import torch
    b = Batch(dev, heads, dim, rows, prior, window=window, seed=window)
    clean = b.expected()
    b.expected = lambda layer=0: clean
    n, p = rows[0], prior[0]
    at = torch.arange(b.total, device=dev)[:, None, None] + p
    own = (at < p + n)
    sees = lambda key: own & (key <= at) & ((key > at - window) if window else own)  # noqa: E731
    of_head = torch.arange(16, device=dev)[None, :, None] * heads // 16
    dims = torch.arange(dim, device=dev)[None, None, :]
    token, cached, last = p + n // 2, max(p - window // 2, 0), heads - 1
    odd = torch.zeros(b.total, 16, dim, dtype=torch.bool, device=dev)
    b.v[n // 2, 0, 3], b.v[n // 2, 0, dim - 1] = math.inf, NAN
    odd |= sees(token) & (of_head == 0) & ((dims == 3) | (dims == dim - 1))
    b.v[n - 1, last] = -math.inf
    odd |= sees(p + n - 1) & (of_head == last)
    if cached < p:
        held = int(b.table[0, cached // 16])
        b.cv[0, held, cached % 16, last, dim // 2] = math.inf
        odd |= sees(cached) & (of_head == last) & (dims == dim // 2)
    outs = [b.run(), b.run()]
    assert torch.equal(outs[0].isfinite(), ~odd)
    for out in outs:
        b.check(torch.where(odd, clean[0].bfloat16(), out))
    # Keys: a row that sees one has no finite weights.
    b.k[n // 2, 0, 5] = NAN
    odd |= sees(token) & (of_head == 0)
    out = b.run()
    assert torch.equal(out.isfinite(), ~odd)
    b.check(torch.where(odd, clean[0].bfloat16(), out))


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_rising_scores(dev, heads, dim):
    """Each tile's scores above the last's: the running maximum moves every time."""
    import torch
    b = Batch(dev, heads, dim, [3], [640])
    for x in (b.ck, b.k):
        x.copy_(torch.ones_like(x))
    b.q.copy_(torch.ones_like(b.q))
    at = torch.arange(640, device=dev)
    held = b.table[0].long()[at // 16]
    b.ck[0, held, at % 16] = (at.float() / 40).bfloat16()[:, None, None]
    b.k.mul_(17.0)
    b.check(b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_layers_share_a_plan_and_strides(dev, heads, dim):
    """Two layers by one plan; q, k and v as slices of one projection's rows."""
    import torch
    b = Batch(dev, heads, dim, [1, 37, 9], [50, 0, 200], layers=2)
    width = (16 + 2 * heads) * dim + 24
    wide = torch.full((b.total, width), NAN, dtype=torch.bfloat16, device=dev)
    q, k, v = wide[:, :16 * dim], wide[:, 16 * dim:(16 + heads) * dim], wide[:, (16 + heads) * dim:-24]
    q.copy_(b.q.view(b.total, -1)), k.copy_(b.k.view(b.total, -1)), v.copy_(b.v.view(b.total, -1))
    for layer in (1, 0):
        out = b.run(layer)
        b.check(out, layer)
        assert torch.equal(out, b.run(layer, q=q, k=k, v=v, q_stride=width, kv_stride=width))


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_buffers_of_a_larger_batch(dev, heads, dim):
    """One plan and one workspace for calls of all sizes, one after another."""
    import torch
    big = Batch(dev, heads, dim, [5] * 30 + [200], [77] * 31)
    for rows, prior in (([1], [3000]), ([5] * 30 + [200], [77] * 31), ([9, 0, 64], [0, 3, 700]), ([1, 1], [0, 0])):
        b = Batch(dev, heads, dim, rows, prior)
        b.plan, b.plan_bytes, b.ws, b.ws_bytes = big.plan, big.plan_bytes, big.ws, big.ws_bytes
        out = b.run()
        b.check(out)
        assert torch.equal(out, b.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_a_plan_of_other_sizes_writes_nothing(dev, heads, dim):
    import torch
    b = Batch(dev, heads, dim, [4, 4], [40, 50])
    b.make_plan()
    other = Batch(dev, heads, dim, [5, 4], [40, 50])
    out = torch.full((9, 16, dim), 7.0, dtype=torch.bfloat16, device=dev)
    plan = torch.zeros(other.plan_bytes, dtype=torch.uint8, device=dev)
    plan[:min(b.plan_bytes, other.plan_bytes)] = b.plan[:min(b.plan_bytes, other.plan_bytes)]
    other.plan = plan
    other.attend(out)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_offsets_that_do_not_ascend(dev, heads, dim):
    """Clamped: rows still belong to at most one sequence, all within the batch."""
    import torch
    b = Batch(dev, heads, dim, [20, 0, 0, 30, 5], [10, 4, 3, 600, 2])
    b.offsets.copy_(torch.tensor([0, 20, -7, 20, 50, 9999], device=dev))
    b.check(b.run())
    b.lengths.copy_(torch.tensor([-5, 4, 3, 2**31 - 1, 2], device=dev))
    out = b.run()  # other keys, the same rows; in bounds
    assert bool((out != 7.0).any())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_captured_step(dev, heads, dim):
    """Plan and two layers in a graph, replayed with other lengths and rows and
    with eager calls between that use buffers of their own."""
    import torch
    b = Batch(dev, heads, dim, [1, 30, 2, 0], [500, 100, 64, 3], layers=2)
    c = Batch(dev, heads, dim, [33, 0, 0, 0], [499, 90, 2, 0], layers=2, seed=9)
    outs = [torch.full((33, 16, dim), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    b.make_plan()
    b.attend(outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.make_plan()
        for layer in range(2):
            b.attend(outs[layer], layer)
    for rows, prior in (([1, 30, 2, 0], [500, 100, 64, 3]), ([0, 1, 1, 31], [9, 100, 60, 3]),
                        ([33, 0, 0, 0], [500, 1, 1, 1]), ([1, 30, 2, 0], [500, 100, 64, 3])):
        b.rows, b.prior = rows, prior
        b.offsets.copy_(torch.tensor(np.cumsum([0] + rows), dtype=torch.int32, device=dev))
        b.lengths.copy_(torch.tensor(prior, dtype=torch.int32, device=dev))
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            b.check(outs[layer], layer)
        c.check(c.run(1), 1)


def test_other_stream(dev):
    import torch
    b = Batch(dev, 8, 256, [5, 1], [60, 900])
    out = torch.full((6, 16, 256), 7.0, dtype=torch.bfloat16, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b.make_plan(stream=s)
    with torch.cuda.stream(s):
        b.attend(out)
    s.synchronize()
    b.check(out)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("seed", range(12))
def test_random(dev, heads, dim, seed):
    rng = np.random.default_rng(100 + seed)
    n = int(rng.integers(1, 9))
    rows = [int(x) for x in np.where(rng.random(n) < 0.4, 1, rng.integers(0, 150, n))]
    prior = [int(x) for x in rng.integers(0, 1500, n)]
    if sum(rows) == 0:
        rows[0] = 1
    ring = bool(rng.random() < 0.4)
    window = int(rng.integers(1, 600)) if ring or rng.random() < 0.5 else 0
    b = Batch(dev, heads, dim, rows, prior, page=int(rng.choice([1, 3, 16, 64])), window=window, ring=ring,
              sinks=0 if ring else int(rng.integers(0, 90)), layers=2, seed=seed)
    b.check(b.run(1), 1, (rows, prior, window, ring))


@pytest.mark.parametrize("heads,dim,ring", [(8, 256, True), (8, 256, False), (1, 512, False)])
def test_a_server_s_steps(dev, heads, dim, ring):
    """Reserve, attend, write, fork, verify a draft, compact, release: the cache that
    results holds each sequence's own tokens, and attention over it is the
    definition's over those."""
    import torch
    page, window, layers, batch = 16, 64, 2, 4
    max_pages = (window + 2 * page - 2) // page if ring else 20
    pages = batch * max_pages
    cfg = gk.make_config(layers, pages, page, max_pages, batch, heads, dim, window if ring else 0)
    table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev)
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)
    ck, cv = (torch.full((layers, pages, page, heads, dim), NAN, dtype=torch.bfloat16, device=dev) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    status = i32([77])
    lens = [0, 0, 0, 0]
    tokens = [[] for _ in range(batch)]  # of each sequence: (k, v) [layers][heads][dim]
    gen = torch.Generator(device="cpu").manual_seed(3)

    def step(rows, kept=None):
        total, prior = sum(rows), list(lens)
        gk.check(gk.kv_cache_reserve_pages(table, refs, cfg, i32(prior), i32([p + n for p, n in zip(prior, rows)]), status))
        assert int(status) == 0
        q, k, v = (torch.randn((layers, total, h, dim), generator=gen).bfloat16().to(dev) for h in (16, heads, heads))
        off = [sum(rows[:i]) for i in range(batch + 1)]
        size = gk.flash_attention_extend_plan_bytes(cfg, batch, total), gk.flash_attention_extend_workspace_bytes(cfg, batch, total)
        plan, ws = (torch.empty(n, dtype=torch.uint8, device=dev) for n in size)
        gk.check(gk.flash_attention_extend_plan(plan, size[0], i32(off), i32(prior), cfg, batch, total, window, 0))
        token_batch = i32([b for b, n in enumerate(rows) for _ in range(n)])
        token_position = i32([p + j for p, n in zip(prior, rows) for j in range(n)])
        for layer in range(layers):
            out = torch.empty(total, 16, dim, dtype=torch.bfloat16, device=dev)
            gk.check(gk.flash_attention_extend_paged_bf16(
                out, q[layer], k[layer], v[layer], ck, cv, table, plan, size[0], cfg, layer, batch, total,
                dim ** -0.5, ws, size[1]))
            gk.check(gk.kv_cache_write_bf16(ck, cv, cfg, table, token_batch, token_position, total, layer, k[layer], v[layer]))
            for b, n in enumerate(rows):
                for j in range(n):
                    mine = tokens[b] + [(k[:, off[b] + i], v[:, off[b] + i]) for i in range(j + 1)]
                    mine = mine[-window:]
                    K, V = (torch.stack([t[x][layer] for t in mine]).double() for x in (0, 1))
                    for h in range(16):
                        x = torch.softmax(K[:, h * heads // 16] @ q[layer, off[b] + j, h].double() * dim ** -0.5, 0)
                        want, size_v = x @ V[:, h * heads // 16], x @ V[:, h * heads // 16].abs()
                        bound = 2.0**-8 * want.abs() + 1.1 * 2.0**-8 * size_v
                        assert bool(((out[off[b] + j, h].double() - want).abs() <= bound).all()), (b, j, h)
        for b, n in enumerate(rows):
            tokens[b] += [(k[:, off[b] + j], v[:, off[b] + j]) for j in range(n)]
            lens[b] += n

    step([37, 5, 0, 0])
    step([1, 50, 0, 0])
    gk.check(gk.kv_cache_fork_bf16(ck, cv, cfg, table, refs, lengths := i32(lens), i32([0, 1]), i32([2, 3]), 2, status))
    assert int(status) == 0 and lengths.tolist() == [38, 55, 38, 55]
    for child, parent in ((2, 0), (3, 1)):
        lens[child], tokens[child] = lens[parent], list(tokens[parent])
    step([1, 3, 1, 0])
    before = lens[1]
    step([0, 8, 0, 9])  # drafts: sequences 1 and 3 keep some
    keep = {1: [0, 2, 5], 3: [0, 1, 4, 8]}
    kept = [[lens[b] - n + j for j in keep[b]] for b, n in ((1, 8), (3, 9))]
    firsts = [lens[1] - 8, lens[3] - 9]
    assert firsts[0] == before
    st = i32([77, 77])
    gk.check(gk.kv_cache_compact_bf16(ck, cv, cfg, table, refs, i32([1, 3]), i32(firsts), i32([0, 3, 7]), i32(kept[0] + kept[1]), 2, 7, st))
    assert st.tolist() == [0, 0]
    for b, f in zip((1, 3), firsts):
        tokens[b] = tokens[b][:f] + [tokens[b][f + j] for j in keep[b]]
        lens[b] = f + len(keep[b])
    if not ring:  # what the shortened sequences and the window no longer need
        gk.check(gk.kv_cache_release_pages(table, refs, cfg, i32(lens), i32([2**31 - 1] * 4)))
        gk.check(gk.kv_cache_release_pages(table, refs, cfg, i32([0] * 4), i32([max(0, n - window) for n in lens])))
    step([1, 1, 1, 1])
    step([40, 1, 2, 3])


@pytest.mark.parametrize("heads,dim,pages", [(8, 256, 21000), (1, 512, 84000)])
def test_a_cache_of_more_than_four_gigabytes(dev, heads, dim, pages):
    """The same pages at the far end of a cache past 2^32 bytes, in its second layer."""
    import torch
    b = Batch(dev, heads, dim, [1, 40, 0, 3], [900, 333, 7, 64], page=64)
    out = b.run()
    b.check(out)
    large = torch.empty((2, 2, pages, 64, heads, dim), dtype=torch.bfloat16, device=dev)
    assert large[0, 0].numel() * 2 > 2**32 and b.pages < 100
    for i, small in enumerate((b.ck, b.cv)):
        large[i, 1, pages - b.pages:] = small[0]
    b.ck, b.cv = large[0], large[1]
    b.table = torch.where(b.table >= 0, b.table + pages - b.pages, b.table)
    b.config = gk.make_config(2, pages, 64, b.max_pages, b.batch, heads, dim, 0)
    assert torch.equal(b.run(1), out)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_every_run_gives_the_same(dev, heads, dim):
    import torch
    b = Batch(dev, heads, dim, [1, 30, 3, 200], [5000, 700, 2049, 100])
    b.v[20, 0, 3] = math.inf  # some rows are worked out again
    out = b.run()
    assert not bool(out.isfinite().all())
    for _ in range(6):
        b.ws.fill_(0xFF)
        assert torch.equal(b.run().view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_two_streams_at_once(dev, heads, dim):
    """Two batches, each with its buffers, on streams that overlap; layers of one batch
    on two streams by one plan, each with its workspace."""
    import torch
    b = Batch(dev, heads, dim, [1, 30, 3], [5000, 700, 2049], layers=2)
    c = Batch(dev, heads, dim, [150, 1], [900, 3000], layers=2, seed=4)
    want = [b.run(0), b.run(1), c.run(0)]
    ws = torch.empty_like(b.ws)
    streams = [torch.cuda.Stream() for _ in range(3)]
    b.make_plan()
    torch.cuda.synchronize()
    outs = [[torch.full_like(w, 7.0) for w in want] for _ in range(8)]
    torch.cuda.synchronize()
    for row in outs:
        with torch.cuda.stream(streams[0]):
            b.attend(row[0], 0)
        with torch.cuda.stream(streams[1]):
            own, b.ws = b.ws, ws
            b.attend(row[1], 1)
            b.ws = own
        with torch.cuda.stream(streams[2]):
            c.make_plan()
            c.attend(row[2], 0)
    torch.cuda.synchronize()
    for row in outs:
        assert all(torch.equal(x, w) for x, w in zip(row, want))


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_graphs_that_share_a_workspace(dev, heads, dim):
    """Two captured steps with one plan buffer and one workspace, replayed in turn with
    eager calls between."""
    import torch
    a = Batch(dev, heads, dim, [1, 40], [3000, 64])
    b = Batch(dev, heads, dim, [20, 21], [10, 900], seed=2)
    b.plan, b.ws = a.plan, a.ws  # the same sizes
    want = [a.run(), b.run()]
    outs = [torch.empty_like(w) for w in want]
    graphs = []
    for x, out in zip((a, b), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.make_plan()
            x.attend(out)
        graphs.append(graph)
    for turn in range(4):
        for o in outs:
            o.fill_(7.0)
        for graph in graphs if turn % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        assert torch.equal((a, b)[turn % 2].run(), want[turn % 2])


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("page,window", [(16, 64), (1, 40), (64, 100)])
def test_prompts_longer_than_the_ring(dev, heads, dim, page, window):
    """Attend, append and attend again where prompts bring several laps of a ring at once,
    beside short ones: the rows of the second step see the last of the first."""
    import torch
    first = [300, 1, 2 * window + 200, 0, 7]
    b = Batch(dev, heads, dim, first, [0, 333, 50, 0, window], page=page, window=window, ring=True)
    b.check(b.run())
    # The second step's batch, its cache and table the first's: every slot mapped.
    slots, i32 = b.max_pages, lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pages = b.batch * slots
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().view(b.batch, slots)
    c = Batch(dev, heads, dim, [3, 1, 30, 2, 9], [n + p for n, p in zip(first, b.prior)], page=page, window=window,
              ring=True, seed=1)
    ck, cv = (torch.full((1, pages, page, heads, dim), NAN, dtype=torch.bfloat16, device=dev) for _ in range(2))
    for i in range(b.batch):
        for j in range(slots):
            if int(b.table[i, j]) >= 0:
                ck[:, table[i, j]], cv[:, table[i, j]] = b.ck[:, int(b.table[i, j])], b.cv[:, int(b.table[i, j])]
    c.table = table.to(dev)
    c.config = gk.make_config(1, pages, page, slots, b.batch, heads, dim, window)
    who = i32([s for s, n in enumerate(first) for _ in range(n)])
    where = [p + j for p, n in zip(b.prior, first) for j in range(n)]
    gk.check(gk.kv_cache_write_bf16(ck, cv, c.config, c.table, who, i32(where), b.total, 0, b.k, b.v))
    c.ck, c.cv = ck, cv
    # What has to be there, row after row.
    at = 0
    for s, (n, p) in enumerate(zip(first, b.prior)):
        for j in range(max(0, n - slots * page), n):
            page_of, offset = int(table[s, (p + j) // page % slots]), (p + j) % page
            assert torch.equal(ck[0, page_of, offset], b.k[at + j]) and torch.equal(cv[0, page_of, offset], b.v[at + j])
        at += n
    c.check(c.run())


@pytest.mark.parametrize("page", [1, 4, 16])
def test_a_shortened_ring_gives_back_what_was_dropped(dev, page):
    """Drafts that were rejected: what lies between the new length and the old goes back
    to the pool, and no key that the next rows see goes with it."""
    import torch
    window, drafts = 40, 23
    slots = -(-(window + drafts) // page) + 1
    old, rows = [700, drafts + 5, 3 * slots * page, 50], [3, 9, 1, 20]
    b = Batch(dev, 8, 256, rows, old, page=page, window=window, ring=True, max_pages=slots, spare=40)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    cut = [drafts, drafts, page, 0]
    b.prior = [n - c for n, c in zip(old, cut)]
    b.lengths.copy_(i32(b.prior))
    want = b.expected()
    before = b.table.clone()
    refs = i32(np.bincount(b.table[b.table >= 0].cpu().numpy(), minlength=b.pages))
    gk.check(gk.kv_cache_release_pages(b.table, refs, b.config, b.lengths, i32(old)))
    for s, (new, was) in enumerate(zip(b.prior, old)):
        gone = {j % slots for j in range(-(-new // page), was // page)}
        assert set(torch.nonzero(before[s] != b.table[s])[:, 0].tolist()) == gone
    status = i32([77])
    gk.check(gk.kv_cache_reserve_pages(b.table, refs, b.config, b.lengths, i32([n + p for n, p in zip(rows, b.prior)]), status))
    assert int(status) == 0
    b.expected = lambda layer=0: want
    b.check(b.run())
