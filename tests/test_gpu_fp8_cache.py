"""The quantised cache: rows written as e4m3 codes, read back, and decode attention over
them, against the definitions.

Codes are compared for equality: the quotient is the correctly rounded one in 32 bits,
as in the definition here, and the code the nearest with ties to even. Values read
back are code * scale in 32 bits rounded to bf16: equal too.

Attention, tolerance before any run: the output is rounded once to bf16 (2^-8 |o|). A
weight meets V as two bf16 numbers, off by 2^-16 of it. A score is a sum in 32 bits of D
products, off by at most D 2^-24 sum |q k| scale, and its factor and exponent by a few
2^-24 of its size: each shifts its weight by that factor, in the numerator and, at
most as much, in the sum. Sums over n keys in 32 bits add n 2^-24 of sum w|v|
each."""
import math

import numpy as np
import pytest

import gemma_kv as gk

pytestmark = pytest.mark.gpu

NAN_CODE = 0x7F


def quantised(x, scale):
    """The definition, on the CPU: codes of x [..., heads, dim] by scale [heads]."""
    import torch
    x = x.float().cpu() / scale.cpu()[:, None]
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)


def values(codes):
    import torch
    return codes.view(torch.float8_e4m3fn)


def same_codes(a, b):
    """Equal, NaN codes of either sign being one."""
    nan_a, nan_b = (a & 0x7F) == NAN_CODE, (b & 0x7F) == NAN_CODE
    return bool(((a == b) | (nan_a & nan_b)).all())


class Cache:
    """Sequences of `lens` keys. What is no live key holds NaN codes: slots behind the
    lengths, unmapped and unused pages."""

    def __init__(self, dev, heads, dim, lens, page=16, window=0, layers=2, seed=0, max_pages=None, holes=(), spare=3,
                 room=0):
        import torch
        self.dev, self.heads, self.dim, self.lens, self.page = dev, heads, dim, lens, page
        self.window, self.layers, self.batch = window, layers, len(lens)
        gen = torch.Generator().manual_seed(seed + 5)
        if max_pages is None:
            max_pages = (window + 2 * page - 2) // page if window else max(1, -(-(max(lens) + room) // page))
        self.max_pages = max_pages
        held = [(b, j) for b, n in enumerate(lens) for j in range(-(-(n + room) // page))
                if (not window or j >= -(-(n + room) // page) - max_pages) and (b, j) not in holes
                and (window or j < max_pages)]
        self.pages = len(held) + spare
        order = torch.randperm(self.pages, generator=gen)
        self.table = torch.full((self.batch, max_pages), -1, dtype=torch.int32)
        codes = torch.full((2, layers, self.pages, page, heads, dim), NAN_CODE, dtype=torch.uint8)
        for (b, j), physical in zip(held, order):
            self.table[b, j % max_pages] = int(physical)
            live = max(0, min(page, lens[b] - j * page))
            x = torch.randn(2, layers, live, heads, dim, generator=gen) * 60
            codes[:, :, physical, :live] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        self.ck, self.cv = (c.contiguous().to(dev) for c in codes)
        self.table = self.table.to(dev)
        self.ks, self.vs = ((0.01 + 0.03 * torch.rand(layers, heads, generator=gen)).to(dev) for _ in range(2))
        self.config = gk.make_config(layers, self.pages, page, max_pages, self.batch, heads, dim, window)
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.scale = 1.0 / math.sqrt(dim)
        normal = lambda *s: torch.randn(s, generator=gen).bfloat16().to(dev)  # noqa: E731
        self.q, self.k, self.v = normal(self.batch, 16, dim), normal(self.batch, heads, dim), normal(self.batch, heads, dim)

    def partials(self, splits):
        import torch
        n = self.batch * 16 * splits
        return [torch.full((n * m,), float("nan"), dtype=torch.float32, device=self.dev) for m in (1, 1, self.dim)]

    def plan(self):
        live = max(min(n, self.window) if self.window else n for n in self.lens)
        return gk.decode_split_plan_fp8(self.config, self.batch, live)

    def decode(self, plan=None, layer=1, append=None, **kw):
        import torch
        size, splits = plan or self.plan()
        out = torch.full((self.batch, 16, self.dim), 7.0, dtype=torch.bfloat16, device=self.dev)
        head = (out, *self.partials(splits), self.q, self.ck, self.cv, self.ks, self.vs, self.table, self.lengths)
        tail = (self.config, layer, self.scale, size, splits, self.batch)
        if append is None:
            gk.check(gk.flash_attention_decode_paged_fp8(*head, *tail, **kw))
        else:
            position = torch.tensor(append, dtype=torch.int32, device=self.dev)
            gk.check(gk.flash_attention_append_decode_paged_fp8(*head, position, self.k, self.v, *tail, **kw))
        torch.cuda.synchronize()
        return out

    def rows(self, b, positions):
        """(page, offset) of those that are mapped."""
        logical = positions // self.page
        if not self.window:
            positions, logical = positions[logical < self.max_pages], logical[logical < self.max_pages]
        held = self.table[b].long()[logical % self.max_pages]
        ok = (held >= 0) & (held < self.pages)
        return held[ok], (positions % self.page)[ok]

    def check(self, out, layer=1, limit=None, what=""):
        import torch
        for b, n in enumerate(self.lens):
            first = max(0, n - self.window) if self.window else 0
            last = n if limit is None else min(n, first + limit)
            at = self.rows(b, torch.arange(first, last, device=self.dev))
            if len(at[0]) == 0:
                assert bool((out[b] == 0).all()), what
                continue
            k, v = (values(c[layer][at]).double() * s[layer].double()[:, None] for c, s in ((self.ck, self.ks), (self.cv, self.vs)))
            for h in range(16):
                kv = h * self.heads // 16
                q = self.q[b, h].double()
                w = torch.softmax(k[:, kv] @ q * self.scale, 0)
                o, a = w @ v[:, kv], w @ v[:, kv].abs()
                s = float((k[:, kv].abs() @ q.abs()).max()) * self.scale
                rel = 2.0**-16 + 2 * (self.dim + 8) * 2.0**-24 * (s + 1) + 2 * len(w) * 2.0**-24
                off = (out[b, h].double() - o).abs()
                bound = 2.0**-8 * o.abs() + a * rel * (1 + 2.0**-7) + 1e-30
                # NaN codes of live keys: the definition is NaN, and so is the output.
                ok = (off <= bound) | (o.isnan() & out[b, h].isnan())
                assert bool(ok.all()), (what, b, h, float((off / bound).max()))


# ---- codes --------------------------------------------------------------------------

@pytest.mark.parametrize("scale", [1.0, 0.037, 2.0**-7, 3.1e-38, 1e30, 1.7])
def test_every_bf16_value(dev, scale):
    import torch
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, 8, 256)
    rows = every.shape[0]
    config = gk.make_config(1, rows, 1, rows, 1, 8, 256, 0)
    table = torch.arange(rows, dtype=torch.int32, device=dev).flip(0).contiguous()
    batch, position = torch.zeros(rows, dtype=torch.int32, device=dev), torch.arange(rows, dtype=torch.int32, device=dev)
    ck, cv = (torch.zeros(rows, 8, 256, dtype=torch.uint8, device=dev) for _ in range(2))
    ks = torch.full((1, 8), scale, device=dev)
    x = every.to(dev)
    gk.check(gk.kv_cache_write_fp8(ck, cv, config, table, batch, position, rows, 0, x, x, ks, None))
    torch.cuda.synchronize()
    assert same_codes(ck.flip(0).cpu(), quantised(every, ks[0]))
    assert same_codes(cv.flip(0).cpu(), quantised(every, torch.ones(8)))
    k, v = (torch.zeros(rows, 8, 256, dtype=torch.bfloat16, device=dev) for _ in range(2))
    gk.check(gk.kv_cache_read_fp8(k, v, ck, cv, config, table, batch, position, rows, 0, ks, None))
    torch.cuda.synchronize()
    for got, codes, s in ((k, ck, scale), (v, cv, 1.0)):
        want = (values(codes.flip(0).cpu()).float() * torch.tensor(s, dtype=torch.float32)).bfloat16()
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512), (3, 48), (2, 16)])
@pytest.mark.parametrize("window,page", [(0, 16), (0, 5), (40, 1), (40, 16)])
def test_rows_written_and_read_by_tokens(dev, heads, dim, window, page):
    """Ragged rows out of a wider projection; tokens that are skipped; laps of a ring."""
    import torch
    rng = np.random.default_rng(heads * 100 + window + page)
    batch, layers, layer = 3, 2, 1
    max_pages = (window + 2 * page - 2) // page if window else 13
    slots = max_pages * page
    pages = batch * max_pages + 2
    config = gk.make_config(layers, pages, page, max_pages, batch, heads, dim, window)
    table = rng.permutation(pages)[:batch * max_pages].reshape(batch, max_pages).astype(np.int32)
    table[1, 2 % max_pages] = -1
    table[2, 1 % max_pages] = pages + 4
    tokens = []
    for b, (start, count) in enumerate([(3, 2 * slots + 7 if window else slots + 9), (slots // 2, 11), (0, 17)]):
        tokens += [(b, start + r) for r in range(count)]
    tokens += [(-1, 0), (batch, 0), (0, -1), (0, -5)]
    n = len(tokens)
    tb, tp = (torch.tensor([t[i] for t in tokens], dtype=torch.int32, device=dev) for i in (0, 1))
    gen = torch.Generator().manual_seed(7)
    wide = (torch.randn(n, 2 * heads * dim + 8, generator=gen) * 3).bfloat16()
    k, v = wide[:, :heads * dim], wide[:, heads * dim:2 * heads * dim]
    ks, vs = (0.02 + torch.rand(layers, heads, generator=gen) * 0.1 for _ in range(2))
    before = torch.randint(0, 256, (2, layers, pages, page, heads, dim), generator=gen, dtype=torch.uint8)
    want = before.clone()
    row = {}
    for i, (b, pos) in enumerate(tokens):  # in order: the newest of a slot stays
        if not 0 <= b < batch or pos < 0 or (not window and pos // page >= max_pages):
            continue
        physical = table[b, pos // page % max_pages]
        if not 0 <= physical < pages:
            continue
        row[i] = (physical, pos % page)
        for c, x, s in ((0, k, ks), (1, v, vs)):
            want[c, layer, physical, pos % page] = quantised(x[i].view(1, heads, dim), s[layer])[0]
    ck, cv = (c.contiguous().to(dev) for c in before)
    on = wide.to(dev)
    gk.check(gk.kv_cache_write_fp8(ck, cv, config, torch.from_numpy(table).to(dev), tb, tp, n, layer, on,
                                   on[:, heads * dim:], ks.to(dev), vs.to(dev), kv_stride=on.stride(0)))
    torch.cuda.synchronize()
    assert torch.equal(ck.cpu(), want[0]) and torch.equal(cv.cpu(), want[1])
    got = torch.full((n, 2 * heads * dim + 8), 7.0, dtype=torch.bfloat16, device=dev)
    gk.check(gk.kv_cache_read_fp8(got, got[:, heads * dim:], ck, cv, config, torch.from_numpy(table).to(dev), tb, tp,
                                  n, layer, ks.to(dev), vs.to(dev), kv_stride=got.stride(0)))
    torch.cuda.synchronize()
    expect = torch.full((n, 2 * heads * dim + 8), 7.0, dtype=torch.bfloat16)
    for i, (physical, offset) in row.items():
        for c, s, at in ((0, ks, 0), (1, vs, heads * dim)):
            x = values(want[c, layer, physical, offset]).float() * s[layer][:, None]
            expect[i, at:at + heads * dim] = x.bfloat16().reshape(-1)
    assert torch.equal(got.cpu(), expect)


def test_rows_far_into_a_large_cache(dev):
    """Code offsets past 2^32, from a layer's base as well as within it."""
    import torch
    heads, dim, page = 8, 256, 64
    pages = 20000  # 2.6 GB a layer
    config = gk.make_config(2, pages, page, pages, 1, heads, dim, 0)
    ck, cv = (torch.zeros(2 * pages * page * heads * dim, dtype=torch.uint8, device=dev) for _ in range(2))
    table = torch.arange(pages, dtype=torch.int32, device=dev)
    position = torch.tensor([0, pages * page - 1, pages * page // 2 + 3], dtype=torch.int32, device=dev)
    batch = torch.zeros(3, dtype=torch.int32, device=dev)
    k, v = (torch.randn(3, heads, dim, device=dev).bfloat16() for _ in range(2))
    gk.check(gk.kv_cache_write_fp8(ck, cv, config, table, batch, position, 3, 1, k, v))
    back = [torch.zeros_like(k) for _ in range(2)]
    gk.check(gk.kv_cache_read_fp8(*back, ck, cv, config, table, batch, position, 3, 1))
    torch.cuda.synchronize()
    one = torch.ones(heads)
    for got, x, c in zip(back, (k, v), (ck, cv)):
        codes = quantised(x, one)
        assert torch.equal(got.cpu(), values(codes).float().bfloat16())
        rows = c.view(2, pages * page, heads, dim)[1, position.long()]
        assert torch.equal(rows.cpu(), codes)
    # Attention over a far part of it: 40 keys around the last row, through a table of
    # their page alone.
    small = gk.make_config(2, pages, page, 1, 1, heads, dim, 0)
    last = torch.tensor([pages - 1], dtype=torch.int32, device=dev)
    rows = torch.arange(page, dtype=torch.int32, device=dev)
    k, v = (torch.randn(page, heads, dim, device=dev).bfloat16() for _ in range(2))
    gk.check(gk.kv_cache_write_fp8(ck, cv, small, last, torch.zeros(page, dtype=torch.int32, device=dev), rows, page, 1,
                                   k, v))
    q = torch.randn(1, 16, dim, device=dev).bfloat16()
    out = torch.zeros_like(q)
    gk.check(gk.flash_attention_decode_paged_fp8(
        out, None, None, None, q, ck, cv, None, None, last, torch.tensor([page], dtype=torch.int32, device=dev), small, 1,
        1 / 16, 64, 1, 1))
    torch.cuda.synchronize()
    kd, vd = (values(quantised(x, one)).double() for x in (k, v))
    for h in range(16):
        w = torch.softmax(kd[:, h // 2] @ q[0, h].cpu().double() / 16, 0)
        assert bool(((out[0, h].cpu().double() - w @ vd[:, h // 2]).abs() <= 2.0**-8 * (w @ vd[:, h // 2].abs())).all())


# ---- attention ------------------------------------------------------------------------

CASES = [
    dict(heads=8, dim=256, lens=[1]),
    dict(heads=1, dim=512, lens=[1]),
    dict(heads=8, dim=256, lens=[33, 0, 31, 32, 64, 65, 1]),
    dict(heads=1, dim=512, lens=[33, 0, 31, 32, 64, 65, 1]),
    dict(heads=8, dim=256, lens=[700, 1500, 129], page=64),
    dict(heads=1, dim=512, lens=[700, 1500, 129], page=64),
    dict(heads=8, dim=256, lens=[2500], window=1024, page=1),
    dict(heads=8, dim=256, lens=[90, 100, 101, 5000, 131], window=100, page=16),
    dict(heads=1, dim=512, lens=[90, 100, 101, 5000, 131], window=100, page=7),
    dict(heads=1, dim=512, lens=[8193], page=64),
    dict(heads=8, dim=256, lens=[8193], page=64),
    dict(heads=1, dim=512, lens=[300] * 30 + [4000], page=16),
    dict(heads=8, dim=256, lens=[300] * 30 + [4000], page=16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c['heads']}x{c['dim']}-{len(c['lens'])}-{max(c['lens'])}-{c.get('window', 0)}")
def test_attention(dev, case):
    c = Cache(dev, **case)
    c.check(c.decode())


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
@pytest.mark.parametrize("plan", [(1, 333), (20, 17), (31, 11), (32, 11), (33, 11), (64, 6), (65, 6), (96, 4), (128, 3),
                                  (160, 3), (1000, 1), (2**31 - 1, 1), (2**31 - 1, 2), (48, 3)])
def test_any_splits(dev, heads, dim, plan):
    """Split sizes of one to four waves, one split, more splits than keys; splits that cover
    a part of the keys attend to that."""
    c = Cache(dev, heads, dim, [333, 5, 64, 0], page=16, seed=3)
    c.check(c.decode(plan), limit=plan[0] * plan[1])


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
def test_unmapped_pages_and_short_tables(dev, heads, dim):
    c = Cache(dev, heads, dim, [400, 200, 64, 48], page=16, holes=[(0, 0), (0, 5), (0, 24), (1, 12), (2, 0), (2, 1), (2, 2), (2, 3)])
    c.check(c.decode())
    c.table[3, 0] = c.pages  # out of the cache
    c.check(c.decode())
    c = Cache(dev, heads, dim, [400, 90], page=16, max_pages=8)  # lengths past the table
    c.check(c.decode())


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
@pytest.mark.parametrize("window,page", [(0, 16), (96, 16), (96, 1)])
def test_append_equals_write_then_attend(dev, heads, dim, window, page):
    import torch
    lens = [1, 300, 97, 32, 33, 640, 64]
    position = [n - 1 for n in lens]
    position[4] = -1  # a sequence without a new token
    for plan in [None, (32, 20), (64, 10), (640, 1)]:
        a, b = (Cache(dev, heads, dim, lens, page=page, window=window, seed=8) for _ in range(2))
        out = a.decode(plan, append=position)
        tokens = torch.arange(len(lens), dtype=torch.int32, device=dev)
        gk.check(gk.kv_cache_write_fp8(b.ck, b.cv, b.config, b.table, tokens,
                                       torch.tensor(position, dtype=torch.int32, device=dev), len(lens), 1, b.k, b.v, b.ks, b.vs))
        assert torch.equal(out, b.decode(plan))
        assert torch.equal(a.ck, b.ck) and torch.equal(a.cv, b.cv)
        a.check(out)


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
def test_append_that_no_split_attends(dev, heads, dim):
    """A position behind the live keys is written and not seen; unmapped and past the table
    nothing is written; a plan of fewer keys leaves the token out of the sums."""
    import torch
    c = Cache(dev, heads, dim, [40, 0, 40, 40, 200], page=16, room=16, holes=[(2, 3)], max_pages=14)
    before = [x.clone() for x in (c.ck, c.cv)]
    out = c.decode((64, 2), append=[41, 0, 48, 14 * 16, 199])
    c.check(out, limit=128)
    for cache, old, new, s in ((c.ck, before[0], c.k, c.ks), (c.cv, before[1], c.v, c.vs)):
        want = old.clone()
        for b, pos in ((0, 41), (1, 0), (4, 199)):
            want[1, c.table[b, pos // 16].item(), pos % 16] = quantised(new[b:b + 1], s[1])[0].to(dev)
        assert same_codes(cache, want)


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
def test_nan_of_a_live_key_reaches_its_head_alone(dev, heads, dim):
    import torch
    for which in range(2):
        for plan in [(32, 10), (1000, 1)]:
            c = Cache(dev, heads, dim, [300, 200], page=16, seed=which)
            page, offset = c.rows(0, torch.tensor([170], device=dev))
            (c.ck, c.cv)[which][1, page, offset, heads - 1, 3] = NAN_CODE
            out = c.decode(plan)
            group = 16 // heads
            nan = out.isnan()
            hit = nan[0, 16 - group:]
            assert bool(hit.all()) if which == 0 else bool(hit[:, 3].all()) and int(hit.sum()) == group
            assert not bool(nan[0, :16 - group].any()) and not bool(nan[1].any())


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
def test_large_scores(dev, heads, dim):
    """Scores that leave one key, far apart in tiles: the running maximum moves late."""
    import torch
    c = Cache(dev, heads, dim, [1000], page=16)
    c.q *= 8
    c.check(c.decode((1000, 1)))
    c.check(c.decode())
    c.ks.fill_(0.5)
    out = c.decode((128, 8))
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
def test_captured_with_other_lengths_and_streams(dev, heads, dim):
    import torch
    c = Cache(dev, heads, dim, [500, 333], page=16, seed=2)
    size, splits = gk.decode_split_plan_fp8(c.config, 2, 500)
    out = torch.zeros(2, 16, dim, dtype=torch.bfloat16, device=dev)
    parts = c.partials(splits)
    position = torch.zeros(2, dtype=torch.int32, device=dev)

    def call():
        gk.check(gk.flash_attention_append_decode_paged_fp8(
            out, *parts, c.q, c.ck, c.cv, c.ks, c.vs, c.table, c.lengths, position, c.k, c.v, c.config, 1, c.scale, size,
            splits, 2))
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([500, 333], [1, 2], [0, 400], [499, 64]):
        c.lens = lens
        c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        position.copy_(torch.tensor([n - 1 for n in lens], dtype=torch.int32))
        c.k.normal_()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
    # Two at once, with partials of their own.
    a, b = Cache(dev, heads, dim, [900, 30], page=16, seed=4), Cache(dev, heads, dim, [64, 1200], page=16, seed=5)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    torch.cuda.synchronize()
    for x, s in zip((a, b), streams):
        with torch.cuda.stream(s):
            size, splits = x.plan()
            o = torch.zeros(2, 16, dim, dtype=torch.bfloat16, device=dev)
            gk.check(gk.flash_attention_decode_paged_fp8(o, *x.partials(splits), x.q, x.ck, x.cv, x.ks, x.vs, x.table, x.lengths,
                                                         x.config, 1, x.scale, size, splits, 2))
            outs.append(o)
    torch.cuda.synchronize()
    for x, o in zip((a, b), outs):
        x.check(o)


def test_runs_are_alike(dev):
    import torch
    c = Cache(dev, 1, 512, [3000, 1234, 77], page=64)
    out = c.decode()
    assert all(torch.equal(out, c.decode()) for _ in range(5))


# ---- the page pool over codes -----------------------------------------------------------

@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
def test_forked_compacted_and_read_into_an_extension(dev, heads, dim):
    """A quantised cache under the pool's operators (rows of half the head_dim as bf16), and
    its keys read back for a prompt's chunk: the attention over bf16 of the same values
    equals the definition over the codes."""
    import torch
    layers, page, max_pages, batch = 2, 16, 12, 3
    pages = 30
    config = gk.make_config(layers, pages, page, max_pages, batch, heads, dim, 0)
    half = gk.make_config(layers, pages, page, max_pages, batch, heads, dim // 2, 0)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, refs = torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev), torch.zeros(pages, dtype=torch.int32, device=dev)
    status, lengths = i32(9), i32(100, 0, 0)
    ck, cv = (torch.full((layers, pages, page, heads, dim), NAN_CODE, dtype=torch.uint8, device=dev) for _ in range(2))
    gk.check(gk.kv_cache_reserve_pages(table, refs, half, i32(0, 0, 0), i32(100, 0, 0), status))
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(layers, 100, heads, dim, generator=gen).bfloat16().to(dev) for _ in range(2))
    ks, vs = (torch.full((layers, heads), s, device=dev) for s in (0.05, 0.03))
    zeros, line = torch.zeros(100, dtype=torch.int32, device=dev), torch.arange(100, dtype=torch.int32, device=dev)
    for layer in range(layers):
        gk.check(gk.kv_cache_write_fp8(ck, cv, config, table, zeros, line, 100, layer, k[layer], v[layer], ks, vs))
    gk.check(gk.kv_cache_fork_bf16(ck.view(torch.bfloat16), cv.view(torch.bfloat16), half, table, refs, lengths, i32(0), i32(2), 1, status))
    torch.cuda.synchronize()
    assert status.item() == 0 and lengths.tolist() == [100, 0, 100]
    # The branch keeps some of its last tokens (those of the begun page, its own).
    kept = [96, 98, 99]
    one = torch.full((1,), 9, dtype=torch.int32, device=dev)
    gk.check(gk.kv_cache_compact_bf16(ck.view(torch.bfloat16), cv.view(torch.bfloat16), half, table, refs, i32(2), i32(96), i32(0, 3), i32(*kept), 1, 3, one))
    torch.cuda.synchronize()
    assert one.item() == 0
    held = list(range(96)) + kept
    rows = torch.tensor(held, device=dev)
    codes = [quantised(x[1], s[1]).to(dev)[rows] for x, s in ((k, ks), (v, vs))]
    # Its keys as rows, which are a cache with one page that counts up.
    n = len(held)
    back = [torch.zeros(128, heads, dim, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    gk.check(gk.kv_cache_read_fp8(*back, ck, cv, config, table, torch.full((n,), 2, dtype=torch.int32, device=dev),
                                  torch.arange(n, dtype=torch.int32, device=dev), n, 1, ks, vs))
    torch.cuda.synchronize()
    for got, c, s in zip(back, codes, (ks, vs)):
        assert torch.equal(got[:n].cpu(), (values(c.cpu()).float() * s[1].cpu()[:, None]).bfloat16())
    plain = gk.make_config(1, 2, 64, 2, 1, heads, dim, 0)
    new = 21
    q, nk, nv = (torch.randn(new, m, dim, generator=gen).bfloat16().to(dev) for m in (16, heads, heads))
    plan = torch.empty(gk.flash_attention_extend_plan_bytes(plain, 1, new), dtype=torch.uint8, device=dev)
    ws = torch.empty(gk.flash_attention_extend_workspace_bytes(plain, 1, new), dtype=torch.uint8, device=dev)
    gk.check(gk.flash_attention_extend_plan(plan, plan.numel(), i32(0, new), i32(n), plain, 1, new, 0, 0))
    out = torch.zeros_like(q)
    gk.check(gk.flash_attention_extend_paged_bf16(out, q, nk, nv, *back, i32(0, 1), plan, plan.numel(), plain, 0, 1, new,
                                                  1 / math.sqrt(dim), ws, ws.numel()))
    torch.cuda.synchronize()
    kd, vd = (torch.cat([b[:n], x]).double() for b, x in zip(back, (nk, nv)))
    hidden = torch.arange(n + new, device=dev) > n + torch.arange(new, device=dev)[:, None]
    for h in range(16):
        kv = h * heads // 16
        x = (q[:, h].double() @ kd[:, kv].t() / math.sqrt(dim)).masked_fill(hidden, -math.inf)
        w = torch.softmax(x, -1)
        o, a = w @ vd[:, kv], w @ vd[:, kv].abs()
        # As for the extension: output and weights rounded to bf16, scores in 32 bits.
        assert bool(((out[:, h].double() - o).abs() <= 2.0**-8 * o.abs() + a * (2.0**-8 + 2.0**-12)).all())
