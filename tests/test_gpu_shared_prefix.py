"""Extension of groups of sequences that share a prefix, against the extension's
definition in 64 bits and its tolerance: the output is rounded once to bf16 (2^-8 |o|),
each weight before it meets V (2^-8 of sum w|v|); a score is a sum in 32 bits of D
products, off by at most D 2^-24 sum |q k| scale, in the numerator and, at most as
much, in the sum; sums over n keys in 32 bits add n 2^-24 of sum w|v| each. Joining
parts multiplies each by factors that are off by a few 2^-24: under 2^-20 for the
parts there are."""
import math

import numpy as np
import pytest

import gemma_kv as gk

pytestmark = pytest.mark.gpu

NAN = float("nan")


class Groups:
    """Groups of sequences; `groups`: (prefix keys, [(rows, keys behind the prefix), ..]).
    Tables share the prefix's whole pages; `alone`: sequences behind the groups. What no
    row sees is NaN: unused pages and slots behind the prior keys."""

    def __init__(self, dev, heads, dim, groups, page=16, alone=(), layers=2, seed=0, extra_rows=0, holes=()):
        import torch
        self.dev, self.heads, self.dim, self.page, self.layers = dev, heads, dim, page, layers
        gen = torch.Generator().manual_seed(seed + 11)
        normal = lambda *s: torch.randn(s, generator=gen).bfloat16()  # noqa: E731
        members, self.group_offsets = [], [0]
        for prefix, seqs in groups:
            members += [(len(self.group_offsets) - 1, prefix, n, own) for n, own in seqs]
            self.group_offsets.append(len(members))
        members += [(-1, 0, n, own) for n, own in alone]
        self.rows = [m[2] for m in members]
        self.prior = [m[1] + m[3] for m in members]
        self.batch, self.total = len(members), sum(self.rows) + extra_rows
        self.max_pages = max(1, max(-(-(p + n) // page) for p, n in zip(self.prior, self.rows)))
        mapped, held, count = [], {}, 0
        for g, prefix, n, own in members:
            row = []
            for j in range(-(-(prefix + own) // page)):
                key = ("group", g, j) if g >= 0 and (j + 1) * page <= prefix else ("own", len(mapped), j)
                if key not in held:
                    held[key] = count
                    count += 1
                row.append(held[key])
            mapped.append(row)
        self.pages = count + 3
        order = torch.randperm(self.pages, generator=gen)
        self.table = torch.full((self.batch, self.max_pages), -1, dtype=torch.int32)
        ck, cv = (torch.full((layers, self.pages, page, heads, dim), NAN, dtype=torch.bfloat16) for _ in range(2))
        for b, row in enumerate(mapped):
            for j, at in enumerate(row):
                self.table[b, j] = int(order[at])
                live = min(page, self.prior[b] - j * page)
                for c in (ck, cv):
                    if bool(c[0, order[at], live - 1].isnan().any()):
                        c[:, order[at], :live] = normal(layers, live, heads, dim)
        for b, j in holes:
            self.table[b, j] = -1
        self.ck, self.cv, self.table = ck.to(dev), cv.to(dev), self.table.to(dev)
        self.q = normal(self.total, 16, dim).to(dev)
        self.k, self.v = normal(self.total, heads, dim).to(dev), normal(self.total, heads, dim).to(dev)
        self.config = gk.make_config(layers, self.pages, page, self.max_pages, self.batch, heads, dim, 0)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        self.offsets, self.lengths = i32(np.cumsum([0] + self.rows).tolist()), i32(self.prior)
        self.group_count, self.group_at = len(groups), i32(self.group_offsets)
        self.scale = 1.0 / math.sqrt(dim)
        shape = (self.config, self.batch, self.total)
        self.plan_bytes = gk.flash_attention_extend_shared_plan_bytes(*shape)
        self.ws_bytes = gk.flash_attention_extend_shared_workspace_bytes(*shape)
        self.plan = torch.full((self.plan_bytes,), 0xFF, dtype=torch.uint8, device=dev)
        self.ws = torch.full((self.ws_bytes,), 0xFF, dtype=torch.uint8, device=dev)

    def make_plan(self, **kw):
        gk.check(gk.flash_attention_extend_shared_plan(
            self.plan, self.plan_bytes, self.offsets, self.lengths, self.table, self.group_at, self.group_count,
            self.config, self.batch, self.total, **kw))

    def attend(self, out, layer=1, **kw):
        gk.check(gk.flash_attention_extend_shared_paged_bf16(
            out, kw.pop("q", self.q), kw.pop("k", self.k), kw.pop("v", self.v), self.ck, self.cv, self.table, self.plan,
            self.plan_bytes, self.config, layer, self.batch, self.total, self.scale, self.ws, self.ws_bytes, **kw))

    def run(self, layer=1, **kw):
        import torch
        out = torch.full((self.total, 16, self.dim), 7.0, dtype=torch.bfloat16, device=self.dev)
        self.make_plan()
        self.attend(out, layer, **kw)
        torch.cuda.synchronize()
        return out

    def blocks(self):
        """The plan's segments: row0, rows, base, prior, sequence, first tile, last tile, partial."""
        import torch
        words = self.plan.cpu().view(torch.int32)
        few = self.total <= (64 if self.heads == 8 else 96)
        size = (16 if few else 64) if self.heads == 8 else (2 if few else 8)
        shares = 32 if self.heads == 8 else 256
        first = 256 + shares * 48
        first = (first + 255) // 256 * 256 // 4
        segments = words[first:first + 8 * int(words[7])].view(-1, 8).tolist()
        assert all(s[1] <= size for s in segments)
        return segments

    def shared_tiles(self, group):
        """Tiles of a group's prefix that its rows attend together: its sequences' own blocks begin there."""
        members = range(self.group_offsets[group], self.group_offsets[group + 1])
        own = {b: [s[5] for s in self.blocks() if s[4] == b and s[3] == self.prior[b]] for b in members if self.rows[b]}
        tiles = {min(x) for x in own.values() if x}
        assert len(tiles) == 1
        return tiles.pop()

    def check(self, out, layer=1):
        import torch
        start = 0
        for b, (n, p) in enumerate(zip(self.rows, self.prior)):
            if n == 0:
                continue
            keys = torch.arange(p, device=self.dev)
            held = self.table[b].long()[keys // self.page]
            keys, held = keys[held >= 0], held[held >= 0]
            new = slice(start, start + n)
            k = torch.cat([self.ck[layer, held, keys % self.page], self.k[new]]).double()
            v = torch.cat([self.cv[layer, held, keys % self.page], self.v[new]]).double()
            at = torch.cat([keys, p + torch.arange(n, device=self.dev)])
            hidden = at > p + torch.arange(n, device=self.dev)[:, None]
            for h in range(16):
                kv = h * self.heads // 16
                x = (self.q[new, h].double() @ k[:, kv].t() * self.scale).masked_fill(hidden, -math.inf)
                w = torch.softmax(x, -1)
                # A key that a row does not see has no part in it, whatever it holds.
                seen = torch.where(hidden[:, :, None], 0.0, v[None, :, kv])
                o, a = (torch.matmul(w[:, None], s)[:, 0] for s in (seen, seen.abs()))
                s = float((self.q[new, h].double().abs() @ k[:, kv].abs().t()).nan_to_num(0, 0, 0).max()) * self.scale
                bound = 2.0**-8 * o.abs() + a * (2.0**-8 + 2.0**-20 + 2 * self.dim * 2.0**-24 * s + 2 * len(at) * 2.0**-24) * (1 + 2.0**-7)
                off = (out[new, h].double() - o).abs()
                ok = (off <= bound + 1e-30) | (o.isnan() & out[new, h].isnan()) | (out[new, h].double() == o)
                assert bool(ok.all()), (b, h, float((off / bound).nan_to_num(0).max()))
            start += n
        assert bool((out[start:] == 7.0).all())


GEOMETRIES = [(8, 256), (1, 512)]


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("page", [16, 64, 24])
@pytest.mark.parametrize("groups,alone", [
    # One token each; some right behind the prefix.
    ([(960, [(1, 0), (1, 5), (1, 200), (1, 31), (1, 64)])], []),
    # Two groups, sequences in none, some without rows, drafts, a message.
    ([(480, [(1, 10), (3, 0), (0, 7), (9, 33)]), (1200, [(1, 1)] * 9 + [(70, 40)])], [(1, 500), (5, 0), (0, 9), (130, 20)]),
    # Prefixes too short to share, groups of one, and of none.
    ([(16, [(1, 3), (1, 4)]), (640, [(2, 9)]), (96, []), (32, [(1, 0)] * 40)], [(1, 0)]),
], ids=["tokens", "mixed", "short"])
def test_groups(dev, heads, dim, page, groups, alone):
    groups = [(p // page * page, m) for p, m in groups]
    g = Groups(dev, heads, dim, groups, page, alone, seed=page)
    g.check(g.run())


# Of both kernels, by the call's rows: geometry, sequences, prefix keys, rows of a block, keys of a tile.
SHARING = [(8, 256, 6, 1024, 16, 64), (1, 512, 25, 7168, 2, 64), (8, 256, 70, 640, 64, 32), (1, 512, 104, 2048, 8, 32)]


@pytest.mark.parametrize("heads,dim,count,prefix,block,tile", SHARING)
def test_the_prefix_is_in_blocks_of_all_rows(dev, heads, dim, count, prefix, block, tile):
    import torch
    g = Groups(dev, heads, dim, [(prefix, [(1, 40)] * count)], 16)
    g.check(g.run())
    segments, tiles = g.blocks(), prefix // tile
    shared = [s for s in segments if s[3] == prefix]
    assert sum(s[1] * (s[6] - s[5]) for s in shared) == count * tiles
    assert max(s[1] for s in shared) == min(block, count) and max(s[6] for s in shared) == tiles
    own = [s for s in segments if s[3] == prefix + 40]
    assert {s[4] for s in own} == set(range(count)) and min(s[5] for s in own) == tiles
    assert len(own) + len(shared) == len(segments) and all(s[1] == 1 for s in own)
    # Tables that part behind 16 keys share no whole tile: sequences of their own.
    g.table[4, 1:] = g.table[3, 1:].flip(0)
    g.make_plan()
    torch.cuda.synchronize()
    assert all(s[1] == 1 and s[3] == prefix + 40 and s[4] in range(count) for s in g.blocks())


@pytest.mark.parametrize("heads,dim,count,prefix,block,tile", SHARING)
@pytest.mark.parametrize("page", [16, 24])
def test_shared_prefixes(dev, heads, dim, count, prefix, block, tile, page):
    """Sharing in both kernels, and what can go wrong there: tokens and drafts, sequences without rows, pages
    that are not mapped (in the prefix for all of the group, behind it for one), infinities and NaN in
    both, rows behind the last sequence, strides, other lengths in a captured graph."""
    import torch
    prefix = prefix // page * page
    seqs = [((1, 1, 0, 2, 1)[b % 5] if count < 30 else (1, 2, 1, 0, 1, 3)[b % 6], (b * 37) % 90 + 1) for b in range(count)]
    hole = 5 * tile // page
    g = Groups(dev, heads, dim, [(prefix, seqs)], page, [(1, 200)], extra_rows=2, seed=page,
               holes=[(b, j) for b in range(count) for j in (0, hole)] + [(3, prefix // page)])
    out = g.run()
    g.check(out)
    tiles = g.shared_tiles(0)
    assert tiles == prefix // tile
    wide = torch.zeros(g.total, (16 + 2 * heads) * dim + 8, dtype=torch.bfloat16, device=dev)
    parts = wide.split([16 * dim, heads * dim, heads * dim, 8], 1)
    for to, x in zip(parts, (g.q, g.k, g.v)):
        to.copy_(x.reshape(g.total, -1))
    assert torch.equal(out, g.run(q=parts[0], k=parts[1], v=parts[2], q_stride=wide.stride(0), kv_stride=wide.stride(0)))
    # Captured, with sequences' rows and lengths that others have.
    captured = torch.zeros_like(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.make_plan()
        g.attend(captured)
    kept = g.rows, g.prior
    for shift in (1, 2, 0):
        g.rows = kept[0][shift:count] + kept[0][:shift] + kept[0][count:]
        g.prior = [p - (p - prefix) * (b == 1) for b, p in enumerate(kept[1])] if shift == 1 else kept[1]
        g.lengths.copy_(torch.tensor(g.prior, dtype=torch.int32))
        g.offsets.copy_(torch.tensor(np.cumsum([0] + g.rows), dtype=torch.int32))
        captured.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        g.check(captured)
    assert torch.equal(out, captured)
    # Values that are no numbers: of the prefix, of a row's own, of a key that later rows of a draft see only.
    first = np.cumsum([0] + g.rows)
    draft = next(b for b in range(count) if g.rows[b] > 1)
    g.v[int(first[draft]) + 1, 0, 5] = math.inf
    g.v[int(first[1]), heads - 1, 7] = NAN
    g.check(g.run())
    g.cv[1, g.table[0, hole + 1].item(), 1, heads - 1, 11] = math.inf
    out = g.run()
    g.check(out)
    assert bool(torch.isinf(out[:int(first[count]), 16 - 16 // heads:, 11]).all())


@pytest.mark.parametrize("heads,dim,count,prefix,block,tile", SHARING)
def test_pages_past_32_bits(dev, heads, dim, count, prefix, block, tile):
    """The same pages far apart: byte offsets past 2^32 within a layer, and the same result."""
    import torch
    g = Groups(dev, heads, dim, [(prefix, [(1 + b % 2, 11 * b % 70) for b in range(count)])], 64, layers=1)
    out = g.run(layer=0)
    g.check(out, layer=0)
    apart = (5 << 30) // (g.pages * 64 * heads * dim * 2)
    caches = []
    for c in (g.ck, g.cv):
        far = torch.empty(1, g.pages * apart, 64, heads, dim, dtype=torch.bfloat16, device=dev)
        far[:, ::apart] = c
        caches.append(far)
    assert caches[0].numel() * 2 > 2**32 and int(g.table.max()) * apart * 64 * heads * dim * 2 > 2**32
    g.ck, g.cv = caches
    g.table = torch.where(g.table >= 0, g.table * apart, g.table)
    g.config = gk.make_config(1, g.pages * apart, 64, g.max_pages, g.batch, heads, dim, 0)
    assert torch.equal(out, g.run(layer=0))


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_a_long_prefix(dev, heads, dim):
    """70000 keys: many steps of a segment, and sums of many."""
    g = Groups(dev, heads, dim, [(70016, [(1, 3), (2, 0), (1, 700)])], 64, layers=1)
    g.check(g.run(layer=0), layer=0)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("count", [2, 17, 33, 64, 65, 100])
def test_many_members(dev, heads, dim, count):
    g = Groups(dev, heads, dim, [(800, [(1 + (b % 3 == 0), b % 50) for b in range(count)])], 16, seed=count)
    g.check(g.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_long_prefix_of_few(dev, heads, dim):
    """A prefix cut into many parts: those that four waves fold."""
    g = Groups(dev, heads, dim, [(6400, [(1, 3), (2, 70)])], 64, layers=1)
    g.check(g.run(layer=0), layer=0)
    g = Groups(dev, heads, dim, [(6400, [(20, 3), (30, 70), (3, 0)])], 64, layers=1)
    g.check(g.run(layer=0), layer=0)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_rows_behind_the_last_sequence_and_strides(dev, heads, dim):
    import torch
    g = Groups(dev, heads, dim, [(320, [(1, 3), (2, 20), (1, 0), (4, 1)])], 16, extra_rows=5)
    g.check(g.run())
    wide = torch.zeros(g.total, (16 + 2 * heads) * dim + 8, dtype=torch.bfloat16, device=dev)
    parts = wide.split([16 * dim, heads * dim, heads * dim, 8], 1)
    for to, x in zip(parts, (g.q, g.k, g.v)):
        to.copy_(x.reshape(g.total, -1))
    same = g.run(q=parts[0], k=parts[1], v=parts[2], q_stride=wide.stride(0), kv_stride=wide.stride(0))
    assert torch.equal(same, g.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_unmapped_pages(dev, heads, dim):
    """Holes in the prefix for all of a group, and behind it for one."""
    g = Groups(dev, heads, dim, [(640, [(1, 100), (2, 50), (1, 0), (1, 90)])], 16,
               holes=[(b, j) for b in range(4) for j in (0, 7, 39)] + [(0, 42), (3, 40)])
    g.check(g.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_infinities_and_nan_of_values(dev, heads, dim):
    """In the prefix: every row sees them. Behind it, in a key that later rows of a draft see and
    earlier ones do not; in wide blocks and narrow ones."""
    import torch
    for groups in ([(320, [(1, 40), (4, 30), (1, 0)])], [(320, [(40, 40), (30, 30), (1, 0)])]):
        g = Groups(dev, heads, dim, groups, 16)
        g.v[3, 0, 5] = math.inf   # a new row's own value
        g.v[2, heads - 1, 7] = NAN
        g.check(g.run())
        page = g.table[1, 21].item()  # behind the prefix, sequence 1 only
        g.cv[1, page, 2, 0, 9] = -math.inf
        g.check(g.run())
        g.cv[1, g.table[0, 3].item(), 1, heads - 1, 11] = math.inf  # in the prefix
        out = g.run()
        g.check(out)
        group = 16 // heads
        assert bool(torch.isinf(out[:sum(g.rows), 16 - group:, 11]).all())


@pytest.mark.parametrize("heads,dim,count,prefix,block,tile", SHARING)
def test_large_scores(dev, heads, dim, count, prefix, block, tile):
    """Scores of hundreds, the largest ones late: the running maximum moves again and again."""
    import torch
    g = Groups(dev, heads, dim, [(prefix, [(1 + b % 2, 40 + b) for b in range(count)])], 16)
    g.q.mul_(24)
    keys = torch.arange(prefix // 16, device=dev) / (prefix // 16)
    pages = g.table[0, :len(keys)].long()
    g.ck[:, pages] *= (0.5 + 0.5 * keys)[None, :, None, None, None].bfloat16()
    g.check(g.run())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("rows", [3, 120])
def test_nan_of_keys_reaches_the_rows_that_see_them(dev, heads, dim, rows):
    """A row's only key, keys of one half of a step or one of its quarters alone, one of a draft."""
    g = Groups(dev, heads, dim, [(320, [(1, 40), (1, 30)])], 16, [(1, 0), (2, 0), (rows, 0), (1, 1), (1, 40), (4, 70)])
    g.k[2] = NAN            # the one key of its row
    g.k[4, heads - 1] = NAN  # the second of two
    first = 5 + rows
    g.ck[1, g.table[5, 0].item(), 0] = NAN
    g.ck[1, g.table[6, 2].item(), 3:] = NAN  # keys 35 .. 39 of 41
    g.k[first + 2 + 2] = NAN                 # of a draft's third row
    out = g.run()
    g.check(out)
    assert bool(out[2].isnan().all()) and not bool(out[3].isnan().any())
    assert bool(out[first].isnan().all()) and bool(out[first + 1].isnan().all())
    assert not bool(out[first + 2:first + 4].isnan().any()) and bool(out[first + 4:first + 6].isnan().all())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("last", [40, 100])
def test_equals_the_extension_without_groups(dev, heads, dim, last):
    """No groups, groups of one, and, beyond a few rows, the extension itself: the same cuts and the same sums."""
    import torch
    rows, keys = [1, 5, 1, last], [300, 20, 0, 77]
    g = Groups(dev, heads, dim, [], 16, alone=list(zip(rows, keys)))
    out = g.run()
    g.check(out)
    one = Groups(dev, heads, dim, [(0, [(n, p)]) for n, p in zip(rows, keys)], 16)
    assert torch.equal(out, one.run())
    plan = torch.empty(gk.flash_attention_extend_plan_bytes(g.config, 4, g.total), dtype=torch.uint8, device=dev)
    ws = torch.empty(gk.flash_attention_extend_workspace_bytes(g.config, 4, g.total), dtype=torch.uint8, device=dev)
    gk.check(gk.flash_attention_extend_plan(plan, plan.numel(), g.offsets, g.lengths, g.config, 4, g.total, 0, 0))
    plain = torch.full_like(out, 7.0)
    args = (plain, g.q, g.k, g.v, g.ck, g.cv, g.table)
    tail = (g.config, 1, 4, g.total, g.scale)
    gk.check(gk.flash_attention_extend_paged_bf16(*args, plan, plan.numel(), *tail, ws, ws.numel()))
    torch.cuda.synchronize()
    if last == 100:
        assert torch.equal(out, plain)
    # A plan of the other kind: nothing is written.
    plain.fill_(7.0)
    other = torch.zeros(max(plan.numel(), g.plan_bytes), dtype=torch.uint8, device=dev)
    other[:g.plan_bytes].copy_(g.plan)
    gk.check(gk.flash_attention_extend_paged_bf16(*args, other, other.numel(), *tail, ws, ws.numel()))
    torch.cuda.synchronize()
    assert bool((plain == 7.0).all())
    other[:plan.numel()].copy_(plan)
    g.plan, g.plan_bytes = other, other.numel()
    g.attend(plain)
    torch.cuda.synchronize()
    assert bool((plain == 7.0).all())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_bad_offsets_stay_within(dev, heads, dim):
    """Group and row offsets that do not ascend or pass the batch: rows are still one sequence's
    and nothing outside is written."""
    import torch
    g = Groups(dev, heads, dim, [(320, [(1, 3)] * 5)], 16, extra_rows=3)
    for groups in ([3, 1, 9], [-4, 2**30, 2], [5, 5, 5]):
        g.group_at, g.group_count = torch.tensor(groups, dtype=torch.int32, device=dev), 2
        g.check(g.run())
    g.group_at, g.group_count = torch.tensor([0, 5], dtype=torch.int32, device=dev), 1
    g.offsets = torch.tensor([0, 2, 1, -9, 400, 3], dtype=torch.int32, device=dev)
    out = g.run()
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_captured_with_other_lengths_and_two_at_once(dev, heads, dim):
    import torch
    g = Groups(dev, heads, dim, [(480, [(1, 30), (1, 40), (2, 50)])], 16)
    out = torch.zeros(g.total, 16, dim, dtype=torch.bfloat16, device=dev)
    g.make_plan()
    g.attend(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.make_plan()
        g.attend(out)
    for prior, rows, offsets in ([510, 520, 530], [1, 1, 2], [0, 3]), ([480, 500, 490], [2, 1, 1], [0, 3]), ([33, 520, 0], [0, 1, 3], [0, 2]):
        g.prior, g.rows = prior, rows
        g.lengths.copy_(torch.tensor(prior, dtype=torch.int32))
        g.offsets.copy_(torch.tensor(np.cumsum([0] + rows), dtype=torch.int32))
        g.group_at.copy_(torch.tensor(offsets, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        g.check(out)
    a = Groups(dev, heads, dim, [(960, [(1, 30)] * 7)], 16, seed=3)
    b = Groups(dev, heads, dim, [(480, [(3, 200)] * 5)], 16, seed=4)
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    torch.cuda.synchronize()
    for x, s in zip((a, b), streams):
        with torch.cuda.stream(s):
            o = torch.full((x.total, 16, dim), 7.0, dtype=torch.bfloat16, device=dev)
            x.make_plan()
            x.attend(o)
            outs.append(o)
    torch.cuda.synchronize()
    for x, o in zip((a, b), outs):
        x.check(o)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_two_graphs_share_a_plan_and_a_workspace(dev, heads, dim):
    """A small call and a large one in the large one's buffers, each a graph, replayed in turn."""
    import torch
    large = Groups(dev, heads, dim, [(1280, [(2, b) for b in range(60)])], 64, seed=1)
    small = Groups(dev, heads, dim, [(8000, [(1, 10 * b) for b in range(20)])], 64, [(3, 50)], seed=2)
    assert small.plan_bytes <= large.plan_bytes and small.ws_bytes <= large.ws_bytes
    small.plan, small.plan_bytes, small.ws, small.ws_bytes = large.plan, large.plan_bytes, large.ws, large.ws_bytes
    outs, graphs = [], []
    for g in (large, small):
        outs.append(torch.full((g.total, 16, dim), 7.0, dtype=torch.bfloat16, device=dev))
        g.make_plan()
        g.attend(outs[-1])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            g.make_plan()
            g.attend(outs[-1])
    for which in (0, 1, 1, 0, 0, 1):
        outs[which].fill_(7.0)
        graphs[which].replay()
        torch.cuda.synchronize()
        (large, small)[which].check(outs[which])


def test_runs_are_alike(dev):
    import torch
    g = Groups(dev, 1, 512, [(2048, [(1, 20 * b) for b in range(12)])], 64, layers=1)
    out = g.run(layer=0)
    assert all(torch.equal(out, g.run(layer=0)) for _ in range(5))


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_a_step_of_branches(dev, heads, dim):
    """Together as a server uses them: a prompt's rows prepared from their projection and
    appended, the prompt forked, the branches' next tokens prepared, attended in their
    group and appended, twice."""
    import torch
    gen = torch.Generator().manual_seed(21)
    page, branches, prompt = 16, 5, 339
    batch, max_pages = branches + 1, 24
    pages = 40
    config = gk.make_config(1, pages, page, max_pages, batch, heads, dim, 0)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev)
    refs, status, lengths = torch.zeros(pages, dtype=torch.int32, device=dev), i32(9), i32(*[0] * batch)
    ck, cv = (torch.full((1, pages, page, heads, dim), NAN, dtype=torch.bfloat16, device=dev) for _ in range(2))
    turns, amplitude = gk.rope_frequencies(dim // 4, 1e6, gk.ROPE_BY_PARTS, 8.0, 32768.0)
    turns = torch.from_numpy(turns).to(dev)
    wq, wk = ((1 + 0.2 * torch.randn(dim, generator=gen)).bfloat16().to(dev) for _ in range(2))
    width = (16 + heads) * dim

    def prepared(positions):
        n = len(positions)
        projected = torch.randn(n, width, generator=gen).bfloat16().to(dev)
        out = [torch.empty(n, m, dim, dtype=torch.bfloat16, device=dev) for m in (16, heads, heads)]
        gk.check(gk.rope_rows_bf16(*out, projected, projected[:, 16 * dim:], None, wq, wk, i32(*positions), turns, amplitude,
                                   dim // 4, False, heads, dim, n, q_stride=width, kv_stride=width))
        return out

    gk.check(gk.kv_cache_reserve_pages(table, refs, config, lengths, i32(prompt, *[0] * branches), status))
    _, k, v = prepared(list(range(prompt)))
    gk.check(gk.kv_cache_write_bf16(ck, cv, config, table, i32(*[0] * prompt), i32(*range(prompt)), prompt, 0, k, v))
    lengths[0] = prompt
    gk.check(gk.kv_cache_fork_bf16(ck, cv, config, table, refs, lengths, i32(*[0] * branches), i32(*range(1, batch)), branches, status))
    torch.cuda.synchronize()
    assert status.item() == 0
    keys = [[(k[:, h], v[:, h]) for h in range(heads)] for _ in range(branches)]
    shape = (config, batch, branches)
    plan = torch.empty(gk.flash_attention_extend_shared_plan_bytes(*shape), dtype=torch.uint8, device=dev)
    ws = torch.empty(gk.flash_attention_extend_shared_workspace_bytes(*shape), dtype=torch.uint8, device=dev)
    for step in range(2):
        at = prompt + step
        end = lengths.clone()
        end[1:] += 1
        gk.check(gk.kv_cache_reserve_pages(table, refs, config, lengths, end, status))
        q, k, v = prepared([at] * branches)
        # The prompt itself brings no row; branches are the group.
        gk.check(gk.flash_attention_extend_shared_plan(plan, plan.numel(), i32(0, 0, *range(1, batch)), lengths, table,
                                                       i32(1, batch), 1, *shape))
        out = torch.zeros(branches, 16, dim, dtype=torch.bfloat16, device=dev)
        gk.check(gk.flash_attention_extend_shared_paged_bf16(out, q, k, v, ck, cv, table, plan, plan.numel(), config, 0, batch,
                                                             branches, 1 / math.sqrt(dim), ws, ws.numel()))
        gk.check(gk.kv_cache_write_bf16(ck, cv, config, table, i32(*range(1, batch)), i32(*[at] * branches), branches, 0, k, v))
        lengths.copy_(end)
        torch.cuda.synchronize()
        assert status.item() == 0
        for b in range(branches):
            for h in range(16):
                kv = h * heads // 16
                kd, vd = (torch.cat([old, x[b:b + 1, kv]]) for old, x in zip(keys[b][kv], (k, v)))
                w = torch.softmax(kd.double() @ q[b, h].double() / math.sqrt(dim), 0)
                o, a = w @ vd.double(), w @ vd.double().abs()
                assert bool(((out[b, h].double() - o).abs() <= 2.0**-8 * o.abs() + a * (2.0**-8 + 2.0**-11)).all()), (step, b, h)
            keys[b] = [tuple(torch.cat([old, x[b:b + 1, kv]]) for old, x in zip(keys[b][kv], (k, v))) for kv in range(heads)]
