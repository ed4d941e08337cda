"""Plans of groups that share a prefix beyond what one round of a workgroup's threads holds:
hundreds of sequences, more row blocks than threads, chunks of thousands of rows. Against
the extension's definition in 64 bits, with the tolerance of test_gpu_shared_prefix.py; the
plan's counts against the sections that hold them, and nothing behind the buffers."""
import numpy as np
import pytest

import gemma_kv as gk
from test_gpu_shared_prefix import Groups

pytestmark = pytest.mark.gpu

GUARD = 4096


def up(n):
    return -(-n // 256) * 256


def sections(heads, batch, rows):
    """What a plan has room for: segments, merged rows, partial rows (batches beyond a few rows)."""
    block, wave_rows, shares = (64, 16, 32) if heads == 8 else (8, 2, 256)
    few = min(batch, rows)
    wide = rows // (wave_rows + 1)
    last = min(block, rows)
    cut = last if last <= wave_rows else -(-last // wave_rows) * wave_rows
    prefixes = rows // block + few // 2

    def part(n):
        return rows + (wave_rows - 1) * min(wide, n)
    return (rows // block + few + shares + prefixes, (shares - 1) * cut + part(prefixes),
            2 * (shares - 1) * cut + part(prefixes) + part(prefixes + batch))


class Guarded(Groups):
    """Buffers of the stated sizes with bytes behind them that stay."""

    def __init__(self, *args, **kw):
        import torch
        super().__init__(*args, **kw)
        self.behind = []
        for name, n in (("plan", self.plan_bytes), ("ws", self.ws_bytes)):
            whole = torch.full((n + GUARD,), 0xA5, dtype=torch.uint8, device=self.dev)
            setattr(self, name, whole[:n])
            self.behind.append(whole[n:])

    def check_plan(self):
        assert all(bool((b == 0xA5).all()) for b in self.behind)
        words = self.plan.cpu().numpy().view(np.int32)
        segments, merges = int(words[7]), int(words[8])
        most = sections(self.heads, self.batch, self.total)
        assert 0 < segments <= most[0] and merges <= most[1]
        block, wave_rows = (64, 16) if self.heads == 8 else (8, 2)
        rows_covered = np.zeros(self.total, dtype=np.int64)
        for row0, rows, base, prior, _, lo, hi, partial in self.blocks():
            assert 0 < rows <= block and lo < hi
            stride = rows if rows <= wave_rows else -(-rows // wave_rows) * wave_rows
            assert -1 <= partial and partial + stride <= most[2]
            rows_covered[base + row0:base + row0 + rows] += min(hi * 32, prior + row0 + rows) - lo * 32
        return rows_covered

    def shared_tiles(self, group):
        """As there, by the sequences behind the first, whose prior a prefix's blocks may have too."""
        first = {}
        for _, _, _, prior, b, lo, _, _ in self.blocks():
            if prior == self.prior[b]:
                first[b] = min(lo, first.get(b, lo))
        members = range(self.group_offsets[group] + 1, self.group_offsets[group + 1])
        tiles = {first[b] for b in members if self.rows[b]}
        assert len(tiles) == 1
        return tiles.pop()

    def check_some(self, out, rows, layer=1):
        """The definition for some rows (of no mapped keys that are no numbers)."""
        import torch
        first = np.cumsum([0] + self.rows)
        for r in rows:
            b = int(np.searchsorted(first, r, side="right")) - 1
            n, p = r - int(first[b]), self.prior[b]
            keys = torch.arange(p, device=self.dev)
            held = self.table[b].long()[keys // self.page]
            new = slice(int(first[b]), r + 1)
            k = torch.cat([self.ck[layer, held, keys % self.page], self.k[new]]).double()
            v = torch.cat([self.cv[layer, held, keys % self.page], self.v[new]]).double()
            q = self.q[r].double().view(self.heads, -1, self.dim)  # [KV head][its queries]
            # (In one contiguous operand a head; 64 bits.)
            kt, vt = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
            w = torch.softmax(torch.matmul(q, kt) * self.scale, -1)
            o, a = (torch.matmul(w, x).reshape(16, self.dim) for x in (vt, vt.abs()))
            s = float(torch.matmul(q.abs(), kt.abs()).max()) * self.scale
            count = p + n + 1
            bound = 2.0**-8 * o.abs() + a * (2.0**-8 + 2.0**-20 + 2 * self.dim * 2.0**-24 * s
                                             + 2 * count * 2.0**-24) * (1 + 2.0**-7)
            off = (out[r].double() - o).abs()
            assert bool((off <= bound).all()), (r, b, float((off / bound).max()))


GEOMETRIES = [(8, 256), (1, 512)]


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("kind", ["tokens", "four_waves", "pairs"])
def test_hundreds_of_sequences(dev, heads, dim, kind):
    """Single tokens of 330 sequences in three groups and some in none; 250 sequences whose blocks pass
    the four waves' threads; 600 sequences in 300 groups."""
    if kind == "tokens":
        groups = [(1280, [(1, 3 + b % 90) for b in range(150)]), (640, [(b % 3 and 1, b % 40) for b in range(120)]),
                  (16, [(1, 2)] * 30)]
        alone = [(1, b) for b in range(30)]
    elif kind == "four_waves":
        groups = [(1920, [(1 + b % 3, b % 33) for b in range(200)])]
        alone = [(1 + 20 * (b % 4 == 0), 7 * b) for b in range(50)]
    else:
        groups = [(160 + 16 * (g % 5), [(1 + g % 2, 5), (2, g % 60)]) for g in range(300)]
        alone = []
    g = Guarded(dev, heads, dim, groups, 16, alone, layers=1, seed=len(kind), extra_rows=3)
    units = g.batch + g.group_count
    assert units > 256 if kind != "four_waves" else units <= 256 and g.total // (64 if heads == 8 else 8) <= 256
    out = g.run(layer=0)
    g.check(out, layer=0)
    covered = g.check_plan()
    assert (covered >= np.concatenate([p + 1 + np.arange(n) for p, n in zip(g.prior, g.rows)] + [np.zeros(3)])).all()
    assert (covered <= np.concatenate([[p + n] * n for p, n in zip(g.prior, g.rows)] + [np.zeros(3)])).all()
    if kind == "tokens":
        assert g.shared_tiles(0) == 40
    if kind == "four_waves":
        assert g.shared_tiles(0) == 60 and len(g.blocks()) > 256


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_blocks_of_many_rounds(dev, heads, dim):
    """More row blocks than the plan's 1024 threads, cut by every share: chunks of thousands of rows and
    single tokens behind one prefix."""
    chunk = 2500 if heads == 1 else 18000
    g = Guarded(dev, heads, dim, [(1024, [(chunk, 70), (1, 5), (chunk // 2, 0), (3, 40)] + [(1, b) for b in range(60)])],
                64, [(chunk, 33), (1, 900), (chunk, 0)], layers=1)
    out = g.run(layer=0)
    rng = np.random.default_rng(3)
    first = np.cumsum([0] + g.rows)
    some = set(rng.integers(0, g.total, 150).tolist()) | {int(r) for r in first[:-1]} | {int(r) - 1 for r in first[1:]}
    g.check_some(out, sorted(some), layer=0)
    covered = g.check_plan()
    assert (covered >= np.concatenate([p + 1 + np.arange(n) for p, n in zip(g.prior, g.rows)])).all()
    assert len(g.blocks()) > 1024
    # The same buffers and plan again: the same result.
    again = g.run(layer=0)
    assert bool((again == out).all())


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_shared_blocks_of_many_rounds(dev, heads, dim):
    """1300 single tokens behind three prefixes: a thread's second block has a prefix, too."""
    groups = [(1280, [(1, b % 9) for b in range(700)]), (960, [(1, b % 7) for b in range(400)]), (640, [(2, 3)] * 200)]
    g = Guarded(dev, heads, dim, groups, 16, layers=1)
    out = g.run(layer=0)
    g.check_some(out, range(0, g.total, 11), layer=0)
    covered = g.check_plan()
    assert (covered >= np.concatenate([p + 1 + np.arange(n) for p, n in zip(g.prior, g.rows)])).all()
    assert len(g.blocks()) > 1024 and g.shared_tiles(0) == 40 and g.shared_tiles(1) == 30


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_all_rows_in_parts(dev, heads, dim):
    """The sections' worst: every row has parts of both kinds, blocks are a row more than a wave's, and
    every share cuts one."""
    rows = 17 if heads == 8 else 3
    g = Guarded(dev, heads, dim, [(3200, [(rows, 200) for _ in range(40)])], 16, layers=1)
    out = g.run(layer=0)
    g.check_some(out, range(0, g.total, 7), layer=0)
    g.check_plan()
    assert g.shared_tiles(0) == 100


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("count", [1, 40])
def test_few_rows_in_large_blocks(dev, heads, dim, count):
    """A stated total_rows beyond the few rows' limit, with rows that no sequence holds, takes the larger
    blocks; those rows need not be there."""
    import torch
    limit = 96 if heads == 1 else 64
    # (A chunk alone, or single tokens behind a prefix.)
    groups, alone = ([], [(40, 9000)]) if count == 1 else ([(6400, [(1, b % 30) for b in range(count)])], [])
    g = Guarded(dev, heads, dim, groups, 64, alone, layers=1, extra_rows=limit + 1 - 40)
    few, rows = 40, slice(0, 40)
    assert g.total == limit + 1
    g.q, g.k, g.v = (x[rows].contiguous() for x in (g.q, g.k, g.v))
    g.make_plan()
    out = torch.full((few + 1, 16, dim), 7.0, dtype=torch.bfloat16, device=dev)
    g.attend(out, layer=0)
    torch.cuda.synchronize()
    g.check_some(out, range(0, few, 3), layer=0)
    assert bool((out[few:] == 7.0).all())
    g.check_plan()
    assert max(s[1] for s in g.blocks()) == (8 if heads == 1 else 40)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_the_most_sequences_and_groups(dev, heads, dim):
    """4096 sequences in 2048 groups, some of none."""
    groups = [(64 + 16 * (g % 3), [(1, g % 4), (g % 2, 5)]) if g % 8 else (32, []) for g in range(2048)]
    alone = [(1, b % 6) for b in range(4096 - sum(len(m) for _, m in groups))]
    g = Guarded(dev, heads, dim, groups, 16, alone, layers=1)
    assert g.batch == 4096 and g.group_count == 2048
    out = g.run(layer=0)
    g.check_some(out, range(0, g.total, 23), layer=0)
    covered = g.check_plan()
    assert (covered >= np.concatenate([p + 1 + np.arange(n) for p, n in zip(g.prior, g.rows)])).all()


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("page", [1, 7, 100, 1024])
@pytest.mark.parametrize("count", [12, 110])
def test_page_sizes(dev, heads, dim, page, count):
    """Pages of one key, of sizes that no tile divides, longer than many tiles; in both kernels."""
    prefix = 2048 // page * page
    g = Guarded(dev, heads, dim, [(prefix, [(1 + (b % 4 == 0), b % 37) for b in range(count)])], page, [(3, 0), (1, 90)], layers=1)
    out = g.run(layer=0)
    g.check_some(out, range(0, g.total, 1 + count // 40), layer=0)
    assert all(bool((b == 0xA5).all()) for b in g.behind)
