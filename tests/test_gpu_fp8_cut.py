"""Decode over codes of batches that are cut by their lengths on the device, where the cut goes
round its corners: rings (by slot and by position), a wave's last lane, batches one beyond it,
cuts that have to grow to the workgroups there are. Against the definition in 64 bits, with the
tolerance of test_gpu_fp8_cache.py."""
import pytest

import gemma_kv as gk
from test_gpu_fp8_cache import Cache

pytestmark = pytest.mark.gpu

GEOMETRIES = [(8, 256), (1, 512)]


def ring_lengths(count):
    """Shorter than the window, its length, one off, far past it, empty."""
    some = [1024, 5000, 1, 1023, 700, 1025, 33, 2048, 0, 1041, 128, 20011]
    return [some[b % len(some)] + (b // len(some)) * 17 * (b % len(some) != 8) for b in range(count)]


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("count", [2, 24, 64])
def test_rings(dev, heads, dim, page, count):
    c = Cache(dev, heads, dim, ring_lengths(count), page=page, window=1024, seed=count)
    size, splits = c.plan()
    assert splits > 1 and (heads == 1 or size >= 128)
    c.check(c.decode())
    c.check(c.decode((256, 4)))


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("count", [2, 24, 64])
def test_rings_append_equals_write_then_attend(dev, heads, dim, page, count):
    import torch
    lens = ring_lengths(count)
    position = [n - 1 for n in lens]
    position[1] = -1 if count > 2 else position[1]
    for plan in [None, (128, 8)]:
        a, b = (Cache(dev, heads, dim, lens, page=page, window=1024, seed=8) for _ in range(2))
        out = a.decode(plan, append=position)
        gk.check(gk.kv_cache_write_fp8(b.ck, b.cv, b.config, b.table, torch.arange(count, dtype=torch.int32, device=dev),
                                       torch.tensor(position, dtype=torch.int32, device=dev), count, 1, b.k, b.v, b.ks, b.vs))
        assert torch.equal(out, b.decode(plan))
        assert torch.equal(a.ck, b.ck) and torch.equal(a.cv, b.cv)
        a.check(out)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("count", [63, 64, 65, 100])
def test_full_caches_of_many(dev, heads, dim, count):
    lens = [(0, 1, 3000, 129, 1700, 32, 640)[b % 7] + 11 * (b // 7) * (b % 7 != 0) for b in range(count)]
    c = Cache(dev, heads, dim, lens, page=16, seed=count, layers=2, room=1)
    c.check(c.decode())
    a = Cache(dev, heads, dim, lens, page=16, seed=count, layers=2, room=1)
    # A sequence without keys appends behind them.
    out = a.decode(append=[max(n - 1, 0) for n in lens])
    a.check(out)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("keys", [513, 544, 545, 1090])
def test_cuts_that_grow(dev, heads, dim, keys):
    """64 equal lengths a little past whole splits: even shares give more splits than workgroups."""
    c = Cache(dev, heads, dim, [keys] * 64, page=64, layers=1)
    c.check(c.decode(layer=0), layer=0)
    c.check(c.decode((128, 9), layer=0), layer=0)


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_one_long_among_empty(dev, heads, dim):
    c = Cache(dev, heads, dim, [0] * 31 + [9000] + [0] * 31 + [1], page=64, layers=1)
    c.check(c.decode(layer=0), layer=0)


def test_longer_than_256_splits_of_512(dev):
    c = Cache(dev, 1, 512, [140_001, 300], page=64, layers=1)
    assert c.plan() == (640, 219)
    c.check(c.decode(layer=0), layer=0)
