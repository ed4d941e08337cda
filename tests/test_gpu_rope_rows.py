"""Preparation of ragged rows (RMSNorm and rotary positions) against its definition in
64 bits.

Tolerance, before any run: an output is rounded once to bf16 (2^-8 |o|). Before that,
in 32 bits: the sum of D squares is off by at most D 2^-24 of itself, the root by
half of that; the root, the division, the weight, the rotation and the amplitude are
under ten roundings of 2^-24. The turns' fraction (at most a half) is rounded to 32
bits, 2^-26 of a turn or 2^-23 of an angle, and sincospi is off by 2 units of its
last place, 2^-23 at most: together 2^-22 of |a| + |b|, the pair's size."""
import math

import numpy as np
import pytest

import gemma_kv as gk

pytestmark = pytest.mark.gpu

GEOMETRIES = [(8, 256), (1, 512)]


class Rows:
    def __init__(self, dev, heads, dim, positions, rotary, interleaved, norm=True, own_v=None, seed=0, pad=0,
                 amplitude=1.0, turns=None):
        import torch
        self.dev, self.heads, self.dim, self.rotary, self.interleaved = dev, heads, dim, rotary, interleaved
        self.norm, self.amplitude, self.rows = norm, amplitude, len(positions)
        self.own_v = heads == 8 if own_v is None else own_v
        gen = torch.Generator().manual_seed(seed)
        widths = [16 * dim, heads * dim] + [heads * dim] * self.own_v
        self.stride = sum(widths) + pad
        self.projected = torch.randn(self.rows, self.stride, generator=gen).bfloat16().to(dev)
        parts = self.projected[:, :sum(widths)].split(widths, 1)
        self.q, self.k, self.v = parts[0], parts[1], parts[2] if self.own_v else None
        self.wq, self.wk = ((1 + 0.5 * torch.randn(dim, generator=gen)).bfloat16().to(dev) for _ in range(2))
        self.position = torch.tensor(positions, dtype=torch.int32, device=dev)
        if turns is None:
            turns = gk.rope_frequencies(rotary, 1e4)[0]
        self.turns = torch.from_numpy(np.asarray(turns)).to(dev)
        self.out = [torch.full((self.rows, n, dim), 7.0, dtype=torch.bfloat16, device=dev) for n in (16, heads, heads)]

    def call(self, with_v=True, **kw):
        return gk.rope_rows_bf16(
            self.out[0], self.out[1], self.out[2] if with_v else None, self.q, self.k,
            self.v if with_v else None, self.wq if self.norm else None, self.wk if self.norm else None,
            self.position, self.turns, self.amplitude, self.rotary, self.interleaved, self.heads, self.dim,
            self.rows, q_stride=self.stride, kv_stride=self.stride, **kw)

    def check(self, with_v=True):
        import torch
        dim, half = self.dim, self.rotary // 2
        angle = torch.remainder(self.position.double()[:, None] * self.turns, 1.0) * 2 * math.pi
        cos, sin = torch.cos(angle)[:, None] * self.amplitude, torch.sin(angle)[:, None] * self.amplitude
        i = torch.arange(half, device=self.dev)
        first, second = (2 * i, 2 * i + 1) if self.interleaved else (i, i + half)
        there = (self.position >= 0)[:, None, None]
        fp32 = dim * 2.0**-25 + 10 * 2.0**-24

        def normed(x):
            x = x.reshape(self.rows, -1, dim).double()
            return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() if self.norm else x
        for got, x, w in ((self.out[0], self.q, self.wq), (self.out[1], self.k, self.wk)):
            y = normed(x) * (w.double() if self.norm else 1.0)
            o, size = y.clone(), y.abs()
            a, b = y[..., first], y[..., second]
            o[..., first], o[..., second] = a * cos - b * sin, a * sin + b * cos
            size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(self.amplitude)
            bound = 2.0**-8 * o.abs() + size * (fp32 + 2.0**-22)
            off = (got.double() - o).abs()
            assert bool(((off <= bound) | ~there).all()), float((off / bound).max())
            assert bool(((got == 7.0) | there).all())
        if with_v:
            x = (self.v if self.own_v else self.k).reshape(self.rows, -1, dim).double()
            o = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
            off = (self.out[2].double() - o).abs()
            assert bool(((off <= o.abs() * (2.0**-8 + fp32)) | ~there).all())
            assert bool(((self.out[2] == 7.0) | there).all())
        else:
            assert bool((self.out[2] == 7.0).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("part", [1, 2, 4, 0])
def test_layouts_and_parts(dev, heads, dim, part, interleaved):
    rotary = dim // part if part else 16
    r = Rows(dev, heads, dim, [0, 1, 7, 1000, -1, 131071], rotary, interleaved, seed=part, pad=24)
    gk.check(r.call())
    r.check()


@pytest.mark.parametrize("rotary", [48, 112, 240, 272, 496])
@pytest.mark.parametrize("interleaved", [False, True])
def test_odd_parts(dev, rotary, interleaved):
    for heads, dim in GEOMETRIES:
        if rotary > dim:
            continue
        r = Rows(dev, heads, dim, list(range(5, 38)), rotary, interleaved, seed=rotary)
        gk.check(r.call())
        r.check()


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_without_norms_and_without_v(dev, heads, dim):
    r = Rows(dev, heads, dim, [3, 99, 4096], dim // 2, False, norm=False)
    gk.check(r.call(with_v=False))
    r.check(with_v=False)
    # v may be normed where q and k are not.
    r = Rows(dev, heads, dim, [3, 99, 4096], dim // 2, True, norm=False, own_v=True)
    gk.check(r.call())
    r.check()


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
@pytest.mark.parametrize("own_v", [False, True])
def test_value_from_key_or_own(dev, heads, dim, own_v):
    r = Rows(dev, heads, dim, [0, 12, 13], dim, False, own_v=own_v, seed=4)
    gk.check(r.call())
    r.check()


@pytest.mark.parametrize("scaling", [gk.ROPE_PLAIN, gk.ROPE_LINEAR, gk.ROPE_BASE, gk.ROPE_BY_PARTS])
@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_far_positions_with_scaled_frequencies(dev, heads, dim, scaling):
    turns, amplitude = gk.rope_frequencies(dim // 4, 1e6, scaling, 16.0, 8192.0)
    positions = [1, 8191, 8192, 131072, 1_000_003, 2**24 + 1, 2**30 + 5, 2**31 - 1]
    r = Rows(dev, heads, dim, positions, dim // 4, False, amplitude=amplitude, turns=turns, seed=scaling)
    gk.check(r.call())
    r.check()


@pytest.mark.parametrize("heads,dim", GEOMETRIES)
def test_equals_the_runtime_tables_preparation(dev, heads, dim):
    """The prefill launcher's prepared rows, from tables of the same frequencies: both are
    the same arithmetic with cos and sin a unit of their last place apart."""
    import torch
    rows, rotary = 33, 256 if heads == 8 else 128
    turns = gk.rope_frequencies(rotary, 1e4 if heads == 8 else 1e6, exponent_dim=dim)[0]
    r = Rows(dev, heads, dim, list(range(rows)), rotary, False, turns=turns)
    gk.check(r.call())
    angle = torch.remainder(r.position.double()[:, None] * r.turns, 1.0) * 2 * math.pi
    cos, sin = torch.cos(angle).float().contiguous(), torch.sin(angle).float().contiguous()
    q, k = r.q.reshape(rows, 16, dim).contiguous(), r.k.reshape(rows, heads, dim).contiguous()
    prepared = [torch.zeros_like(x) for x in (q, q, k, k)]
    if heads == 8:
        v = r.v.reshape(rows, heads, dim).contiguous()
        gk.check(gk.flash_attention_sliding_fwd_bf16_norm_rope(
            *prepared, q, k, v, r.wq, r.wk, cos, sin, r.position, 1, rows, rows, 1024, 1 / 16))
    else:
        gk.check(gk.flash_attention_global_fwd_bf16_norm_rope(
            *prepared, q, k, r.wq, r.wk, cos, sin, r.position, 1, rows, rows, 1 / 32))
    # Two roundings to bf16 of values 2^-21 of the pair's size apart.
    for got, other in zip(r.out, prepared[1:]):
        size = other.double().abs().amax(-1, keepdim=True) * 2 * 2.0**-21
        assert bool(((got.double() - other.double()).abs() <= 2.0**-7 * other.double().abs() + size).all())


def test_many_rows_packed_and_other_stream(dev):
    import torch
    turns = torch.from_numpy(gk.rope_frequencies(256, 1e4)[0]).to(dev)
    r = Rows(dev, 8, 256, [int(x) for x in np.random.default_rng(2).integers(0, 40000, 4100)], 256, False, seed=9)
    q, k, v = (x.reshape(r.rows, -1, 256).contiguous() for x in (r.q, r.k, r.v))
    r.q, r.k, r.v, r.turns = q, k, v, turns
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gk.check(gk.rope_rows_bf16(*r.out, q, k, v, r.wq, r.wk, r.position, turns, 1.0, 256, False, 8, 256, r.rows))
    torch.cuda.current_stream().wait_stream(side)
    r.check()


def test_captured_and_replayed(dev):
    import torch
    r = Rows(dev, 1, 512, [5, 6, 7], 128, False)
    gk.check(r.call())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gk.check(r.call())
    for step in range(3):
        r.position.copy_(torch.tensor([step, 70 * step + 1, 2**20 + step], dtype=torch.int32))
        r.projected.copy_(torch.randn_like(r.projected))
        for o in r.out:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        r.check()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_keeps_inner_products_of_positions(dev, interleaved):
    """q at i and k at j depend on i - j only: shifting both leaves their product, up to the
    roundings of each side (2^-8 of each element, twice each)."""
    import torch
    base = Rows(dev, 1, 512, [100, 100], 512, interleaved, norm=False, seed=3)
    shifted = Rows(dev, 1, 512, [700_100, 700_100], 512, interleaved, norm=False, seed=3)
    dots, sizes = [], []
    for r in (base, shifted):
        gk.check(r.call(with_v=False))
        torch.cuda.synchronize()
        q, k = r.out[0][0].double(), r.out[1][1].double()
        dots.append(q @ k[0])
        sizes.append(q.abs() @ k[0].abs())
    assert bool(((dots[0] - dots[1]).abs() <= (sizes[0] + sizes[1]) * 2 * 2.0**-8 * (1 + 2.0**-8)).all())
