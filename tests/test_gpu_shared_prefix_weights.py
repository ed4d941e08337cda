"""What a few rows keep of their weights in the extension of groups.

Tolerance before any run: as in test_gpu_shared_prefix.py, but a weight meets V as two bf16
numbers, the nearest and the rest, off by 2^-8 of 2^-8 of it at most, 2^-16, where one
would be off by 2^-8."""
import math

import pytest

import gemma_kv as gk  # noqa: F401
from test_gpu_shared_prefix import Groups

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim", [(8, 256), (1, 512)])
@pytest.mark.parametrize("groups,alone", [
    ([(640, [(1, 0), (1, 5), (1, 200), (2, 31), (1, 64)])], [(1, 0), (1, 1), (3, 70)]),
    ([(4096, [(1, b % 40) for b in range(50)])], []),
    ([], [(1, 1500), (40, 10), (16, 100), (1, 64)]),
], ids=["tokens", "prefix", "alone"])
def test_weights_are_two_numbers(dev, heads, dim, groups, alone):
    import torch
    g = Groups(dev, heads, dim, groups, 16, alone, layers=1, seed=5)
    assert g.total <= 64
    out = g.run(layer=0)
    start = 0
    for b, (n, p) in enumerate(zip(g.rows, g.prior)):
        keys = torch.arange(p, device=dev)
        held = g.table[b].long()[keys // g.page]
        new = slice(start, start + n)
        k, v = (torch.cat([c[0, held, keys % g.page], x[new]]).double() for c, x in ((g.ck, g.k), (g.cv, g.v)))
        hidden = torch.arange(p + n, device=dev) > p + torch.arange(n, device=dev)[:, None]
        for h in range(16):
            kv = h * heads // 16
            q = g.q[new, h].double()
            w = torch.softmax((q @ k[:, kv].t() * g.scale).masked_fill(hidden, -math.inf), -1)
            o, a = w @ v[:, kv], w @ v[:, kv].abs()
            s = float((q.abs() @ k[:, kv].abs().t()).max()) * g.scale
            bound = 2.0**-8 * o.abs() + a * (2.0**-16 + 2.0**-20 + 2 * dim * 2.0**-24 * s
                                             + 2 * (p + n) * 2.0**-24) * (1 + 2.0**-7)
            off = (out[new, h].double() - o).abs()
            assert bool((off <= bound).all()), (b, h, float((off / bound).max()))
        start += n
