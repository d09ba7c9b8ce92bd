"""NaN in a cache of 8 or 4 bits that another writer filled: the e4m3 codes 0x7f and 0xff under any scale byte, and scale
byte 255 over any codes. Such a component of V makes that component of the output NaN in the rows that see its key, one
of K the whole row, and every other value is what it was, bit for bit: the sums have one order whatever they hold.
"""
import numpy as np
import pytest
from test_paged_gpu import Batch
from test_paged_quant_gpu import hold, run

pytestmark = pytest.mark.gpu

SHAPES = [([4, 3], [50, 600], 4, 2, 64), ([16], [16], 1, 1, 32), ([40, 150], [100, 200], 8, 2, 128), ([300], [2500], 12, 12, 64),
          ([7], [3000], 4, 4, 96), ([129, 64], [129, 3000], 4, 2, 96), ([17, 5], [33, 400], 20, 1, 128), ([130], [260], 3, 3, 32),
          ([1, 1, 1], [700, 64, 3000], 8, 2, 128), ([9, 33, 2], [9, 33, 2], 8, 2, 64)]


@pytest.mark.parametrize("bits,kind", [(8, "code"), (8, "negative"), (8, "group"), (4, "group")])
@pytest.mark.parametrize("part", ["v", "k"])
@pytest.mark.parametrize("q,kv,nH,nKV,d", SHAPES)
def test_nan_reaches_its_rows_and_components(mi, dev, bits, kind, part, q, kv, nH, nKV, d):
    """code: one component's; group: byte 255 over codes of all ones, in 8 bits NaN themselves."""
    import torch

    b = hold(mi, Batch(q, kv, 16, nH, nKV, d, seed=9, one_each=max(q) == 1), bits)
    ways = [({}, *run(mi, b)), (dict(workspace=None), *run(mi, b, workspace=None)), (dict(causal=False), *run(mi, b, causal=False))]
    want = ways[0][1]
    codes, scale = (b.c.v, b.c.v_scale) if part == "v" else (b.c.k, b.c.k_scale)
    r = np.random.default_rng(d)
    seen = torch.zeros_like(want, dtype=torch.bool)
    everyone = seen.clone()
    for s, (n, m) in enumerate(zip(q, kv)):
        # new tokens of different heads, and one that was there before
        marks = [(m - n + j, j) for j in sorted({n // 3, n // 2, n - 1})] + [((m - n) // 2, 0)] * (m > n)
        for i, (at, first_row) in enumerate(marks):
            h, c, page = i % nKV, int(r.integers(d)), int(b.table[s, at // 16])
            if kind == "group":
                g = c // 32
                codes[page, h, at % 16, g * 4 * bits:(g + 1) * 4 * bits] = 255
                scale[page, h, at % 16, g] = 255
                comps = slice(32 * g, 32 * g + 32)
            else:
                codes[page, h, at % 16, c] = 0x7F if kind == "code" else 0xFF
                comps = slice(c, c + 1)
            if part == "k":
                comps = slice(None)
            heads = slice(h * (nH // nKV), (h + 1) * (nH // nKV))
            seen[b.starts[s] + first_row:b.starts[s + 1], heads, comps] = True
            everyone[b.starts[s]:b.starts[s + 1], heads, comps] = True
    for kw, o, l in ways:
        none = seen if kw.get("causal", True) else everyone
        got, lse = run(mi, b, **kw)
        assert torch.equal(torch.isnan(got), none)
        assert torch.equal(got[~none], o[~none])
        gone = none.any(-1) if part == "k" else torch.zeros_like(none[..., 0])
        assert torch.equal(torch.isnan(lse), gone) and torch.equal(lse[~gone], l[~gone])


@pytest.mark.parametrize("q,kv", [([5], [700]), ([200], [500])])
def test_several_keys_of_one_component(mi, dev, q, kv):
    """The first of them counts for a row, wherever the others lie: each component has its own."""
    import torch

    b = hold(mi, Batch(q, kv, 16, 4, 2, 128, seed=3), 8)
    want, _ = run(mi, b)
    r = np.random.default_rng(1)
    first = np.full((2, 128), 10 ** 9)
    for c in range(0, 128, 3):
        for h in range(2):
            for at in r.integers(kv[0] - q[0], kv[0], 3):
                b.c.v[int(b.table[0, at // 16]), h, at % 16, c] = 0x7F
                first[h, c] = min(first[h, c], at)
    row = np.arange(q[0])[:, None, None] + kv[0] - q[0]
    none = torch.tensor(np.repeat(row >= first, 2, axis=1)).cuda()
    got, _ = run(mi, b)
    assert torch.equal(torch.isnan(got), none) and torch.equal(got[~none], want[~none])
