"""A paged cache of 8 or 4 bits: what mi_kv_append_quant writes and mi_kv_read_quant reads back, against the
format's definition in 64 bits (quant_numbers).

Tolerances. Codes and scale bytes are compared exactly, and so is what they stand for, which bf16 and fp32 hold. A
rotated component a cos - b sin is computed in 64 bits with an angle that both sides round once alike: cosine and
sine are off by a few 2^-53, the products and the sum by as much, together below 2^-48 (|a| + |b|); only a value that
close to the border of two codes (or a group that close to the next power of two) may differ, and it is left out of
the comparison. Q as in the tests of mi_rope.
"""
import numpy as np
import pytest
from quant_numbers import grid, pack, quantise, unpack, unsure, values

pytestmark = pytest.mark.gpu


def make(shape, seed, std=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def i32(x):
    import torch

    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def filled(mi, num, nKV, P, d, bits, order="phsd", byte=0xA5):
    """A cache of nothing but `byte`, in one of two orders of slots and heads, its scales apart by an odd stride."""
    import torch

    c = mi.quant_cache(num, nKV, P, d, bits)
    out = []
    for t in c:
        n = t.shape[3]
        if order == "pshd":
            t = torch.empty((num, P, nKV, n), dtype=torch.uint8, device="cuda").transpose(1, 2)
        elif n < 16:  # scale bytes with gaps
            t = torch.empty((num, nKV, P, n + 3), dtype=torch.uint8, device="cuda")[..., 1:n + 1]
        t.fill_(byte)
        out.append(t)
    return mi.QuantCache(*out)


def same(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return bool(((a == b) | (np.isnan(a) & np.isnan(b))).all())


# ---- the numbers ------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_all_codes_read_back(mi, dev, bits, dtype):
    """Every code at every scale byte that an append writes, and what 0 and 255 give."""
    import torch

    bytes_ = [27, 28, 60, 100, 126, 127, 128, 129, 150, 200, 240, 255] + ([252] if bits == 4 else [244])
    n = len(bytes_)
    codes = np.tile(np.arange(256), (n, 1)).astype(np.uint8).reshape(n, 1, -1, 32 * bits // 8)  # rows of one group
    P = codes.shape[2]
    c = mi.quant_cache(n, 1, P, 32, bits)
    c.k.copy_(torch.tensor(codes))
    c.v.copy_(torch.tensor(codes[:, :, ::-1].copy()))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.tensor(np.array(bytes_, np.uint8))[:, None, None, None].expand(t.shape))
    pages, kv = i32(np.arange(n)[:, None]), i32([P] * n)
    start = i32(np.arange(n + 1) * P)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    k, v = mi.kv_read_quant(c, pages, kv, q_start=start, rows=n * P, dtype=dt)
    for got, held in ((k, c.k), (v, c.v)):
        want = values(unpack(held.cpu().numpy()[:, 0], bits), np.array(bytes_)[:, None, None].repeat(P, 1), bits)
        assert got.dtype == dt and same(got.double().cpu().numpy().reshape(want.shape), want)


@pytest.mark.parametrize("bits", [8, 4])
def test_every_bf16_is_quantised(mi, dev, bits):
    """All 65536 bf16 numbers, in groups of neighbours and in groups whose largest lies just at, below and above
    each border of a power of two, ties among them; infinities, NaN and the largest magnitudes too."""
    import torch

    r = np.random.default_rng(1)
    every = np.arange(65536, dtype=np.uint16)
    spread = r.permutation(65536).astype(np.uint16)
    # one magnitude of each exponent that is a tie or a border, times random smaller ones
    x = torch.tensor(every.astype(np.int32)).to(torch.int16).view(torch.bfloat16)
    top = []
    for e in (-60, -3, 0, 1, 40, 100):
        for m in (6.0, 6.5, 7.0, 7.03125, 3.5, 3.515625, 448, 464, 466, 232, 233, 1.0, 1.9921875):
            row = r.integers(-128, 129, 32) / 128 * m
            row[r.integers(32)] = m * r.choice([-1, 1])
            top.append(row * 2.0 ** e)
            g = grid(bits)
            ties = (g[1:] + g[:-1]) / 2 * r.choice([-1, 1], len(g) - 1)
            ties = r.choice(ties, 31)
            top.append(np.append(ties, g[-1]) * 2.0 ** e)
    top = torch.tensor(np.array(top), dtype=torch.float64).to(torch.bfloat16).reshape(-1)
    rows = torch.cat([x, torch.tensor(spread.astype(np.int32)).to(torch.int16).view(torch.bfloat16), top,
                      torch.zeros(32, dtype=torch.bfloat16)])
    n = rows.numel() // 32
    k = rows.view(n, 1, 32).cuda()
    c = mi.quant_cache(n, 1, 1, 32, bits)
    mi.kv_append_quant(k, k.flip(0).contiguous(), c, i32(np.arange(n)[:, None]), i32([1] * n))
    h = k.double().cpu().numpy()
    for codes, scale, x in ((c.k, c.k_scale, h), (c.v, c.v_scale, h[::-1])):
        want, byte = quantise(x, bits)
        assert np.array_equal(scale.cpu().numpy().reshape(n, 1, 1), byte)
        assert np.array_equal(codes.cpu().numpy().reshape(n, 1, -1), pack(want, bits))
    # what is read back is the nearest number, within half a step of the largest
    v = values(*quantise(h, bits), bits)
    fine = np.isfinite(v).all(-1)
    assert np.abs(v - h)[fine].max(-1, initial=0).size and (np.abs(v - h)[fine] <= np.maximum(
        np.abs(h[fine]).max(-1, keepdims=True) * (2 / 7 if bits == 4 else 2.0 ** -4), 2.0 ** -101)).all()


# ---- the append ---------------------------------------------------------------------------

def turned(x, pos, f, interleaved, scale):
    """x [n, heads, d] rotated, 64 bits."""
    n = len(f)
    a = np.asarray(pos, np.float64)[:, None] * f.astype(np.float64)
    c, s = (np.cos(a) * np.float64(np.float32(scale)))[:, None], (np.sin(a) * np.float64(np.float32(scale)))[:, None]
    y = x.copy()
    re, im = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., re], y[..., im] = x[..., re] * c - x[..., im] * s, x[..., im] * c + x[..., re] * s
    return y


def written(t, page, slot):
    return t.cpu().numpy()[page, :, slot]


APPENDS = [(4, 2, 64, 64, [1, 1, 1], [1, 17, 100], 16), (8, 2, 128, 64, [5, 0, 40, 1], [9, 3, 40, 64], 32),
           (2, 1, 32, 8, [130, 3], [131, 3], 1), (3, 3, 96, 2, [2], [2], 64), (16, 4, 128, 128, [700, 333], [1700, 400], 64),
           (12, 12, 64, 24, [3, 20], [100000, 20], 1024), (2, 2, 160, 160, [9], [9], 4), (1, 1, 1024, 1024, [3], [4], 2)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("order", ["phsd", "pshd"])
@pytest.mark.parametrize("nH,nKV,d,rot,q_len,kv_len,P", APPENDS)
def test_append_and_read(mi, dev, bits, interleaved, order, nH, nKV, d, rot, q_len, kv_len, P):
    import torch
    from test_rope_gpu import check as rope_check
    from test_rope_gpu import reference

    r = np.random.default_rng(d)
    S, n = len(q_len), sum(q_len)
    need = [-(-m // P) for m in kv_len]
    table = np.full((S, max(need) + 1), -1, np.int64)
    ids, at = r.permutation(sum(need) + 2), 0
    for s, m in enumerate(need):
        table[s, :m] = ids[at:at + m]
        at += m
    c = filled(mi, sum(need) + 2, nKV, P, d, bits, order)
    before = [t.clone() for t in c]
    f, _ = mi.rope_frequencies(rot)
    rows = n + 4
    qkv = make((rows, nH + 2 * nKV, d), 77, 3.0)
    q, k, v = qkv.split((nH, nKV, nKV), dim=1)
    starts = np.concatenate([[0], np.cumsum(q_len)])
    q_start, pages, kv = i32(starts), i32(table), i32(kv_len)
    q_out = torch.full((rows, nH, d), 5.0, dtype=torch.bfloat16, device="cuda")
    assert mi.kv_append_quant(k, v, c, pages, kv, q_start=q_start, q=q, q_out=q_out, inv_freq=f, interleaved=interleaved,
                              scale=1.5) is q_out
    assert (q_out[n:] == 5.0).all()
    fh = f.cpu().numpy()
    seq = np.repeat(np.arange(S), q_len)
    pos = np.array([kv_len[s] - q_len[s] + i - starts[s] for i, s in enumerate(seq)])
    page, slot = table[seq, pos // P], pos % P
    h = lambda t: t[:n].double().cpu().numpy()  # noqa: E731
    y, size = reference(h(q)[None], pos[None], fh, interleaved, 1.5)
    rope_check(h(q_out), y[0], size[0], True)

    def check_k(pos, scale):
        turned_k = turned(h(k), pos, fh, interleaved, scale)
        codes, byte = quantise(turned_k, bits)
        # components that do not turn, and position 0, are exact on both sides, ties among them
        turns = (np.arange(d) < rot) & (pos != 0)[:, None, None]
        size = 2 * np.abs(h(k)).max(-1, keepdims=True) * scale
        open_ = unsure(turned_k, np.where(turns, 2.0 ** -48 * size, 0.0), bits)
        assert open_.mean() < 1e-3
        sure_group = ~open_.reshape(n, nKV, -1, 32).all(-1)
        assert (written(c.k_scale, page, slot) == byte)[sure_group].all()
        assert (unpack(written(c.k, page, slot), bits) == codes)[~open_].all()

    check_k(pos, 1.5)
    codes, byte = quantise(h(v), bits)
    assert np.array_equal(written(c.v, page, slot), pack(codes, bits)) and np.array_equal(written(c.v_scale, page, slot), byte)
    # read back: rows behind the last sequence stay
    outs = [torch.full((rows, nKV, d), 9.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    mi.kv_read_quant(c, pages, kv, q_start=q_start, k_out=outs[0], v_out=outs[1])
    for out, t, sc in zip(outs, (c.k, c.v), (c.k_scale, c.v_scale)):
        assert same(h(out), values(unpack(written(t, page, slot), bits), written(sc, page, slot), bits))
        assert (out[n:] == 9.0).all()
    # nothing else was written
    pt, st = torch.tensor(page).cuda(), torch.tensor(slot).cuda()
    for now, old in zip(c, before):
        now, old = now.clone(), old.clone()
        now[pt, :, st] = 0
        old[pt, :, st] = 0
        assert torch.equal(now, old)
    # with positions of its own, in place, and without rotation
    own = torch.arange(rows, dtype=torch.int32, device="cuda") * 1237 + 7
    x = q.clone()
    mi.kv_append_quant(k, v, c, pages, kv, q_start=q_start, q=x, q_out=x, inv_freq=f, positions=own, interleaved=interleaved)
    y, size = reference(h(q)[None], own[:n].cpu().numpy()[None], fh, interleaved, 1.0)
    rope_check(h(x), y[0], size[0], True)
    check_k(own[:n].cpu().numpy(), 1.0)
    assert mi.kv_append_quant(k, v, c, pages, kv, q_start=q_start) is None
    codes, byte = quantise(h(k), bits)
    assert np.array_equal(written(c.k, page, slot), pack(codes, bits)) and np.array_equal(written(c.k_scale, page, slot), byte)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("offset,pitch", [(0, 67), (1, 64), (3, 71)])
def test_rows_at_any_alignment(mi, dev, bits, offset, pitch):
    """Rows that are no whole vectors give the codes that aligned ones give."""
    import torch

    k, v, q = make((30, 2, 64), 1), make((30, 2, 64), 2), make((30, 4, 64), 3)
    f, _ = mi.rope_frequencies(48)

    def moved(t):
        n = t.shape[0] * t.shape[1]
        w = torch.zeros((n * pitch + offset,), dtype=torch.bfloat16, device="cuda")
        w = torch.as_strided(w, t.shape, (t.shape[1] * pitch, pitch, 1), offset)
        w.copy_(t)
        return w

    pages, kv, start = i32([[0, 1], [2, 3]]), i32([20, 25]), i32([0, 10, 30])
    a, b = mi.quant_cache(4, 2, 16, 64, bits), mi.quant_cache(4, 2, 16, 64, bits)
    qa = mi.kv_append_quant(k, v, a, pages, kv, q_start=start, q=q, inv_freq=f)
    qb = mi.kv_append_quant(moved(k), moved(v), b, pages, kv, q_start=start, q=moved(q), q_out=moved(q), inv_freq=f)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(qa, qb)
    for dt in (torch.bfloat16, torch.float32):
        want = mi.kv_read_quant(a, pages, kv, q_start=start, rows=30, dtype=dt)
        base = torch.full((30 * 2 * pitch + offset,), 7.0, dtype=dt, device="cuda")
        out = torch.as_strided(base, (30, 2, 64), (2 * pitch, pitch, 1), offset)
        got = mi.kv_read_quant(a, pages, kv, q_start=start, k_out=out, parts="k")
        assert got[1] is None and torch.equal(got[0], want[0])
        rest = base.clone()
        torch.as_strided(rest, (30, 2, 64), (2 * pitch, pitch, 1), offset).fill_(7.0)
        assert (rest == 7.0).all()
        got = mi.kv_read_quant(a, pages, kv, q_start=start, rows=30, parts="v", dtype=dt)
        assert got[0] is None and torch.equal(got[1], want[1])
        # [heads, tokens, d], as attention over whole sequences takes it
        t = torch.empty((2, 30, 64), dtype=dt, device="cuda").transpose(0, 1)
        mi.kv_read_quant(a, pages, kv, q_start=start, k_out=t, v_out=torch.empty_like(want[1]))
        assert torch.equal(t, want[0])


@pytest.mark.parametrize("bits", [8, 4])
def test_bad_places(mi, dev, bits):
    """Pages outside the cache, tokens before position 0: nothing written, zeros read."""
    import torch

    c = filled(mi, 6, 1, 16, 64, bits)
    pages = i32([[0, 6, 1], [2, 3, -1], [4, 2 ** 31 - 1, -7]])
    kv, start = i32([20, 40, 1]), i32([0, 1, 3, 6])  # the third: its first two rows before position 0
    want = [t.clone() for t in c]
    k, v = make((8, 1, 64), 5), make((8, 1, 64), 6)
    mi.kv_append_quant(k, v, c, pages, kv, q_start=start)
    for t, w, x in zip(c, want, (k, v, k, v)):
        codes, byte = quantise(x[5].double().cpu().numpy(), bits)
        w[4, :, 0] = torch.tensor(pack(codes, bits) if w.shape[3] > 8 else byte).cuda()
        assert torch.equal(t, w)
    out = [torch.full((8, 1, 64), 3.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    mi.kv_read_quant(c, pages, kv, q_start=start, k_out=out[0], v_out=out[1])
    for o, x in zip(out, (k, v)):
        assert (o[:5] == 0).all() and (o[6:] == 3.0).all()
        assert same(o[5].double().cpu().numpy(), values(*quantise(x[5].double().cpu().numpy(), bits), bits))
    # a cache without pages, and longer than the table
    mi.kv_append_quant(k, v, mi.quant_cache(0, 1, 16, 64, bits), pages, kv, q_start=start)
    kv[1] = 2 ** 31 - 1
    mi.kv_append_quant(k, v, c, pages, kv, q_start=start)
    got = mi.kv_read_quant(c, pages, kv, q_start=start, rows=8)[0]
    assert (got[1:3] == 0).all()


@pytest.mark.parametrize("S", [64, 65, 300, 5000])
def test_many_sequences(mi, dev, S):
    import torch

    r = np.random.default_rng(S)
    q = r.integers(0, 3, S) * (r.random(S) < 0.7)
    kv = q + r.integers(0, 5, S)
    n = int(q.sum())
    need = -(-kv // 4)
    table = np.full((S, 3), -1, np.int64)
    ids, at = r.permutation(need.sum() + 1), 0
    for s in range(S):
        table[s, :need[s]] = ids[at:at + need[s]]
        at += need[s]
    c = mi.quant_cache(int(need.sum()) + 1, 1, 4, 32, 4)
    starts = np.concatenate([[0], np.cumsum(q)])
    k, v = make((n, 1, 32), 1), make((n, 1, 32), 2)
    mi.kv_append_quant(k, v, c, i32(table), i32(kv), q_start=i32(starts))
    got = mi.kv_read_quant(c, i32(table), i32(kv), q_start=i32(starts), rows=n)
    for x, y in zip(got, (k, v)):
        assert same(x.double().cpu().numpy(), values(*quantise(y.double().cpu().numpy(), 4), 4))
    seq = np.repeat(np.arange(S), q)
    pos = kv[seq] - q[seq] + np.arange(n) - starts[seq]
    page, slot = torch.tensor(table[seq, pos // 4]).cuda(), torch.tensor(pos % 4).cuda()
    assert np.array_equal(c.v[page, :, slot].cpu().numpy(), pack(quantise(v.double().cpu().numpy(), 4)[0], 4))


@pytest.mark.parametrize("bits", [8, 4])
def test_offsets_past_32_bits(mi, dev, bits):
    """Codes and scales whose pages lie gigabytes apart."""
    import torch

    stride, top = 1 << 27, 40
    big = torch.zeros((top * stride,), dtype=torch.uint8, device="cuda")
    n = 64 * bits // 8
    view = lambda w, at: torch.as_strided(big, (top, 2, 16, w), (stride, 16 * w, w, 1), at)  # noqa: E731
    c = mi.QuantCache(view(n, 0), view(n, 1 << 20), view(2, 2 << 20), view(2, 3 << 20))
    small = mi.quant_cache(top, 2, 16, 64, bits)
    pages, kv, start = i32([[39, 20], [1, 38]]), i32([17, 30]), i32([0, 17, 40])
    k, v = make((40, 2, 64), 1), make((40, 2, 64), 2)
    for cache in (c, small):
        mi.kv_append_quant(k, v, cache, pages, kv, q_start=start)
    assert all(torch.equal(a, b) for a, b in zip(c, small))
    got = mi.kv_read_quant(c, pages, kv, q_start=start, rows=40)
    assert same(got[0].double().cpu().numpy(), values(*quantise(k.double().cpu().numpy(), bits), bits))
    assert same(got[1].double().cpu().numpy(), values(*quantise(v.double().cpu().numpy(), bits), bits))


@pytest.mark.parametrize("bits", [8, 4])
def test_far_positions(mi, dev, bits):
    """Positions of millions: the angle's product is rounded to 64 bits, 2^-53 of up to 2^31 rad."""
    import torch

    f, _ = mi.rope_frequencies(64)
    pos = np.array([0, 1, 99999, 1 << 20, 12345678, 2 ** 31 - 1, 2 ** 30 + 7])
    n = len(pos)
    k = make((n, 2, 64), 4)
    c = mi.quant_cache(n, 2, 1, 64, bits)
    mi.kv_append_quant(k, k, c, i32(np.arange(n)[:, None]), i32([1] * n), inv_freq=f, positions=i32(pos))
    want = turned(k.double().cpu().numpy(), pos, f.cpu().numpy(), False, 1.0)
    codes, byte = quantise(want, bits)
    open_ = unsure(want, np.full(want.shape, 2.0 ** -20 * np.abs(want).max()), bits)
    assert open_.mean() < 0.01
    assert (unpack(c.k.cpu().numpy()[:, :, 0], bits) == codes)[~open_].all()


def test_empty_calls(mi, dev):
    import torch

    c = mi.quant_cache(2, 1, 16, 64, 4)
    none = torch.empty((0, 1, 64), dtype=torch.bfloat16, device="cuda")
    pages, kv, start = i32([[0]]), i32([3]), i32([0, 0])
    assert mi.kv_append_quant(none, none, c, pages, kv, q_start=start, q=none).shape == (0, 1, 64)
    assert mi.kv_read_quant(c, pages, kv, q_start=start, rows=0)[0].shape == (0, 1, 64)
    empty = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    mi.kv_append_quant(none, none, c, empty, empty[:, 0].contiguous())
    assert mi.kv_read_quant(c, empty, empty[:, 0].contiguous())[1].shape == (0, 1, 64)
