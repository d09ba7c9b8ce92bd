"""Rotated keys next to the border of two codes, and every scale byte: what a rotation or a rounding in fewer bits, or
an angle reduced with a short 1/pi, would get wrong.

The values are chosen on the host so that the border lies closer than 32 bits tell apart and farther than the rotation's
own 64 bits miss. Cosine, sine, two products and a sum in 64 bits are each off by a few 2^-53 of |a| + |b|, together
below 2^-48, and values are taken from 2^-46 on; the far angle is the product rounded to 64 bits on both sides
(mi_gemm.h), whose cosine and sine the host has to 2^-63. So codes and scale bytes are compared exactly.
"""
import numpy as np
import pytest
from quant_numbers import grid, pack, quantise, unpack, values

pytestmark = pytest.mark.gpu


def i32(x):
    import torch

    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def append(mi, k, bits, f, pos, scale=1.0, interleaved=True):
    """Codes [n, 1, d] and scale bytes of k [n, d] appended at positions pos."""
    import torch

    n, d = k.shape
    c = mi.quant_cache(n, 1, 1, d, bits)
    x = torch.tensor(k, dtype=torch.float64).to(torch.bfloat16)
    assert (x.double().numpy() == k).all()
    x = x[:, None].cuda()
    mi.kv_append_quant(x, x, c, i32(np.arange(n)[:, None]), i32([1] * n), inv_freq=torch.tensor(f, device="cuda"),
                       positions=i32(pos), scale=scale, interleaved=interleaved)
    return unpack(c.k.cpu().numpy()[:, 0, 0], bits), c.k_scale.cpu().numpy()[:, 0, 0]


def borders(bits):
    g = grid(bits)
    return (g[1:] + g[:-1]) / 2


def bf16_of_8_bits():
    """Every bf16 from 2^-6 to 2^9."""
    return (np.arange(128, 256)[None] * 2.0 ** np.arange(-13, 2)[:, None]).reshape(-1)


def near_borders(r, bits, positions, f, size):
    """(pos, a, b) with a cos - b sin, pos f the angle, between 2^-46 and 2^-28 of `size` from a border, both to be held
    with 2^0: for each a and border the b that comes closest, of which a few come that close."""
    out = []
    a, at = bf16_of_8_bits(), borders(bits)
    for pos in positions:
        angle = np.longdouble(np.float64(pos) * np.float64(f))
        c, s = np.cos(angle), np.sin(angle)
        x = ((a[:, None] * np.float64(c) - at) / np.float64(s)).reshape(-1)  # what b should be
        aa = np.repeat(a, len(at))
        m, e = np.frexp(x)
        b = np.ldexp(np.round(m * 256), e - 8)
        y = aa * np.float64(c) - b * np.float64(s)
        border = np.tile(at, len(a))
        some = np.flatnonzero((np.abs(y - border) < 2.0 ** -28 * border) & (np.abs(b) < 500) & (np.abs(b) > 2.0 ** -10))
        for i in some[:8]:
            exact = np.longdouble(aa[i]) * c - np.longdouble(b[i]) * s
            other = np.longdouble(b[i]) * c + np.longdouble(aa[i]) * s
            room = 2.0 ** -46 * (aa[i] + abs(b[i]))
            if abs(exact - border[i]) > room and abs(other) < size and \
                    np.abs(np.abs(np.float64(other)) - at).min() > room:
                out.append((pos, aa[i], b[i], exact, other))
    return out


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("rot", [2, 16])
def test_rotated_next_to_a_border(mi, dev, bits, far, rot):
    """rot 2: components one by one; 16: vectors. The group's largest component does not turn and fixes its power."""
    r = np.random.default_rng(bits + far)
    f = np.float32(0.7310585)
    size = 400.0 if bits == 8 else 6.0
    lo, hi = (1 << 27, 1 << 31) if far else (1, 100000)
    positions = r.integers(lo, hi, 150 if bits == 8 else 9000)
    found = near_borders(r, bits, [int(p) for p in positions], f, size)
    assert len(found) >= 40
    pos, a, b, y, z = (np.array(x) for x in zip(*found))
    k = np.zeros((len(found), 32))
    k[:, 0], k[:, 1], k[:, 31] = a, b, 448.0 if bits == 8 else 6.0
    freq = np.full(rot // 2, f, np.float32)
    codes, byte = append(mi, k, bits, freq, pos)
    at, sizes = borders(bits), codes & ((1 << (bits - 1)) - 1)
    for column, want in ((0, y), (1, z)):
        n = np.searchsorted(at, np.abs(want).astype(np.longdouble))  # none lies on a border
        assert np.array_equal(sizes[:, column], n)
        assert np.array_equal(codes[:, column] >> (bits - 1), want < 0)
    assert (byte == 127).all() and (sizes[:, 31] == len(at)).all() and (sizes[:, 2:31] == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rot", [2, 32])
def test_product_next_to_a_tie(mi, dev, bits, rot):
    """cos 1 and sin 0: a times the rotation's scale lies off a tie by less than half a step of 32 bits, on the side
    that ties to even would not take."""
    r = np.random.default_rng(rot)
    n = np.arange(len(grid(bits)) - 1)
    done = 0
    while done < 24:
        i = int(r.choice(n[1:]))
        tie = borders(bits)[i]
        up = i % 2 == 0  # the number below is the even one: the product lies above the tie
        a_int = int(r.integers(129, 256)) | 1
        a = a_int / 128.0
        m, e = np.frexp(tie / a)
        lattice = 2.0 ** (int(e) - 24)
        t = tie / a / lattice
        scale_int = np.ceil(t) if up else np.floor(t)
        scale = np.float32(scale_int * lattice)
        y = np.float64(a) * np.float64(scale)  # exact: 8 and 24 bits
        if scale_int >= 2 ** 24 or y == tie or (y > tie) != up or np.float32(y) != np.float32(tie):
            continue
        done += 1
        top = np.float64(448.0 if bits == 8 else 6.0)
        k = np.zeros((3, 32))
        k[:, 0], k[:, 1] = a, -a
        if rot == 2:
            k[:, 31] = top
        else:  # the largest turns, too: a power of two times the scale, between half the top and the top
            k[:, 31] = 2.0 ** np.floor(np.log2(top / np.float64(scale)))
        turned = k.copy()
        turned[:, :rot] *= np.float64(scale)
        codes, byte = append(mi, k, bits, np.zeros(rot // 2, np.float32), [0, 5, 2 ** 31 - 1], float(scale))
        want, want_byte = quantise(turned, bits)
        assert np.array_equal(codes, want) and np.array_equal(byte, want_byte)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_every_scale_byte_reads_back(mi, dev, bits, dtype):
    """Every byte that an append writes, 27 to 246 or 252, and 255, with every code."""
    import torch

    bytes_ = np.array(list(range(27, 253 if bits == 4 else 247)) + [255])
    n = len(bytes_)
    codes = np.tile(np.arange(256), (n, 1)).astype(np.uint8).reshape(n, 1, -1, 32 * bits // 8)
    P = codes.shape[2]
    c = mi.quant_cache(n, 1, P, 32, bits)
    for t in (c.k, c.v):
        t.copy_(torch.tensor(codes))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.tensor(bytes_.astype(np.uint8))[:, None, None, None].expand(t.shape))
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    k, v = mi.kv_read_quant(c, i32(np.arange(n)[:, None]), i32([P] * n), q_start=i32(np.arange(n + 1) * P), rows=n * P, dtype=dt)
    want = values(unpack(codes[:, 0], bits), bytes_[:, None, None].repeat(P, 1), bits)
    for got in (k, v):
        got = got.double().cpu().numpy().reshape(want.shape)
        assert ((got == want) | (np.isnan(got) & np.isnan(want))).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_largest_and_smallest_groups(mi, dev, bits):
    """The borders of the bytes written: groups of zeros, below 2^-100 L, and up to the largest below 2^127."""
    tops = [0.0, 2.0 ** -133, 2.0 ** -101, 2.0 ** -100, 2.0 ** -98, 7 * 2.0 ** -100, 464 * 2.0 ** -100, 255 * 2.0 ** 119,
            2.0 ** 126, 2.0 ** 127, -2.0 ** 127, 255 * 2.0 ** 120]
    k = np.zeros((len(tops), 32))
    k[:, 7] = tops
    k[:, 9] = np.array(tops) / 2
    k[1, 9] = 0
    codes, byte = append(mi, k, bits, np.zeros(1, np.float32), [0] * len(tops))
    want, want_byte = quantise(k, bits)
    assert np.array_equal(codes, want) and np.array_equal(byte, want_byte)
    assert byte[0] == 27 and byte[7] == (252 if bits == 4 else 246) and (byte[9:] == 255).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_a_cleared_cache_holds_zeros(mi, dev, bits):
    """Scale byte 0 over codes of 0, as quant_cache makes them: tokens that no one wrote read back, and count, as zeros."""
    import torch

    c = mi.quant_cache(3, 2, 16, 64, bits)
    pages, kv, start = i32([[2, 0]]), i32([20]), i32([0, 20])
    for dt in (torch.bfloat16, torch.float32):
        k, v = mi.kv_read_quant(c, pages, kv, q_start=start, rows=20, dtype=dt)
        assert (k == 0).all() and (v == 0).all()
    q = torch.ones((20, 4, 64), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((20, 4), device="cuda")
    o = mi.paged_attn_quant(q, c, pages, kv, q_start=start, max_q_len=20, lse=lse)
    n = np.log(np.arange(1, 21))[:, None]
    assert (o == 0).all() and (np.abs(lse.double().cpu().numpy() - n) <= 2.0 ** -20 * np.maximum(n, 1)).all()
