"""Attention over a paged cache of 8 or 4 bits (mi_paged_attn_quant) against 64-bit formulas on the values that the
cache stands for, which bf16 holds exactly; the bound is derived in test_paged_weights_gpu and is the one of the cache
in bf16 (`bound`: scores, the weights as two bf16, sums of n terms, the output's own rounding).
"""
import numpy as np
import pytest
from quant_numbers import pack, quantise, values
from test_paged_gpu import Batch, make
from test_paged_weights_gpu import bound, close, one_way_batch

pytestmark = pytest.mark.gpu


def hold(mi, b, bits, order="phsd", spread=0.0, seed=0):
    """b's cache in 8 or 4 bits: b.c, and what it stands for as b's keys and values. Every byte of a slot without a
    token is 255: NaN in 8 bits, and a group of NaN in both. spread: sizes of groups apart by that many powers of
    two."""
    import torch

    r = np.random.default_rng(seed)
    shape = (b.num_pages, b.nKV, b.P)
    n = (b.d * bits // 8, b.d // 32)
    if order == "phsd":
        t = [torch.full((*shape, n[i]), 255, dtype=torch.uint8, device="cuda") for i in (0, 0, 1, 1)]
    else:
        t = [torch.full((b.num_pages, b.P, b.nKV, n[i]), 255, dtype=torch.uint8, device="cuda").transpose(1, 2)
             for i in (0, 0, 1, 1)]
    b.c = mi.QuantCache(*t)
    for s, m in enumerate(b.kv):
        for name, codes, scale in (("hk", b.c.k, b.c.k_scale), ("hv", b.c.v, b.c.v_scale)):
            x = np.asarray(getattr(b, name)[s], np.float64)
            if spread:
                x = x * np.repeat(2.0 ** r.integers(-spread, 1, (b.nKV, m, b.d // 32)), 32, -1)
            q, byte = quantise(x, bits)
            getattr(b, name)[s] = values(q, byte, bits)
            for i in range(-(-m // b.P)):
                rows = slice(i * b.P, min(m, (i + 1) * b.P))
                k = rows.stop - rows.start
                codes[int(b.table[s, i]), :, :k] = torch.tensor(pack(q[:, rows], bits)).cuda()
                scale[int(b.table[s, i]), :, :k] = torch.tensor(byte[:, rows]).cuda()
    return b


def run(mi, b, **kw):
    import torch

    lse = torch.full((b.rows, b.nH), 7.0, dtype=torch.float32, device="cuda")
    kw.setdefault("max_q_len", max(b.q_len + [1]))
    kw.setdefault("max_kv_len", max(b.kv + [1]))
    if b.q_start is None:
        kw.pop("max_q_len")
    return mi.paged_attn_quant(b.q, b.c, b.pages, b.kv_len, q_start=b.q_start, lse=lse, **kw), lse


HEADS = [(4, 4, 64), (8, 2, 128), (8, 1, 96), (6, 2, 32), (16, 4, 128), (17, 1, 64), (3, 1, 32)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nH,nKV,d", HEADS)
@pytest.mark.parametrize("P", [1, 16, 64, 256])
def test_decode(mi, dev, bits, nH, nKV, d, P):
    import torch

    kv = [1, 2, 63, 64, 65, 300, 129, 31]
    b = hold(mi, Batch([1] * len(kv), kv, P, nH, nKV, d, seed=P + d, one_each=True), bits)
    ref = b.reference()
    close(*run(mi, b), ref, 300)
    b.q_start = torch.arange(len(kv) + 1, dtype=torch.int32, device="cuda")
    close(*run(mi, b), ref, 300)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nH,nKV,d", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(mi, dev, bits, nH, nKV, d, causal):
    b = hold(mi, Batch([5, 1, 70, 0, 33, 16, 2], [5, 90, 130, 40, 33, 17, 2], 16, nH, nKV, d, seed=d + nH), bits)
    close(*run(mi, b, causal=causal), b.reference(causal), 130)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("order", ["phsd", "pshd"])
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([200], [1000], 8, 2, 128), ([129, 1, 64], [400, 700, 64], 4, 4, 64),
                                           ([257], [257], 4, 1, 128), ([40, 3], [2600, 1900], 4, 2, 128),
                                           ([33, 40], [700, 2048], 1, 1, 96), ([130], [4000], 3, 3, 32)])
def test_long_chunks(mi, dev, bits, order, q, kv, nH, nKV, d):
    b = hold(mi, Batch(q, kv, 32, nH, nKV, d, seed=3), bits, order)
    ref = b.reference()
    close(*run(mi, b), ref, max(kv))
    close(*run(mi, b, workspace=None), ref, max(kv))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n", [1, 500, 1023, 4096])
@pytest.mark.parametrize("d", [64, 128])
def test_long_context_split(mi, dev, bits, n, d):
    import torch

    b = hold(mi, Batch([1], [n], 16, 8, 2, d, seed=n, one_each=True), bits)
    ref = b.reference()
    full = mi.paged_attn_quant_workspace_size(8, 2, d, 1, 1, 1, n)
    for ws in ("auto", None, torch.empty((max(full // 2 // 16 * 16, 16),), dtype=torch.uint8, device="cuda"),
               torch.empty((16,), dtype=torch.uint8, device="cuda")):
        close(*run(mi, b, workspace=ws), ref, n)
    close(*run(mi, b, max_kv_len=1), ref, n)        # a sequence longer than the host said
    close(*run(mi, b, max_kv_len=1 << 20), ref, n)  # and one far shorter
    a, c = run(mi, b), run(mi, b)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("S,nH,nKV,d,P", [(140, 4, 2, 64, 16), (70, 8, 4, 128, 1), (300, 1, 1, 32, 64), (1024, 2, 1, 32, 32)])
def test_decode_many_uneven(mi, dev, bits, S, nH, nKV, d, P):
    import torch

    r = np.random.default_rng(S)
    kv = [int(x) for x in np.exp(r.uniform(0, np.log(1500), S))]
    kv[0], kv[S // 2], kv[S - 1], kv[3] = 2500, 2100, 0, 0
    b = hold(mi, Batch([1] * S, kv, P, nH, nKV, d, seed=S, one_each=True), bits)
    ref = b.reference()
    close(*run(mi, b), ref, 2500)
    n = mi.paged_attn_quant_workspace_size(nH, nKV, d, S, S, 1, max(kv))
    ws = torch.full((n + 16,), 255, dtype=torch.uint8, device="cuda")
    close(*run(mi, b, workspace=ws[:n]), ref, 2500)
    assert (ws[n:] == 255).all()
    close(*run(mi, b, workspace=ws[:n // 2 // 16 * 16]), ref, 2500)
    a, c = run(mi, b), run(mi, b)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kv,nKV,d", [([140000, 5], 1, 128), ([7, 66000], 2, 64)])
def test_one_sequence_cut_by_all_workgroups(mi, dev, bits, kv, nKV, d):
    """A share sums a thousand keys at most and the join as many parts: n = 2^11 of the bound."""
    b = hold(mi, Batch([1, 1], kv, 64, 2, nKV, d, seed=d, one_each=True), bits)
    close(*run(mi, b), b.reference(), 2 ** 11)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("kv,nH,nKV,d", [([5, 600], 2, 1, 32), ([100] * 200, 4, 4, 64), ([1, 0, 129, 128, 127] * 31, 8, 2, 128)])
def test_shares_of_short_sequences(mi, dev, bits, kv, nH, nKV, d):
    """Far shorter than the host said: shares that begin or end before a sequence's first key, and have none."""
    import torch

    b = hold(mi, Batch([1] * len(kv), kv, 16, nH, nKV, d, seed=len(kv), one_each=True), bits)
    ref = b.reference()
    close(*run(mi, b, max_kv_len=1 << 16), ref, max(kv))
    n = mi.paged_attn_quant_workspace_size(nH, nKV, d, len(kv), len(kv), 1, 1 << 16)
    ws = torch.full((n + 16,), 255, dtype=torch.uint8, device="cuda")  # a part that no one wrote would be NaN
    close(*run(mi, b, max_kv_len=1 << 16, workspace=ws[:n]), ref, max(kv))
    assert (ws[n:] == 255).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("most", [0, 1, 3, 10 ** 6])
@pytest.mark.parametrize("nH,nKV,d", [(8, 2, 128), (4, 4, 64)])
def test_bounds_only_shape_the_launch(mi, dev, bits, most, nH, nKV, d):
    b = hold(mi, Batch([5, 300, 0, 1], [5, 700, 40, 1500], 16, nH, nKV, d, seed=most % 97), bits)
    close(*run(mi, b, max_q_len=most, max_kv_len=most), b.reference(), 1500)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("d", [64, 128])
def test_long_page_tables(mi, dev, bits, d):
    """More pages in a workgroup's keys than it looks up at a time (pages of one token)."""
    b = hold(mi, Batch([1, 1, 1], [5000, 1, 2999], 1, 2, 1, d, seed=d, one_each=True), bits)
    ref = b.reference()
    close(*run(mi, b), ref, 5000)
    close(*run(mi, b, workspace=None), ref, 5000)
    close(*run(mi, b, max_kv_len=1), ref, 5000)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([200, 1, 70, 0, 33, 16], [700, 90, 130, 40, 33, 1500], 8, 2, 128),
                                           ([1] * 4, [4096, 3, 64, 1000], 4, 2, 64), ([300], [4096], 12, 12, 64),
                                           ([4, 2, 3], [900, 2, 2500], 12, 12, 64)])
def test_weights_are_not_rounded_once(mi, dev, bits, q, kv, nH, nKV, d):
    """Weights that all round one way in bf16 (the scores' numbers are some that the cache holds)."""
    import test_paged_weights_gpu as w

    b = one_way_batch(q, kv, 16, nH, nKV, d, seed=7)
    hold(mi, b, bits)
    # q 0 = 1 and a held score of 0: scores and signs are put into q instead, which bf16 holds
    for s, n in enumerate(kv):
        k = w.one_way(n, d)[0]
        x = np.where(k[:, :1] == 0, 0.0, 1.0) * np.where(k[:, :1] == w.UP, [1.0, 0.0], [0.0, 1.0])
        kk = np.zeros((nKV, n, d))
        kk[:, :, :2] = x
        b.hk[s] = kk
    b.q[:, :, 0], b.q[:, :, 1] = w.UP, w.DOWN
    hold(mi, b, bits)
    close(*run(mi, b, scale=1.0), b.reference(scale=1.0), max(kv))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([1, 1], [700, 33], 8, 2, 128), ([150, 3], [400, 90], 4, 4, 96)])
def test_groups_of_unlike_size(mi, dev, bits, q, kv, nH, nKV, d):
    """Powers of two from 2^-40 to 1 side by side: each group is multiplied by its own."""
    b = hold(mi, Batch(q, kv, 16, nH, nKV, d, seed=5), bits, spread=40)
    close(*run(mi, b), b.reference(), max(kv))


@pytest.mark.parametrize("bits", [8, 4])
def test_scale_and_large_scores(mi, dev, bits):
    b = hold(mi, Batch([3, 1], [50, 200], 16, 4, 2, 64, seed=9), bits)
    close(*run(mi, b, scale=0.02), b.reference(scale=0.02), 200)
    b.q *= 64  # scores of hundreds: one key takes almost all, and the running maximum moves far
    o, A, lse = b.reference()
    got, l = run(mi, b)
    # a score is off by up to 64 * 2^-24 * 64 * 16 and p by as much, 2^-8
    tol = bound(o, A, 200) + 2.0 ** -8 * 2 * A
    assert (np.abs(got.double().cpu().numpy() - o) <= tol).all()
    assert np.allclose(l.double().cpu().numpy(), lse, rtol=2.0 ** -20, atol=2.0 ** -8)


@pytest.mark.parametrize("bits", [8, 4])
def test_rows_without_keys_and_rows_behind(mi, dev, bits):
    import torch

    b = hold(mi, Batch([2, 4, 1, 3], [0, 1, 0, 30], 16, 4, 2, 64, seed=2, tail_rows=5), bits)
    ref = b.reference()
    lse = torch.full((b.rows, 4), 7.0, device="cuda")
    out = torch.full((b.rows, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    mi.paged_attn_quant(b.q, b.c, b.pages, b.kv_len, q_start=b.q_start, max_q_len=4, max_kv_len=30, out=out, lse=lse)
    n = sum(b.q_len)
    close(out[:n], lse[:n], tuple(t[:n] for t in ref), 30)
    assert (out[n:] == 3.0).all() and (lse[n:] == 7.0).all()
    assert (out[:2] == 0).all() and torch.isneginf(lse[:2]).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_bad_pages_are_not_seen(mi, dev, bits):
    import torch

    b = hold(mi, Batch([1, 2, 40], [112, 64, 90], 16, 4, 2, 64, seed=4), bits)
    table = b.table.copy()
    table[0, 2], table[1, 0], table[2, 5] = b.num_pages, -7, 2 ** 31 - 1
    b.pages.copy_(torch.tensor(table))
    gone = {0: 2, 1: 0, 2: 5}
    close(*run(mi, b), b.reference(seen=lambda s, keys: keys // 16 != gone[s]), 112)
    b.kv_len[0] += 1000  # longer than the table: the keys it names are all there is
    b.pages[0].copy_(torch.tensor(b.table[0]))
    got, lse = run(mi, b, max_q_len=40, max_kv_len=112)
    close(got[:1], lse[:1], tuple(t[:1] for t in b.reference()), 112)


@pytest.mark.parametrize("bits", [8, 4])
def test_strides_and_in_place(mi, dev, bits):
    import torch

    b = hold(mi, Batch([7, 1, 20], [7, 40, 77], 16, 4, 2, 64, seed=6), bits)
    ref = b.reference()
    wide = torch.full((b.rows, 4 + 4, 72), float("nan"), dtype=torch.bfloat16, device="cuda")
    q = wide[:, 2:6, :64]
    q.copy_(b.q)
    lse = torch.empty((b.rows, 4), device="cuda")
    out = torch.empty((4, b.rows, 64), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    how = dict(q_start=b.q_start, max_q_len=20, lse=lse)
    mi.paged_attn_quant(q, b.c, b.pages, b.kv_len, out=out, **how)
    close(out, lse, ref, 77)
    mi.paged_attn_quant(q, b.c, b.pages, b.kv_len, out=q, **how)
    close(q, lse, ref, 77)
    assert torch.isnan(wide[:, :2]).all() and torch.isnan(wide[:, 6:]).all() and torch.isnan(wide[:, :, 64:]).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_offsets_past_32_bits(mi, dev, bits):
    import torch

    b = hold(mi, Batch([1, 30], [70, 45], 16, 4, 2, 64, seed=8), bits)
    stride, top, n = 1 << 27, 40, b.num_pages
    big = torch.empty((top * stride,), dtype=torch.uint8, device="cuda")
    c = []
    for i, t in enumerate(b.c):
        w = t.shape[3]
        x = torch.as_strided(big, (top, 2, 16, w), (stride, 16 * w, w, 1), i << 20)
        x[top - n:] = t
        c.append(x)
    b.c = mi.QuantCache(*c)
    b.pages = torch.where(b.pages >= 0, b.pages + top - n, b.pages)
    close(*run(mi, b), b.reference(), 70)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q,kv", [([1, 1, 1], [100, 64, 2000]), ([40, 150, 2], [100, 200, 2000])])
def test_groups_of_nan(mi, dev, bits, q, kv):
    """A group that reads back as NaN among the last keys that a row sees: of K, the row is NaN; of V, its components."""
    import torch

    b = hold(mi, Batch(q, kv, 16, 4, 2, 64, seed=1), bits)
    last = lambda s: (int(b.table[s, (kv[s] - 1) // 16]), (kv[s] - 1) % 16)  # noqa: E731
    want, _ = run(mi, b)
    page, slot = last(0)
    b.c.k_scale[page, 1, slot, 0] = 255
    page, slot = last(1)
    b.c.v_scale[page, 0, slot, 1] = 255
    got, lse = run(mi, b)
    rows = [int(b.starts[s + 1]) - 1 for s in range(3)]
    assert torch.isnan(got[rows[0], 2:]).all() and torch.isnan(lse[rows[0], 2:]).all()
    assert torch.equal(got[rows[0], :2], want[rows[0], :2])
    assert torch.isnan(got[rows[1], :2, 32:]).all()
    assert torch.equal(got[rows[1], :2, :32], want[rows[1], :2, :32]) and torch.equal(got[rows[1], 2:], want[rows[1], 2:])
    assert torch.equal(got[b.starts[2]:], want[b.starts[2]:])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([1] * 5, [900, 1, 2000, 64, 33], 16, 4, 128), ([300, 1, 7], [700, 90, 1000], 12, 12, 64),
                                           ([64, 64], [64, 3000], 8, 1, 96)])
def test_as_over_the_values_in_bf16(mi, dev, bits, q, kv, nH, nKV, d):
    """Against mi_paged_attn over a cache of the values read back: both are within E of one value before their own
    rounding."""
    import torch

    b = hold(mi, Batch(q, kv, 16, nH, nKV, d, seed=2, one_each=max(q) == 1), bits)
    got, lse = run(mi, b)
    S = len(kv)
    start = torch.tensor(np.concatenate([[0], np.cumsum(kv)]), dtype=torch.int32, device="cuda")
    k, v = mi.kv_read_quant(b.c, b.pages, b.kv_len, q_start=start, rows=sum(kv))
    mi.kv_append(k, v, b.k, b.v, b.pages, b.kv_len, q_start=start)
    for s in range(S):
        assert np.array_equal(k[start[s]:start[s + 1]].double().cpu().numpy().transpose(1, 0, 2), b.hk[s])
    lse2 = torch.empty_like(lse)
    want = mi.paged_attn(b.q, b.k, b.v, b.pages, b.kv_len, q_start=b.q_start, max_q_len=max(q), max_kv_len=max(kv), lse=lse2)
    o, A, _ = b.reference()
    assert (np.abs(got.double().cpu().numpy() - want.double().cpu().numpy()) <= 2 * bound(np.abs(o) + A * 2.0 ** -8, A, max(kv))).all()
    assert torch.allclose(lse, lse2, rtol=2.0 ** -21, atol=2.0 ** -10)


@pytest.mark.parametrize("S", [64, 65, 300, 5000])
def test_many_sequences(mi, dev, S):
    r = np.random.default_rng(S)
    q = [int(x) for x in r.integers(0, 3, S)]
    kv = [n + int(x) for n, x in zip(q, r.integers(0, 5, S))]
    b = hold(mi, Batch(q, kv, 4, 2, 1, 32, seed=S), 4)
    close(*run(mi, b), b.reference(), 7)


# ---- together -------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [8, 4])
def test_prompt_then_decode(mi, dev, bits):
    """A prompt enters in two chunks, then tokens one by one, two sequences of unequal length, as a serving loop
    does it; what the chain's reference sees is read back from the cache, whose codes have tests of their own."""
    import torch

    nH, nKV, d, P = 8, 2, 128, 16
    f, _ = mi.rope_frequencies(d)
    c = mi.quant_cache(16, nKV, P, d, bits)
    pages = torch.tensor([[3, 9, 1, 15, 0, 7], [2, 14, 5, 6, 11, 8]], dtype=torch.int32, device="cuda")
    lens, keys = [0, 0], [np.zeros((0, nKV, d))] * 2
    for step, q_len in enumerate([[20, 33], [11, 30], [1, 1], [1, 1], [1, 0], [3, 1]]):
        n = sum(q_len)
        qkv = make((n, nH + 2 * nKV, d), 40 + step)
        q, k, v = qkv.split((nH, nKV, nKV), dim=1)
        lens = [a + m for a, m in zip(lens, q_len)]
        kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        start = torch.tensor(np.concatenate([[0], np.cumsum(q_len)]), dtype=torch.int32, device="cuda")
        how = dict(q_start=None if q_len == [1, 1] else start)
        qr = mi.kv_append_quant(k, v, c, pages, kv_len, q=q, inv_freq=f, sync=False, **how)
        if how["q_start"] is not None:
            how["max_q_len"] = max(q_len)
        lse = torch.empty((n, nH), device="cuda")
        o = mi.paged_attn_quant(qr, c, pages, kv_len, max_kv_len=max(lens), lse=lse, **how)
        whole = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device="cuda")
        rk, rv = mi.kv_read_quant(c, pages, kv_len, q_start=whole, rows=sum(lens))
        b = Batch.__new__(Batch)
        b.q, b.rows, b.nH, b.nKV, b.d, b.q_len, b.kv = qr, n, nH, nKV, d, q_len, lens
        b.starts = np.concatenate([[0], np.cumsum(q_len)])
        cut = [slice(0, lens[0]), slice(lens[0], sum(lens))]
        b.hk, b.hv = ([t[x].double().cpu().numpy().transpose(1, 0, 2) for x in cut] for t in (rk, rv))
        for s in range(2):  # what was there before is there still, and the new values are near their own
            now = b.hv[s].transpose(1, 0, 2)
            assert np.array_equal(now[:len(keys[s])], keys[s])
            keys[s] = now
            new = v[b.starts[s]:b.starts[s + 1]].double().cpu().numpy()
            assert np.array_equal(now[lens[s] - q_len[s]:], values(*quantise(new, bits), bits))
        close(o, lse, b.reference(), max(lens))


@pytest.mark.parametrize("bits", [8, 4])
def test_streams_and_graph(mi, dev, bits):
    import torch

    b = hold(mi, Batch([1] * 6, [100, 3, 2000, 64, 1, 777], 16, 8, 2, 128, seed=1, one_each=True), bits)
    f, _ = mi.rope_frequencies(128)
    qkv = make((6, 12, 128), 3)
    q, k, v = qkv.split((8, 2, 2), dim=1)

    def step(ws="auto"):
        qr = mi.kv_append_quant(k, v, b.c, b.pages, b.kv_len, q=q, inv_freq=f, sync=False)
        o = mi.paged_attn_quant(qr, b.c, b.pages, b.kv_len, max_kv_len=2000, workspace=ws, sync=False)
        return (o,) + mi.kv_read_quant(b.c, b.pages, b.kv_len, sync=False)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    n = mi.paged_attn_quant_workspace_size(8, 2, 128, 6, 6, 1, 2000)
    ws = torch.empty((max(n, 16),), dtype=torch.uint8, device="cuda")
    graphs = []
    for _ in range(2):  # two graphs on one workspace, replayed in turn on one stream
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(ws)
        graphs.append((g, out))
    for seed in (5, 6, 7):
        qkv.copy_(make(qkv.shape, seed))
        b.kv_len.copy_(torch.tensor([90 + seed, 3, 1990 + seed, 64, 1, 770], dtype=torch.int32))
        eager = [t.clone() for t in step()]
        for g, out in graphs:
            for t in out:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q,kv", [([1] * 5, [900, 64, 2000, 3, 33]), ([70, 3, 200], [90, 2500, 700])])
def test_two_streams_at_once(mi, dev, bits, q, kv):
    """Two calls in flight, each with parts of its own, and the same in a graph."""
    import torch

    b = hold(mi, Batch(q, kv, 16, 8, 2, 128, seed=4, one_each=max(q) == 1), bits)
    qs = [b.q, make(b.q.shape, 77)]
    how = dict(q_start=b.q_start, max_kv_len=max(kv), sync=False)
    if b.q_start is not None:
        how["max_q_len"] = max(q)

    def call(x):
        return mi.paged_attn_quant(x, b.c, b.pages, b.kv_len, **how)

    want = [call(x).clone() for x in qs]
    main, streams = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in qs]

    def both():
        main = torch.cuda.current_stream()
        out = []
        for x, s in zip(qs, streams):
            s.wait_stream(main)
            with torch.cuda.stream(s):
                out.append(call(x))
        for s in streams:
            main.wait_stream(s)
        return out

    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(both(), want))
    main.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    for seed in (8, 9):
        for x in qs:
            x.copy_(make(x.shape, seed))
        want = [call(x).clone() for x in qs]
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q,kv", [([1] * 4, [900, 64, 2000, 3]), ([3, 40, 150], [2100, 300, 200])])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_a_query_of_nan_stays_in_its_row(mi, dev, bits, q, kv, what):
    import torch

    b = hold(mi, Batch(q, kv, 16, 4, 2, 64, seed=6, one_each=max(q) == 1), bits)
    want, wl = run(mi, b)
    row = sum(q) // 2
    b.q[row, 1, 5] = what
    got, gl = run(mi, b)
    assert torch.isnan(got[row, 1]).all()
    others = torch.ones(got.shape[:2], dtype=torch.bool, device="cuda")
    others[row, 1] = False
    assert torch.equal(got[others], want[others]) and torch.equal(gl[others], wl[others])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([4, 3], [50, 600], 4, 2, 64), ([16], [16], 1, 1, 32), ([40, 150], [100, 200], 8, 2, 128),
                                           ([300], [2500], 12, 12, 64), ([7], [3000], 4, 4, 96), ([129, 64], [129, 3000], 4, 2, 96),
                                           ([17, 5], [33, 400], 20, 1, 128)])
def test_nan_reaches_no_row_before_its_key(mi, dev, bits, q, kv, nH, nKV, d):
    """Groups of NaN of new tokens: rows before the token are what they were, the others NaN (of V: in the group)."""
    import torch

    b = hold(mi, Batch(q, kv, 16, nH, nKV, d, seed=9), bits)
    ways = [({}, *run(mi, b)), (dict(workspace=None), *run(mi, b, workspace=None))]
    want = ways[0][1]
    for part in ("v", "k"):
        scale = b.c.v_scale if part == "v" else b.c.k_scale
        marks, none = [], torch.zeros_like(want, dtype=torch.bool)
        for s, (n, m) in enumerate(zip(q, kv)):
            for i, j in enumerate(sorted({n // 3, n // 2, n - 1})):
                at = m - n + j
                h, group = i % nKV, (i + s) % (d // 32)
                marks.append((int(b.table[s, at // 16]), h, at % 16, group))
                comps = slice(32 * group, 32 * group + 32) if part == "v" else slice(None)
                none[b.starts[s] + j:b.starts[s + 1], h * (nH // nKV):(h + 1) * (nH // nKV), comps] = True
        was = [int(scale[x]) for x in marks]
        for x in marks:
            scale[x] = 255
        for kw, o, l in ways:
            got, lse = run(mi, b, **kw)
            assert torch.equal(torch.isnan(got), none)
            assert torch.equal(got[~none], o[~none])
            gone = none.any(-1) if part == "k" else torch.zeros_like(none[..., 0])
            assert torch.equal(torch.isnan(lse), gone) and torch.equal(lse[~gone], l[~gone])
        for x, y in zip(marks, was):
            scale[x] = y


@pytest.mark.parametrize("bits", [8, 4])
def test_scales_anywhere_and_padded_codes(mi, dev, bits):
    """Scale bytes at odd addresses with odd strides, codes with gaps: appended to, read back and attended over."""
    import torch

    b = hold(mi, Batch([3, 1, 150], [50, 700, 260], 16, 8, 2, 64, seed=12), bits)
    want, lse = run(mi, b)
    n, kv, P, nb = b.c.k.shape
    c = []
    for t in b.c[:2]:
        x = torch.full((n, kv + 1, P + 1, nb + 16), 255, dtype=torch.uint8, device="cuda")[:, :kv, 1:, 16:]
        c.append(x.copy_(t))
    for t in b.c[2:]:
        x = torch.full((n * (kv * P * 7 + 3) + 9,), 255, dtype=torch.uint8, device="cuda")
        x = x.as_strided(t.shape, (kv * P * 7 + 3, P * 7, 7, 1), 5)
        c.append(x.copy_(t))
    plain, b.c = b.c, mi.QuantCache(*c)
    got, lse2 = run(mi, b)
    assert torch.equal(got, want) and torch.equal(lse, lse2)
    k, v = make((154, 2, 64), 1), make((154, 2, 64), 2)
    for cache in (plain, b.c):
        mi.kv_append_quant(k, v, cache, b.pages, b.kv_len, q_start=b.q_start)
    for x, y in zip(plain, b.c):
        assert torch.equal(x, y)
    for x, y in zip(*(mi.kv_read_quant(cache, b.pages, b.kv_len, q_start=b.q_start, rows=154) for cache in (plain, b.c))):
        assert torch.equal(x, y)


def test_tables_wider_than_their_pages(mi, dev):
    """Views of a wider page table, and of longer tables of lengths."""
    import torch

    b = hold(mi, Batch([3, 1, 20], [50, 700, 64], 16, 4, 2, 64, seed=8), 4)
    want, lse = run(mi, b)
    wide = torch.full((3, b.pages.shape[1] + 5), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, :b.pages.shape[1]] = b.pages
    b.pages = wide[:, :b.pages.shape[1]]
    b.kv_len = torch.cat([b.kv_len, b.kv_len])[:3]
    got, lse2 = run(mi, b)
    assert torch.equal(got, want) and torch.equal(lse, lse2)


def test_empty_calls(mi, dev):
    import torch

    c = mi.quant_cache(4, 1, 16, 64, 4)
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    pages, kv = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.ones((1,), dtype=torch.int32, device="cuda")
    start = torch.zeros((2,), dtype=torch.int32, device="cuda")
    assert mi.paged_attn_quant(none, c, pages, kv, q_start=start, max_q_len=0).shape == (0, 2, 64)
    mi.paged_attn_quant(none, c, pages[:0], kv[:0], q_start=start[:1], max_q_len=1)
