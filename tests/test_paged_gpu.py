"""The paged cache: append (mi_kv_append) and attention (mi_paged_attn) against 64-bit formulas.

Tolerances. Attention takes bf16 q, k, v as they are and accumulates in fp32. Probabilities are
rounded to bf16 before the product with V, 2^-8 of each, so the output is off by at most 2^-8 of
A = sum p |v|; its own rounding adds 2^-8 of |o|. A score is a sum of d products, off by at most
d * 2^-24 * scale * sum |q k|, below 2^-13 at these sizes (d <= 128, sum |q k| * scale <= 16), and moves
p by as much; exponentials, the running sum and its joins add n * 2^-24 at n keys (n <= 2^12): together
under 2^-11 of A. lse: the same absolute 2^-11 at most from the sum and the scores. Rotated rows as in
the tests of mi_rope.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def make(shape, seed, std=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)


class Batch:
    """Sequences with new rows and cached keys; every slot that holds no key is NaN."""

    def __init__(self, q_len, kv_len, P, nH, nKV, d, seed=0, order="phsd", spare=3, tail_rows=0, one_each=False):
        import torch

        r = np.random.default_rng(seed)
        S = len(q_len)
        self.q_len, self.kv, self.P, self.nH, self.nKV, self.d = q_len, kv_len, P, nH, nKV, d
        need = [-(-n // P) for n in kv_len]
        width = max(need + [1]) + 1
        self.num_pages = sum(need) + spare
        ids = r.permutation(self.num_pages)
        self.table = np.full((S, width), -1, np.int64)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + n]
            at += n
        shape = (self.num_pages, nKV, P, d) if order == "phsd" else (self.num_pages, P, nKV, d)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=torch.bfloat16, device="cuda") for _ in "kv")
        if order == "pshd":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.hk, self.hv = [], []
        for s, n in enumerate(kv_len):
            kk, vv = make((nKV, n, d), seed * 100 + 2 * s + 1), make((nKV, n, d), seed * 100 + 2 * s + 2)
            for i in range(need[s]):
                m = min(P, n - i * P)
                self.k[int(self.table[s, i]), :, :m] = kk[:, i * P:i * P + m]
                self.v[int(self.table[s, i]), :, :m] = vv[:, i * P:i * P + m]
            self.hk.append(kk.double().cpu().numpy())
            self.hv.append(vv.double().cpu().numpy())
        self.rows = sum(q_len) + tail_rows
        self.q = make((self.rows, nH, d), seed + 5000)
        self.pages = torch.tensor(self.table, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
        self.starts = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int64)
        self.q_start = None if one_each else torch.tensor(self.starts, dtype=torch.int32, device="cuda")

    def args(self):
        return self.q, self.k, self.v, self.pages, self.kv_len

    def reference(self, causal=True, scale=None, seen=None):
        """(o, A, lse) float64; seen(s, key indices) -> bool drops keys."""
        nH, d = self.nH, self.d
        g = nH // self.nKV
        scale = scale or 1.0 / np.sqrt(d)
        q = self.q.double().cpu().numpy()
        o, A, lse = np.zeros((self.rows, nH, d)), np.zeros((self.rows, nH, d)), np.full((self.rows, nH), -np.inf)
        for s, (n, m) in enumerate(zip(self.q_len, self.kv)):
            for j in range(n):
                row, pos = self.starts[s] + j, m - n + j
                keys = np.arange(max(0, min(m, pos + 1) if causal else m))
                if seen is not None:
                    keys = keys[seen(s, keys)]
                if not keys.size:
                    continue
                for h in range(nH):
                    x = self.hk[s][h // g][keys] @ q[row, h] * scale
                    mx = x.max()
                    e = np.exp(x - mx)
                    lse[row, h] = mx + np.log(e.sum())
                    v = self.hv[s][h // g][keys]
                    o[row, h], A[row, h] = e @ v / e.sum(), e @ np.abs(v) / e.sum()
        return o, A, lse


def check(got, lse, ref):
    o, A, want = ref
    got, lse = got.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(got).all()
    tol = 2.0 ** -8 * (np.abs(o) + A) + 2.0 ** -11 * A
    err = np.abs(got - o)
    assert (err <= tol).all(), (float((err - tol).max()), np.argwhere(err > tol)[:5])
    none = np.isneginf(want)
    assert np.array_equal(np.isneginf(lse), none)
    assert (np.abs(lse[~none] - want[~none]) <= 2.0 ** -11 + 2.0 ** -22 * np.abs(want[~none])).all()


def run(mi, b, **kw):
    import torch

    lse = torch.full((b.rows, b.nH), 7.0, dtype=torch.float32, device="cuda")
    kw.setdefault("max_q_len", max(b.q_len + [1]))
    kw.setdefault("max_kv_len", max(b.kv + [1]))
    if b.q_start is None:
        kw.pop("max_q_len")
    return mi.paged_attn(*b.args(), q_start=b.q_start, lse=lse, **kw), lse


HEADS = [(4, 4, 64), (8, 2, 128), (8, 1, 96), (6, 2, 40), (3, 1, 8), (16, 4, 128)]


@pytest.mark.parametrize("nH,nKV,d", HEADS)
@pytest.mark.parametrize("P", [1, 16, 64, 256])
def test_decode(mi, dev, nH, nKV, d, P):
    import torch

    kv = [1, 2, 63, 64, 65, 300, 129, 31]
    b = Batch([1] * len(kv), kv, P, nH, nKV, d, seed=P + d, one_each=True)
    check(*run(mi, b), b.reference())
    b.q_start = torch.arange(len(kv) + 1, dtype=torch.int32, device="cuda")
    check(*run(mi, b), b.reference())


@pytest.mark.parametrize("nH,nKV,d", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(mi, dev, nH, nKV, d, causal):
    b = Batch([5, 1, 70, 0, 33, 16, 2], [5, 90, 130, 40, 33, 17, 0 + 2], 16, nH, nKV, d, seed=d + nH)
    check(*run(mi, b, causal=causal), b.reference(causal))


@pytest.mark.parametrize("order", ["phsd", "pshd"])
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([200], [1000], 8, 2, 128), ([129, 1, 64], [400, 700, 64], 4, 4, 64),
                                           ([257], [257], 4, 1, 128), ([40, 3], [2600, 1900], 4, 2, 128),
                                           ([33, 40], [700, 2048], 1, 1, 72)])
def test_long_chunks(mi, dev, order, q, kv, nH, nKV, d):
    b = Batch(q, kv, 32, nH, nKV, d, seed=3, order=order)
    check(*run(mi, b), b.reference())


@pytest.mark.parametrize("n", [1, 500, 1023, 4096])
@pytest.mark.parametrize("d", [64, 128])
def test_long_context_split(mi, dev, n, d):
    """One sequence over many workgroups, with all, less and no workspace: the joins change roundings only."""
    import torch

    b = Batch([1], [n], 16, 8, 2, d, seed=n, one_each=True)
    ref = b.reference()
    full = mi.paged_attn_workspace_size(8, 2, d, 1, 1, 1, n)
    for ws in ("auto", None, torch.empty((max(full // 2 // 16 * 16, 16),), dtype=torch.uint8, device="cuda"),
               torch.empty((16,), dtype=torch.uint8, device="cuda")):
        check(*run(mi, b, workspace=ws), ref)
    check(*run(mi, b, max_kv_len=1), ref)        # a sequence longer than the host said
    check(*run(mi, b, max_kv_len=1 << 20), ref)  # and one far shorter
    a, c = run(mi, b), run(mi, b)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("S,nH,nKV,d,P", [(140, 4, 2, 64, 16), (70, 8, 4, 128, 1), (300, 1, 1, 40, 64), (1024, 2, 1, 8, 32)])
def test_decode_many_uneven(mi, dev, S, nH, nKV, d, P):
    """Sequences of very unequal length, some without a key, whose keys the workgroups share evenly; a row
    that is cut is joined from its shares, and a share may run over many sequences."""
    import torch

    r = np.random.default_rng(S)
    kv = [int(x) for x in np.exp(r.uniform(0, np.log(1500), S))]
    kv[0], kv[S // 2], kv[S - 1], kv[3] = 2500, 2100, 0, 0
    b = Batch([1] * S, kv, P, nH, nKV, d, seed=S, one_each=True)
    ref = b.reference()
    check(*run(mi, b), ref)
    n = mi.paged_attn_workspace_size(nH, nKV, d, S, S, 1, max(kv))
    ws = torch.full((n + 16,), 255, dtype=torch.uint8, device="cuda")
    check(*run(mi, b, workspace=ws[:n]), ref)
    assert (ws[n:] == 255).all()
    check(*run(mi, b, workspace=ws[:n // 2 // 16 * 16]), ref)
    a, c = run(mi, b), run(mi, b)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("kv,nKV,d", [([140000, 5], 1, 128), ([140001, 140000], 1, 64), ([7, 66000], 2, 40)])
def test_one_sequence_cut_by_all_workgroups(mi, dev, kv, nKV, d):
    """Few KV heads and two sequences, one of which holds most keys: its row is joined from several hundred
    shares. A share sums a thousand keys at most and the join as many parts, 2^11 * 2^-24 together."""
    b = Batch([1, 1], kv, 64, 2, nKV, d, seed=d, one_each=True)
    ref = b.reference()
    check(*run(mi, b), ref)


@pytest.mark.parametrize("most", [0, 1, 3, 10 ** 6])
@pytest.mark.parametrize("nH,nKV,d", [(8, 2, 128), (4, 4, 64)])
def test_bounds_only_shape_the_launch(mi, dev, most, nH, nKV, d):
    b = Batch([5, 300, 0, 1], [5, 700, 40, 1500], 16, nH, nKV, d, seed=most % 97)
    check(*run(mi, b, max_q_len=most, max_kv_len=most), b.reference())


@pytest.mark.parametrize("d", [64, 128])
def test_long_page_tables(mi, dev, d):
    """More pages in a workgroup's keys than it looks up at a time (pages of one token)."""
    b = Batch([1, 1, 1], [5000, 1, 2999], 1, 2, 1, d, seed=d, one_each=True)
    ref = b.reference()
    check(*run(mi, b), ref)
    check(*run(mi, b, workspace=None), ref)
    check(*run(mi, b, max_kv_len=1), ref)


def test_scale_and_large_scores(mi, dev):
    b = Batch([3, 1], [50, 200], 16, 4, 2, 64, seed=9)
    check(*run(mi, b, scale=0.02), b.reference(scale=0.02))
    b.q *= 64  # scores of hundreds: one key takes almost all, and the running maximum moves far
    o, A, lse = b.reference()
    got, l = run(mi, b)
    # a score is off by up to 64 * 2^-24 * 64 * 16 and p by as much, 2^-8 in place of 2^-13
    tol = 2.0 ** -8 * (np.abs(o) + 2 * A) + 2.0 ** -11 * A
    assert (np.abs(got.double().cpu().numpy() - o) <= tol).all()
    assert np.allclose(l.double().cpu().numpy(), lse, rtol=2.0 ** -20, atol=2.0 ** -8)


def test_rows_without_keys_and_rows_behind(mi, dev):
    import torch

    # an empty cache, more new rows than tokens (the first of them at negative positions), rows behind
    b = Batch([2, 4, 1, 3], [0, 1, 0, 30], 16, 4, 2, 64, seed=2, tail_rows=5)
    ref = b.reference()
    lse = torch.full((b.rows, 4), 7.0, device="cuda")
    out = torch.full((b.rows, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    mi.paged_attn(*b.args(), q_start=b.q_start, max_q_len=4, max_kv_len=30, out=out, lse=lse)
    n = sum(b.q_len)
    check(out[:n], lse[:n], tuple(t[:n] for t in ref))
    assert (out[n:] == 3.0).all() and (lse[n:] == 7.0).all()
    assert (out[:2] == 0).all() and torch.isneginf(lse[:2]).all()


def test_bad_pages_are_not_seen(mi, dev):
    """Pages outside the cache, and places past the table, hold no keys."""
    import torch

    b = Batch([1, 2, 40], [112, 64, 90], 16, 4, 2, 64, seed=4)
    table = b.table.copy()
    table[0, 2], table[1, 0], table[2, 5] = b.num_pages, -7, 2 ** 31 - 1
    b.pages.copy_(torch.tensor(table))
    gone = {0: 2, 1: 0, 2: 5}
    ref = b.reference(seen=lambda s, keys: keys // 16 != gone[s])
    check(*run(mi, b), ref)
    b.kv_len[0] += 1000  # longer than the table: the keys it names are all there is
    b.pages[0].copy_(torch.tensor(b.table[0]))
    lse = torch.empty((b.rows, 4), device="cuda")
    got = mi.paged_attn(*b.args(), q_start=b.q_start, max_q_len=40, max_kv_len=112, lse=lse)
    check(got[:1], lse[:1], tuple(t[:1] for t in b.reference()))  # the new row sees all of them: causal or not


def test_strides_and_in_place(mi, dev):
    import torch

    b = Batch([7, 1, 20], [7, 40, 77], 16, 4, 2, 64, seed=6)
    ref = b.reference()
    wide = torch.full((b.rows, 4 + 4, 72), float("nan"), dtype=torch.bfloat16, device="cuda")
    q = wide[:, 2:6, :64]
    q.copy_(b.q)
    lse = torch.empty((b.rows, 4), device="cuda")
    out = torch.empty((4, b.rows, 64), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    mi.paged_attn(q, *b.args()[1:], q_start=b.q_start, max_q_len=20, out=out, lse=lse)
    check(out, lse, ref)
    mi.paged_attn(q, *b.args()[1:], q_start=b.q_start, max_q_len=20, out=q, lse=lse)
    check(q, lse, ref)
    assert torch.isnan(wide[:, :2]).all() and torch.isnan(wide[:, 6:]).all() and torch.isnan(wide[:, :, 64:]).all()


def test_offsets_past_32_bits(mi, dev):
    """A cache of 2.5 * 2^31 elements, of which the sequences use pages at its far end."""
    import torch

    b = Batch([1, 30], [70, 45], 16, 4, 2, 64, seed=8)
    stride = 1 << 27
    n = b.num_pages
    top = 40
    big = torch.empty((top * stride,), dtype=torch.bfloat16, device="cuda")
    k = torch.as_strided(big, (top, 2, 16, 64), (stride, 1024, 64, 1))
    v = torch.as_strided(big, (top, 2, 16, 64), (stride, 1024, 64, 1), 1 << 20)
    k[top - n:] = b.k
    v[top - n:] = b.v
    pages = torch.where(b.pages >= 0, b.pages + top - n, b.pages)
    lse = torch.empty((b.rows, 4), device="cuda")
    got = mi.paged_attn(b.q, k, v, pages, b.kv_len, q_start=b.q_start, max_q_len=30, max_kv_len=70, lse=lse)
    check(got, lse, b.reference())
    # and the append writes there: the last token of each sequence again, with other values
    kk, vv = make((31, 2, 64), 1), make((31, 2, 64), 2)
    mi.kv_append(kk, vv, k, v, pages, b.kv_len, q_start=b.q_start)
    for s, (m, r) in enumerate(((70, 0), (45, 30))):
        page, slot = int(pages[s, (m - 1) // 16]), (m - 1) % 16
        assert page * stride > 1 << 31
        assert torch.equal(k[page, :, slot], kk[r]) and torch.equal(v[page, :, slot], vv[r])


# ---- append -------------------------------------------------------------------------

def rotated(x, pos, f, interleaved, scale):
    from test_rope_gpu import reference

    y, size = reference(x[None], np.asarray(pos)[None], f, interleaved, scale)
    return y[0], size[0]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("order", ["phsd", "pshd"])
@pytest.mark.parametrize("nH,nKV,d,rot,q_len,kv_len,P", [
    (4, 2, 64, 64, [1, 1, 1], [1, 17, 100], 16), (8, 2, 128, 64, [5, 0, 40, 1], [9, 3, 40, 64], 32),
    (2, 1, 40, 8, [130, 3], [131, 3], 1), (3, 3, 8, 2, [2], [2], 64)])
def test_append(mi, dev, interleaved, order, nH, nKV, d, rot, q_len, kv_len, P):
    import torch
    from test_rope_gpu import check as rope_check

    b = Batch(q_len, kv_len, P, nH, nKV, d, seed=1, order=order, tail_rows=4)
    f, _ = mi.rope_frequencies(rot)
    qkv = make((b.rows, nH + 2 * nKV, d), 77)
    q, k, v = qkv.split((nH, nKV, nKV), dim=1)
    before_k, before_v = b.k.clone(), b.v.clone()
    q_out = torch.full((b.rows, nH, d), 5.0, dtype=torch.bfloat16, device="cuda")
    got = mi.kv_append(k, v, b.k, b.v, b.pages, b.kv_len, q_start=b.q_start, q=q, q_out=q_out, inv_freq=f,
                       interleaved=interleaved, scale=1.5)
    assert got is q_out
    n = sum(q_len)
    assert (q_out[n:] == 5.0).all()
    fh = f.cpu().numpy()
    seq = np.repeat(np.arange(len(q_len)), q_len)
    pos = np.array([kv_len[s] - q_len[s] + r - b.starts[s] for r, s in enumerate(seq)])
    h = lambda t: t[:n].double().cpu().numpy()  # noqa: E731
    rope_check(h(q_out), *rotated(h(q), pos, fh, interleaved, 1.5), True)
    page = torch.tensor(b.table[seq, pos // P]).cuda()
    slot = torch.tensor(pos % P).cuda()
    rope_check(b.k[page, :, slot].double().cpu().numpy(), *rotated(h(k), pos, fh, interleaved, 1.5), True)
    assert torch.equal(b.v[page, :, slot], v[:n])
    for now, old in ((b.k, before_k), (b.v, before_v)):  # nothing else was written
        now, old = now.clone(), old.clone()
        now[page, :, slot] = 0
        old[page, :, slot] = 0
        assert torch.equal(now.view(torch.int16), old.view(torch.int16))
    # with positions of its own, in place, and without rotation
    own = torch.arange(b.rows, dtype=torch.int32, device="cuda") * 3 + 7
    x = q.clone()
    mi.kv_append(k, v, b.k, b.v, b.pages, b.kv_len, q_start=b.q_start, q=x, q_out=x, inv_freq=f, positions=own,
                 interleaved=interleaved)
    rope_check(h(x), *rotated(h(q), own[:n].cpu().numpy(), fh, interleaved, 1.0), True)
    assert mi.kv_append(k, v, b.k, b.v, b.pages, b.kv_len, q_start=b.q_start) is None
    assert torch.equal(b.k[page, :, slot], k[:n])


def test_append_to_bad_places(mi, dev):
    import torch

    b = Batch([1, 2, 3], [20, 40, 1], 16, 2, 1, 64, seed=1)  # the third: its first two rows before position 0
    b.pages[0, 1] = b.num_pages
    b.pages[1, 2] = -1
    want_k, want_v = b.k.clone(), b.v.clone()
    k, v = make((6, 1, 64), 5), make((6, 1, 64), 6)
    page = int(b.table[2, 0])
    want_k[page, :, 0], want_v[page, :, 0] = k[5], v[5]
    mi.kv_append(k, v, b.k, b.v, b.pages, b.kv_len, q_start=b.q_start)
    assert torch.equal(b.k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(b.v.view(torch.int16), want_v.view(torch.int16))


@pytest.mark.parametrize("S", [64, 65, 300, 5000])
def test_many_sequences(mi, dev, S):
    """The search for a row's sequence over more sequences than a wave has lanes, some without rows."""
    r = np.random.default_rng(S)
    q = [int(x) for x in r.integers(0, 3, S)]
    kv = [n + int(x) for n, x in zip(q, r.integers(0, 5, S))]
    b = Batch(q, kv, 4, 2, 1, 8, seed=S)
    check(*run(mi, b), b.reference())
    import torch

    k, v = make((b.rows, 1, 8), 1), make((b.rows, 1, 8), 2)
    mi.kv_append(k, v, b.k, b.v, b.pages, b.kv_len, q_start=b.q_start)
    seq = np.repeat(np.arange(S), q)
    pos = np.array([kv[s] - q[s] + i - b.starts[s] for i, s in enumerate(seq)])
    page, slot = torch.tensor(b.table[seq, pos // 4]).cuda(), torch.tensor(pos % 4).cuda()
    assert torch.equal(b.k[page, :, slot], k) and torch.equal(b.v[page, :, slot], v)


# ---- together -------------------------------------------------------------------------

def test_prompt_then_decode(mi, dev):
    """A prompt enters in two chunks, then tokens one by one, two sequences of unequal length, as a
    serving loop does it; each step's attention against the 64-bit chain from the same QKV rows. The
    rotated rows are compared where they land, so the chain's reference takes them from the cache."""
    import torch

    nH, nKV, d, P = 8, 2, 128, 16
    f, _ = mi.rope_frequencies(d)
    b = Batch([0, 0], [0, 0], P, nH, nKV, d, seed=1, spare=16)
    pages = torch.tensor([[3, 9, 1, 15, 0, 7], [2, 14, 5, 6, 11, 8]], dtype=torch.int32, device="cuda")
    lens = [0, 0]
    keys, vals = [[], []], [[], []]
    for step, q_len in enumerate([[20, 33], [11, 30], [1, 1], [1, 1], [1, 0], [3, 1]]):
        n = sum(q_len)
        qkv = make((n, nH + 2 * nKV, d), 40 + step)
        q, k, v = qkv.split((nH, nKV, nKV), dim=1)
        lens = [a + c for a, c in zip(lens, q_len)]
        kv_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        start = torch.tensor(np.concatenate([[0], np.cumsum(q_len)]), dtype=torch.int32, device="cuda")
        how = dict(q_start=None if q_len == [1, 1] else start)
        qr = mi.kv_append(k, v, b.k, b.v, pages, kv_len, q=q, inv_freq=f, sync=False, **how)
        if how["q_start"] is not None:
            how["max_q_len"] = max(q_len)
        lse = torch.empty((n, nH), device="cuda")
        o = mi.paged_attn(qr, b.k, b.v, pages, kv_len, max_kv_len=max(lens), lse=lse, **how)
        c = Batch.__new__(Batch)
        c.q, c.rows, c.nH, c.nKV, c.d, c.q_len, c.kv = qr, n, nH, nKV, d, q_len, lens
        c.starts = np.concatenate([[0], np.cumsum(q_len)])
        c.hk, c.hv = [], []
        for s in range(2):
            place = np.arange(lens[s])
            pg, sl = pages[s].cpu().numpy()[place // P], place % P
            got = [t[torch.tensor(pg).long().cuda(), :, torch.tensor(sl).cuda()].double().cpu().numpy().transpose(1, 0, 2)
                   for t in (b.k, b.v)]
            new = slice(c.starts[s], c.starts[s + 1])
            pos = place[lens[s] - q_len[s]:]
            from test_rope_gpu import check as rope_check

            y, size = rotated(k[new].double().cpu().numpy(), pos, f.cpu().numpy(), False, 1.0)
            rope_check(got[0][:, lens[s] - q_len[s]:].transpose(1, 0, 2), y, size, True)
            c.hk.append(got[0])
            c.hv.append(got[1])
        check(o, lse, c.reference())


def test_streams_and_graph(mi, dev):
    import torch

    b = Batch([1] * 6, [100, 3, 2000, 64, 1, 777], 16, 8, 2, 128, seed=1, one_each=True)
    f, _ = mi.rope_frequencies(128)
    qkv = make((6, 12, 128), 3)
    q, k, v = qkv.split((8, 2, 2), dim=1)

    def step(ws="auto"):
        qr = mi.kv_append(k, v, b.k, b.v, b.pages, b.kv_len, q=q, inv_freq=f, sync=False)
        return mi.paged_attn(qr, *b.args()[1:], max_kv_len=2000, workspace=ws, sync=False)

    want = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    n = mi.paged_attn_workspace_size(8, 2, 128, 6, 6, 1, 2000)
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
        eager = step().clone()
        for g, out in graphs:
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


def test_empty_calls(mi, dev):
    import torch

    b = Batch([1], [5], 16, 2, 1, 64, one_each=True)
    none = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    start = torch.zeros((2,), dtype=torch.int32, device="cuda")
    assert mi.paged_attn(none, *b.args()[1:], q_start=start, max_q_len=0).shape == (0, 2, 64)
    mi.kv_append(none[:, :1], none[:, :1], b.k, b.v, b.pages, b.kv_len, q_start=start)
    empty = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    mi.paged_attn(none, b.k, b.v, empty, empty[:, 0].contiguous(), q_start=start[:1], max_q_len=1)
