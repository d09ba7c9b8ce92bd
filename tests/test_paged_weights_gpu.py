"""How exactly mi_paged_attn carries the softmax weights into their product with V, in every kernel.

The weights enter as the sum of two bf16: rounding twice leaves 2^-16 of each. A score is off by
at most d * 2^-24 * scale * sum |q k|, below 2^-13 at these sizes (d <= 128, sum |q k| * scale <= 16), and moves the
weights above and below the division by as much, 2^-12 together; sums of n terms, above and below
too, n * 2^-23; exponentials, the division and the joins stay below 2^-16. So an output before its own
rounding is off by at most E = (2^-12 + n * 2^-23 + 2^-15) A, A = sum p |v|, and after it by 2^-8 |o| more. A
weight rounded to bf16 once is off by up to 2^-8 of itself. Random weights hide that: they round both
ways. `one_way` has keys whose weights round up by 0.92 * 2^-8 with V = +1 and others whose weights round
down by 0.96 * 2^-8 with V = -1, so that the output is nearly 0 and every rounding counts.
"""
import numpy as np
import pytest
from test_paged_gpu import Batch, make, run

UP, DOWN = -1.3515625, -1.359375  # scores (bf16 numbers) whose exponentials round up and down


def one_way(n, d):
    """k, v [n, d] of a head, to go with a query of 1, 0, 0 ... and scale 1: in every 32 keys two of the largest
    score, which weigh 1 and hold no V, so that all blocks share one maximum, and 15 of each kind."""
    i = np.arange(n)
    score = np.where(i % 32 < 2, 0.0, np.where(i % 2 == 0, UP, DOWN))
    sign = np.where(i % 32 < 2, 0.0, np.where(i % 2 == 0, 1.0, -1.0))
    k = np.zeros((n, d))
    k[:, 0] = score
    return k, sign[:, None] * np.where(np.arange(d) % 2 == 0, 1.0, -1.0)


def bound(o, A, n):
    return 2.0 ** -8 * np.abs(o) + (1 + 2.0 ** -8) * (2.0 ** -12 + n * 2.0 ** -23 + 2.0 ** -15) * A


def close(got, lse, ref, n):
    o, A, want = ref
    got, lse = got.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - o) - bound(o, A, n)
    assert (over <= 0).all(), (float(over.max()), np.argwhere(over > 0)[:5])
    none = np.isneginf(want)
    assert np.array_equal(np.isneginf(lse), none)
    assert (np.abs(lse[~none] - want[~none]) <= 2.0 ** -11 + 2.0 ** -22 * np.abs(want[~none])).all()


def one_way_batch(*args, **kw):
    import torch

    b = Batch(*args, **kw)
    b.q.zero_()
    b.q[:, :, 0] = 1.0
    for s, n in enumerate(b.kv):
        k, v = one_way(n, b.d)
        b.hk[s], b.hv[s] = np.broadcast_to(k, (b.nKV, n, b.d)), np.broadcast_to(v, (b.nKV, n, b.d))
        for i in range(-(-n // b.P)):
            m = min(b.P, n - i * b.P)
            for cache, rows in ((b.k, k), (b.v, v)):
                cache[int(b.table[s, i]), :, :m] = torch.tensor(rows[i * b.P:i * b.P + m]).to(cache)
    return b


# ---- without a GPU: what the bound can tell apart --------------------------------------------

def test_the_bound_tells_one_rounding_from_two():
    import torch

    def bf16(x):
        return torch.tensor(x, dtype=torch.float32).to(torch.bfloat16).double().numpy()

    for n in (70, 1000, 4096):
        k, v = one_way(n, 8)
        e = np.exp(k[:, 0])
        o, A = e @ v / e.sum(), e @ np.abs(v) / e.sum()
        once = bf16(e)
        twice = once + bf16(e - once)
        assert (np.abs(twice @ v / e.sum() - o) <= bound(o, A, n)).all()
        assert (np.abs(once @ v / e.sum() - o) > 3 * bound(o, A, n)).all()
        assert (np.abs((once - bf16(e - once)) @ v / e.sum() - o) > 3 * bound(o, A, n)).all()  # the rest's sign


# ---- on the GPU ----------------------------------------------------------------------------------

HEADS = [(4, 4, 64), (8, 2, 128), (8, 1, 96), (6, 2, 40), (16, 4, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("nH,nKV,d", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_weights_of_many_rows(mi, dev, nH, nKV, d, causal):
    """Tiles of many rows, of few, and decode rows between them."""
    b = one_way_batch([200, 1, 70, 0, 33, 16], [700, 90, 130, 40, 33, 1500], 16, nH, nKV, d, seed=d)
    close(*run(mi, b, causal=causal, scale=1.0), b.reference(causal, scale=1.0), 1500)


@pytest.mark.gpu
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([1024], [1024], 16, 4, 128), ([130, 300], [4000, 2100], 4, 2, 128),
                                           ([300], [4096], 12, 12, 64)])
def test_weights_of_split_chunks(mi, dev, q, kv, nH, nKV, d):
    b = one_way_batch(q, kv, 64, nH, nKV, d, seed=7)
    ref = b.reference(scale=1.0)
    close(*run(mi, b, scale=1.0), ref, max(kv))
    close(*run(mi, b, scale=1.0, workspace=None), ref, max(kv))


@pytest.mark.gpu
@pytest.mark.parametrize("nH,nKV,d", HEADS)
@pytest.mark.parametrize("P", [1, 16, 64])
def test_weights_of_decode_rows(mi, dev, nH, nKV, d, P):
    b = one_way_batch([1] * 8, [1, 2, 63, 64, 65, 300, 129, 31], P, nH, nKV, d, seed=P, one_each=True)
    close(*run(mi, b, scale=1.0), b.reference(scale=1.0), 300)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,nH,nKV,d", [([4096], 8, 2, 128), ([4001], 4, 1, 64), ([3, 2500] + [40] * 138, 4, 2, 64),
                                         ([2048, 0, 1800, 7] * 25, 8, 4, 128)])
def test_weights_of_split_and_shared_decode(mi, dev, kv, nH, nKV, d):
    b = one_way_batch([1] * len(kv), kv, 16, nH, nKV, d, seed=3, one_each=True)
    ref = b.reference(scale=1.0)
    close(*run(mi, b, scale=1.0), ref, max(kv))
    close(*run(mi, b, scale=1.0, workspace=None), ref, max(kv))


@pytest.mark.gpu
@pytest.mark.parametrize("nH,nKV,d,P,kv", [
    (8, 2, 128, 16, [1, 2, 63, 64, 65, 300, 129, 31]), (3, 1, 8, 256, [700, 1]), (6, 2, 40, 1, [5, 1000, 64]),
    (8, 2, 128, 16, [4096]), (8, 2, 64, 16, [1023]), (2, 1, 64, 1, [4000, 1, 2999])])
def test_random_decode(mi, dev, nH, nKV, d, P, kv):
    b = Batch([1] * len(kv), kv, P, nH, nKV, d, seed=P + d, one_each=True)
    close(*run(mi, b), b.reference(), max(kv))


@pytest.mark.gpu
@pytest.mark.parametrize("S,nH,nKV,d,P", [(140, 4, 2, 64, 16), (70, 8, 4, 128, 1), (300, 1, 1, 40, 64)])
def test_random_shared_decode(mi, dev, S, nH, nKV, d, P):
    r = np.random.default_rng(S + 1)
    kv = [int(x) for x in np.exp(r.uniform(0, np.log(1500), S))]
    kv[0], kv[S // 2], kv[S - 1], kv[3] = 2500, 2100, 0, 0
    b = Batch([1] * S, kv, P, nH, nKV, d, seed=S, one_each=True)
    close(*run(mi, b), b.reference(), 2500)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,nKV,d", [([140000, 5], 1, 128), ([7, 66000], 2, 40)])
def test_random_decode_of_hundreds_of_shares(mi, dev, kv, nKV, d):
    """A share sums a thousand keys at most and the join as many parts: n = 2^11 of the bound."""
    b = Batch([1, 1], kv, 64, 2, nKV, d, seed=d, one_each=True)
    close(*run(mi, b), b.reference(), 2 ** 11)


@pytest.mark.gpu
@pytest.mark.parametrize("q,kv,nH,nKV,d", [([200], [1000], 8, 2, 128), ([129, 1, 64], [400, 700, 64], 4, 4, 64),
                                           ([33, 40], [700, 2048], 1, 1, 72), ([257], [257], 4, 1, 96)])
def test_random_chunks(mi, dev, q, kv, nH, nKV, d):
    b = Batch(q, kv, 32, nH, nKV, d, seed=5)
    close(*run(mi, b), b.reference(), max(kv))


@pytest.mark.gpu
@pytest.mark.parametrize("n,nH,nKV,d", [(1000, 8, 2, 128), (333, 4, 4, 64)])
def test_a_token_alone_and_in_a_chunk(mi, dev, n, nH, nKV, d):
    """The last rows of a prompt in chunks of other sizes, and by themselves: each is within E and its own
    rounding of one value, so two of them differ by twice that at most."""
    import torch

    b = Batch([n], [n], 16, nH, nKV, d, seed=11)
    o, A, _ = b.reference()
    whole, _ = run(mi, b)
    whole = whole.double().cpu().numpy()
    for size in (1, 3, 4, 40, 129):
        last = b.q[n - size:].contiguous()
        start = torch.tensor([0, size], dtype=torch.int32, device="cuda")
        got = mi.paged_attn(last, b.k, b.v, b.pages, b.kv_len, q_start=start, max_q_len=size, max_kv_len=n)
        got = got.double().cpu().numpy()
        tol = 2 * bound(np.abs(o[n - size:]) + A[n - size:] * 2.0 ** -8, A[n - size:], n)
        assert (np.abs(got - whole[n - size:]) <= tol).all(), size
