"""Decode with more heads a KV head than a tile of few rows holds, a few tokens at a time, and captured calls of
the kernel that shares all keys evenly, whose sums of the lengths go through the workspace."""
import numpy as np
import pytest
from test_paged_gpu import Batch, run
from test_paged_weights_gpu import close, one_way_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("make", [Batch, one_way_batch])
@pytest.mark.parametrize("nH,nKV,d", [(16, 1, 128), (17, 1, 64), (32, 1, 128), (64, 2, 64), (48, 1, 40), (130, 1, 128),
                                      (260, 2, 64), (257, 1, 8)])
def test_many_heads_of_a_kv_head(mi, dev, make, nH, nKV, d):
    """One new token for each sequence, with and without q_start: tiles of 16, 32, 128 rows and the ends of such."""
    import torch

    kv = [1, 40, 0, 700, 130, 64, 1300]
    b = make([1] * len(kv), kv, 16, nH, nKV, d, seed=nH, one_each=True)
    how = dict(scale=1.0) if make is one_way_batch else {}
    ref = b.reference(**how)
    first = run(mi, b, **how)
    close(*first, ref, 1300)
    close(*run(mi, b, workspace=None, **how), ref, 1300)
    b.q_start = torch.arange(len(kv) + 1, dtype=torch.int32, device="cuda")
    again = run(mi, b, **how)
    close(*again, ref, 1300)


@pytest.mark.parametrize("nH,nKV,d", [(16, 4, 128), (12, 12, 64), (8, 8, 96), (32, 1, 64)])
@pytest.mark.parametrize("n", [2, 4, 5, 8, 9, 17])
def test_a_few_tokens_at_a_time(mi, dev, nH, nKV, d, n):
    """Speculated tokens: the same few new rows for each sequence."""
    kv = [n, 33 + n, 500, 1100]
    b = Batch([n] * len(kv), kv, 32, nH, nKV, d, seed=n + d)
    close(*run(mi, b), b.reference(), 1100)


def shared(S, nH, nKV, d, longest, seed):
    """A batch that the kernel of even shares takes (its workspace then holds sums of the lengths)."""
    r = np.random.default_rng(seed)
    kv = [int(x) for x in np.exp(r.uniform(0, np.log(1200), S))]
    kv[0] = longest
    return Batch([1] * S, kv, 16, nH, nKV, d, seed=seed, one_each=True)


def test_captured_shares(mi, dev):
    """Two graphs on one workspace, replayed in turn with lengths rewritten between: rows that were cut become
    whole, whole ones are cut, some have no key left, and the sums of one graph lie where the other's lay."""
    import torch

    S, nH, nKV, d, longest = 140, 4, 2, 64, 2500
    b = shared(S, nH, nKV, d, longest, 1)
    r = np.random.default_rng(2)
    b.pages.copy_(torch.tensor(r.integers(0, b.num_pages, b.pages.shape), dtype=torch.int32))  # any page, any row
    b.k.nan_to_num_(0.25)
    b.v.nan_to_num_(0.5)
    n = mi.paged_attn_workspace_size(nH, nKV, d, S, S, 1, longest)
    shares = 3 * torch.cuda.get_device_properties(0).multi_processor_count // nKV
    assert n == 2 * shares * nH * (d + 1) * 4 + (S + 1) * 4  # shares, not pieces
    ws = torch.empty((n,), dtype=torch.uint8, device="cuda")
    other = torch.flip(b.kv_len, (0,)).contiguous()

    def step(lens):
        lse = torch.empty((S, nH), device="cuda")
        return mi.paged_attn(b.q, b.k, b.v, b.pages, lens, max_kv_len=longest, lse=lse, workspace=ws, sync=False), lse

    step(b.kv_len)
    graphs = []
    for lens in (b.kv_len, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(lens)
        graphs.append((g, lens, out))
    full = torch.full((S,), longest, dtype=torch.int32, device="cuda")
    for turn in range(5):
        if turn == 1:  # the long ones short, the short ones long, some empty
            b.kv_len.copy_(torch.tensor([1 if i % 7 == 0 else 0 if i % 7 == 1 else longest for i in range(S)]))
            other.zero_()
            other[S - 1] = longest
        if turn == 2:
            b.kv_len.zero_()
            other.copy_(full)
        if turn == 3:
            b.kv_len.copy_(torch.arange(S, dtype=torch.int32) * 17)
            other.copy_(torch.tensor([longest, 3] * (S // 2)))
        if turn == 4:
            b.kv_len.copy_(full - torch.arange(S, device="cuda", dtype=torch.int32) * 13)
            other.fill_(-1)
        for g, lens, (out, lse) in graphs:
            out.fill_(7.0)
            lse.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            own = mi.paged_attn(b.q, b.k, b.v, b.pages, lens, max_kv_len=longest, sync=False)  # a workspace of its own
            plain = mi.paged_attn(b.q, b.k, b.v, b.pages, lens, max_kv_len=longest, workspace=None)  # no shares at all
            assert torch.equal(out, own)
            # the same sums in another order, each rounded once: two roundings of 2^-8, and E twice
            o, p = out.double(), plain.double()
            size = b.v.double().abs().max()
            assert ((o - p).abs() <= 2 * 2.0 ** -8 * p.abs() + 2 * (2.0 ** -12 + 2500 * 2.0 ** -23 + 2.0 ** -15) * size).all()
            none = lens <= 0
            assert (out[none] == 0).all() and torch.isneginf(lse[none]).all() and torch.isfinite(lse[~none]).all()


def test_shares_on_another_stream(mi, dev):
    import torch

    b = shared(90, 8, 4, 128, 2100, 3)
    want = run(mi, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(mi, b, sync=False)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    close(*want, b.reference(), 2100)
