"""Sampling (mi_sample) against the definition in 64 bits: tokens are equal, without tolerance. The
definition counts weights in whole multiples of 2^-(62 - b) (2^-50 at
most), b the bits of V - 1, and so does the oracle.

The picked token's share is a quotient of two sums of 64-bit weights, rounded once to fp32: 2^-24 of
its value, with 2^-40 for the weights' own rounding.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def reference(x, u, T, k, p, low):
    """(token, share) of one row, float64 throughout, by sorting."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(x.size), -x))
    top = x[order[0]]
    if top == -np.inf:
        return -1, 0.0
    n = x.size
    if not T > 0:
        n, T = 1, 1.0
    elif k > 0:
        n = min(k, n)
    y = x[order[:n]]
    with np.errstate(invalid="ignore"):
        w = np.where(y == top, 1.0, np.where(y == -np.inf, 0.0, np.exp((y - top) / T)))
    unit = 2.0 ** min(50, 62 - int(x.size - 1).bit_length())
    exact, w = w, np.rint(w * unit)
    if p < 1:
        mass = np.cumsum(w)
        before = mass - w
        before[0] = 0.0
        w = w[(before < p * mass[-1]) | (np.arange(n) == 0)]
    if low > 0:
        keep = exact[:w.size] >= low
        keep[0] = True
        w = w[keep]
    kept = order[:w.size]
    by = np.argsort(kept)
    mass = np.cumsum(w[by])
    at = int(np.searchsorted(mass, u * mass[-1], side="right"))
    at = min(at, int(np.flatnonzero(w[by])[-1]))
    return int(kept[by[at]]), float(w[by[at]] / mass[-1])


def check(mi, x, u, T=1.0, k=0, p=1.0, low=0.0):
    """x [rows, V] on the GPU, settings numbers or per-row tensors."""
    import torch

    rows = x.shape[0]
    prob = torch.full((rows,), -1.0, device="cuda")
    got = mi.sample(x, u, temperature=T, top_k=k, top_p=p, min_p=low, prob=prob)
    each = [(v.cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, np.float32(v))) for v in (T, k, p, low)]
    h, uh = x.float().cpu().numpy(), u.cpu().numpy().astype(np.float64)
    ref = [reference(h[r], uh[r], float(each[0][r]), int(each[1][r]), float(each[2][r]), float(each[3][r]))
           for r in range(rows)]
    assert got.cpu().tolist() == [t for t, _ in ref]
    share = np.array([s for _, s in ref])
    assert (np.abs(prob.double().cpu().numpy() - share) <= (2.0 ** -24 + 2.0 ** -40) * share + 2.0 ** -60).all()
    return got


def make(rows, V, dtype, seed, std=2.5):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    return (torch.randn((rows, V), generator=g, device="cuda") * std).to(dt), \
        torch.rand((rows,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1024, 4099, 32000, 32001, 70000, 151936])
@pytest.mark.parametrize("how", [dict(), dict(T=0.0), dict(k=1), dict(k=7, T=0.7), dict(k=50, p=0.9), dict(p=0.5),
                                 dict(p=0.95, T=1.5), dict(low=0.05), dict(k=40, p=0.9, low=0.1, T=0.8), dict(p=0.0),
                                 dict(k=10 ** 6, p=0.999)])
def test_settings(mi, dev, dtype, V, how):
    x, u = make(5, V, dtype, V)
    check(mi, x, u, **how)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 3, 64, 300])
def test_each_row_its_own(mi, dev, dtype, rows):
    import torch

    x, u = make(rows, 5003, dtype, rows)
    g = torch.Generator(device="cuda").manual_seed(9)
    pick = lambda v, dt: torch.tensor(v, dtype=dt, device="cuda")[  # noqa: E731
        torch.randint(0, len(v), (rows,), generator=g, device="cuda")]
    check(mi, x, u, T=pick((0.0, 0.3, 1.0, 2.0, -1.0), torch.float32), k=pick((0, 1, 5, 100, -3), torch.int32),
          p=pick((1.0, 0.2, 0.9, 0.99, 2.0), torch.float32), low=pick((0.0, 0.01, 0.5, 1.0, -1.0), torch.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("how", [dict(), dict(k=3), dict(k=700), dict(p=0.3), dict(p=0.9, k=800), dict(low=1.0),
                                 dict(T=0.0), dict(low=0.5, T=0.5)])
def test_ties(mi, dev, dtype, how):
    """Few distinct logits: borders fall inside runs of equal ones, which go by index."""
    import torch

    for values, V in (((0.0,), 3001), ((-0.0, 0.0), 777), ((1.0, 1.0, 0.5, -2.0), 5000), ((-3.0, -3.0, -50.0), 20000)):
        g = torch.Generator(device="cuda").manual_seed(V)
        x = torch.tensor(values, device="cuda")[torch.randint(0, len(values), (6, V), generator=g, device="cuda")]
        x = x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)
        u = torch.tensor([0.0, 0.25, 0.5, 0.7501, 0.999, 1 - 2.0 ** -24], device="cuda")
        check(mi, x, u, **how)
        check(mi, x.repeat(50, 1), u.repeat(50), **how)  # more rows than CUs


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("how", [dict(), dict(k=4), dict(p=0.9), dict(T=0.0), dict(low=0.2), dict(k=2, p=0.5, T=3.0)])
def test_infinities_and_nan(mi, dev, dtype, how):
    import torch

    inf, nan = float("inf"), float("nan")
    big = 3e38
    rows = [[-inf] * 8, [nan] * 8, [-inf, nan, -inf, 1.0, -inf, nan, -inf, -inf], [inf, 0.0, inf, 1.0, 2.0, inf, nan, -inf],
            [-big, -big, -inf, -big, nan, -inf, -big, -big], [big, -big, big, 0.0, 1.0, -inf, big, nan],
            [1e-45, 0.0, -1e-45, -0.0, 1e-40, -inf, -inf, -inf], [5.0, 4.0, 3.0, nan, 2.0, 1.0, 0.0, -1.0]]
    x = torch.tensor(rows, device="cuda").to(torch.bfloat16 if dtype == "bf16" else torch.float32)
    for a in (0.0, 0.4, 0.99):
        check(mi, x, torch.full((8,), a, device="cuda"), **how)
        check(mi, x.repeat(40, 1), torch.full((320,), a, device="cuda"), **how)


def test_extreme_settings(mi, dev):
    import torch

    x, u = make(4, 999, "f32", 1)
    inf = float("inf")
    check(mi, x, u, T=1e-30)            # the largest takes all
    check(mi, x, u, T=1e-45)            # a denormal
    check(mi, x, u, T=1e30)             # all alike
    check(mi, x, u, k=-(2 ** 31))
    check(mi, x, u, k=2 ** 31 - 1)
    check(mi, x, u, p=-1.0)
    check(mi, x, u, low=2.0)
    check(mi, x * 1e4, u, p=0.9)
    same = mi.sample(x, u, temperature=inf, top_p=float("nan"), min_p=float("nan"))  # filters that say nothing are off
    assert same.tolist() == mi.sample(x * 0, u).tolist()
    assert mi.sample(x, u, temperature=float("nan")).tolist() == x.argmax(1).tolist()
    # numbers outside [0, 1) and NaN stay within what is kept
    odd = torch.tensor([-1.0, 1.0, inf, float("nan")], device="cuda")
    got, order = mi.sample(x, odd, top_k=3).tolist(), x.argsort(1, descending=True)[:, :3].sort(1).values.tolist()
    assert got == [order[0][0], order[1][2], order[2][2], order[3][0]]


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("how", [dict(k=100), dict(k=160, p=0.9), dict(k=161, p=0.5), dict(k=255), dict(k=2000, p=0.99),
                                 dict(p=0.9), dict(p=0.999, low=1e-4), dict(k=30, p=0.8, low=0.03, T=0.5)])
def test_peaked_and_flat_rows(mi, dev, rows, how):
    """Rows whose top tokens lie together in one lane's run, rows that are nearly flat, and rows with a tail."""
    import torch

    x, u = make(rows, 9001, "f32", rows)
    x[::3, 500:700] += 30.0
    x[1::3] *= 1e-3
    check(mi, x, u, **how)
    check(mi, x.bfloat16(), u, **how)


@pytest.mark.parametrize("rows", [1, 13, 300])
@pytest.mark.parametrize("how", [dict(p=0.9), dict(p=0.5, low=0.2, T=0.6), dict(k=257), dict(k=1000, p=0.9, low=1e-3),
                                 dict(k=8999, T=2.0), dict(p=0.999999, T=5.0), dict(p=0.9, T=1e-3)])
def test_long_rows_of_bf16(mi, dev, rows, how):
    """Rows by what their distinct logits are: a few, thousands, zeros of both signs, masked and infinite
    ones, the smallest and largest."""
    import torch

    x, u = make(rows, 9000, "bf16", rows)
    inf = float("inf")
    x[1::13] = x[1::13].float().round().bfloat16()          # ties by the hundred
    x[2::13, 17:] = -inf                                    # nearly all masked
    x[3::13] = -inf
    x[4::13, 8999:] = inf
    x[5::13, 100:120] = float("nan")
    x[6::13] = (x[6::13].float() * 2.0 ** 70).bfloat16()
    x[7::13, 5] = 1e-30
    x[8::13] = torch.tensor([0.0, -0.0], device="cuda").bfloat16().repeat(4500)
    x[9::13] = (torch.arange(9000, device="cuda") - 4500 + 0x3f80).to(torch.int16).view(torch.bfloat16)  # all distinct
    x[10::13] = (torch.arange(9000, device="cuda") // 3 + 0x3f80 - 1500).to(torch.int16).view(torch.bfloat16)
    x[11::13] = x[11::13] - 60.0                            # none above 0
    x[12::13, ::2] = -1.8e19                                # the lowest places but two
    x[12::13, ::3] = -1.85e19
    check(mi, x, u, **how)


@pytest.mark.parametrize("V", [8191, 8192, 8193, 65535, 65536, 65537, 140001, 300000])
@pytest.mark.parametrize("how", [dict(p=0.9), dict(k=5000, p=0.99)])
def test_lengths_of_long_rows_of_bf16(mi, dev, V, how):
    import torch

    x, u = make(3, V + 3, "bf16", V)
    check(mi, x[:, :V], u, **how)
    check(mi, x[:, 1:V + 1], u, **how)
    check(mi, x[:1, 2:V + 2], u[:1], **how)
    check(mi, (x[:, 2:V + 2] * 0).contiguous(), u, **how)  # all alike: one counter for the whole row
    check(mi, (x[:, 2:V + 2] * 0 + 1).contiguous(), u, **how)
    check(mi, (x[:, 2:V + 2] * 0 + 1.0078125).contiguous(), u, **how)
    one = torch.full((3, V), -30.0, device="cuda").bfloat16()
    one[0, 0] = one[1, V // 2] = one[2, V - 1] = 2.0
    check(mi, one, u, **how)


def test_settings_of_long_rows(mi, dev):
    """In one batch: rows without borders, greedy ones, and those with each of the borders."""
    import torch

    x, u = make(300, 10007, "bf16", 11)
    t = lambda v, dt: torch.tensor(v, dtype=dt, device="cuda").repeat(300 // len(v))  # noqa: E731
    check(mi, x, u, T=t((1.0, 0.0, 0.7, 1.3, 0.9), torch.float32), k=t((0, 0, 40, 256, 257, 5000), torch.int32),
          p=t((1.0, 0.9, 0.3, 0.99), torch.float32), low=t((0.0, 0.0, 0.05), torch.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_row_pitch_and_alignment(mi, dev, dtype):
    import torch

    base, u = make(7, 4099, dtype, 3)
    base[:, 4000:] = 50.0  # what lies behind a row is not part of it
    base[:, :3] = 50.0
    keep = base.clone()
    for a, b in ((3, 4000), (3, 3999), (4, 4000), (8, 3528), (3, 4)):
        check(mi, base[:, a:b], u, k=20, p=0.9)
    assert torch.equal(base, keep)
    check(mi, base[:1, 3:500], u[:1])


def test_uniform_numbers_cover_the_distribution(mi, dev):
    """Over an even grid of u each token comes up as often as its weight says, to within one."""
    import torch

    n = 4096
    x = torch.tensor([2.0, -1.0, 0.5, -float("inf"), 2.0, 0.0], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = mi.sample(x.expand(n, 6).contiguous(), u, temperature=0.9).cpu().numpy()
    w = np.exp(np.array([2.0, -1.0, 0.5, -np.inf, 2.0, 0.0]) / 0.9)
    assert (np.diff(got) >= 0).all()  # index order
    assert (np.abs(np.bincount(got, minlength=6) - n * w / w.sum()) <= 1.0).all()


def test_streams_and_graph(mi, dev):
    import torch

    x, u = make(16, 32000, "bf16", 5)
    k = torch.arange(16, dtype=torch.int32, device="cuda") * 5
    want = mi.sample(x, u, top_k=k, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mi.sample(x, u, top_k=k, top_p=0.9, sync=False)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mi.sample(x, u, top_k=k, top_p=0.9, sync=False)
    for seed in (6, 7, 8):
        y, w = make(16, 32000, "bf16", seed)
        x.copy_(y)
        u.copy_(w)
        eager = mi.sample(x, u, top_k=k, top_p=0.9)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_graph_of_long_rows(mi, dev):
    """Counted rows, and after them rows that the counts cannot hold, from one captured call."""
    import torch

    x, u = make(300, 9000, "bf16", 5)
    p = torch.full((300,), 0.9, device="cuda")
    g = torch.cuda.CUDAGraph()
    mi.sample(x, u, top_p=p)
    with torch.cuda.graph(g):
        out = mi.sample(x, u, top_p=p, sync=False)
    for seed in (6, 7, 8):
        y, w = make(300, 9000, "bf16", seed)
        if seed == 7:
            y[::2, 9] = 1e-30
        x.copy_(y)
        u.copy_(w)
        p.copy_(w * 0.5 + 0.4)
        eager = check(mi, x, u, p=p)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_logits_of_the_head(mi, dev):
    """The LM head's product, then its tokens, as a decode step ends: hidden rows -> logits -> tokens."""
    import torch

    h, _ = make(8, 256, "bf16", 1, 1.0)
    W, _ = make(256, 1999, "bf16", 2, 0.1)
    _, u = make(8, 1, "f32", 3)
    logits = mi.matmul(h, W)
    check(mi, logits, u, T=0.8, k=50, p=0.95)
