"""Rotary positions (mi_rope) against the 64-bit formula.

Tolerance. The kernel rotates in fp32 and rounds once. A cosine or sine is off by at most four
half-steps of fp32 (its argument, in half turns, is rounded once, and sincospi adds two units), the
two products, their sum and the scale round once each: together at most 8 * 2^-24 = 2^-21 of
scale * (|a| + |b|). A bf16 result is rounded by another half step, 2^-8 of its value.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def reference(x, pos, freq, interleaved, scale=1.0, inverse=False):
    """x [B, T, H, d], pos [B, T] -> (rotated, |a| + |b| of each component's pair), float64."""
    x = x.astype(np.float64)
    n = freq.size
    ang = pos.astype(np.float64)[..., None] * freq.astype(np.float64)
    c, s = np.cos(ang)[:, :, None], np.sin(ang)[:, :, None] * (-1.0 if inverse else 1.0)
    ia = np.arange(0, 2 * n, 2) if interleaved else np.arange(n)
    ib = ia + 1 if interleaved else ia + n
    a, b = x[..., ia], x[..., ib]
    y, size = x.copy(), np.abs(x)
    y[..., ia], y[..., ib] = scale * (a * c - b * s), scale * (b * c + a * s)
    size[..., ia] = size[..., ib] = np.abs(scale) * (np.abs(a) + np.abs(b))
    return y, size


def check(got, ref, size, bf16):
    tol = 2.0 ** -21 * size + (2.0 ** -8 * np.abs(ref) * (1 + 2.0 ** -8) if bf16 else 0.0)
    err = np.abs(got.astype(np.float64) - ref)
    assert np.isfinite(got).all() and (err <= tol).all(), float((err - tol).max())


def host(t):
    return t.detach().float().cpu().numpy()


def make(shape, dtype, seed=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,T,H,d,rot", [
    (1, 1, 1, 128, 128), (2, 37, 5, 64, 64), (1, 300, 3, 128, 64), (3, 7, 2, 96, 24), (2, 5, 3, 6, 2),
    (1, 9, 2, 10, 10), (1, 4, 1, 1024, 1024), (2, 3, 40, 80, 16), (1, 2, 3, 2, 2), (1, 33, 24, 128, 32)])
def test_forward_and_inverse(mi, dev, dtype, interleaved, B, T, H, d, rot):
    import torch

    bf16 = dtype == "bf16"
    x = make((B, T, H, d), torch.bfloat16 if bf16 else torch.float32, B * T + d)
    f, one = mi.rope_frequencies(rot)
    assert one == 1.0
    pos = np.broadcast_to(np.arange(T), (B, T))
    fh = f.cpu().numpy()
    y = mi.rope(x, f, interleaved=interleaved)
    check(host(y), *reference(host(x), pos, fh, interleaved), bf16)
    y = mi.rope(x, f, interleaved=interleaved, pos0=1000, scale=1.25, inverse=True)
    check(host(y), *reference(host(x), pos + 1000, fh, interleaved, 1.25, True), bf16)


@pytest.mark.parametrize("start", [0, 131071, 2 ** 24 + 1, 2 ** 31 - 40, -(2 ** 31)])
def test_far_positions(mi, dev, start):
    import torch

    x = make((2, 33, 2, 64), torch.float32, 3)
    f, _ = mi.rope_frequencies(64)
    pos = (torch.arange(33, device="cuda") + start).to(torch.int32)
    two = torch.stack([pos, pos.flip(0)])
    for p, q in ((pos, pos.expand(2, 33)), (two, two)):
        check(host(mi.rope(x, f, positions=p)), *reference(host(x), q.cpu().numpy(), f.cpu().numpy(), False), False)


def test_positions_beyond_32_bits_from_pos0(mi, dev):
    import torch

    x = make((1, 5, 2, 32), torch.float32, 4)
    f = torch.full((16,), 2.0 ** -20, device="cuda")  # exact products
    pos = (np.arange(5) + 2 ** 40)[None]
    check(host(mi.rope(x, f, pos0=2 ** 40)), *reference(host(x), pos, f.cpu().numpy(), False), False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_layouts_and_in_place(mi, dev, dtype):
    import torch

    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    f, _ = mi.rope_frequencies(48)
    fh = f.cpu().numpy()
    B, T, H, d = 2, 19, 3, 64
    pos = np.broadcast_to(np.arange(T), (B, T))
    for pad, off in ((0, 0), (8, 8), (1, 1), (2, 4)):  # odd row pitches and addresses
        base = make((B, T, H * d + pad + off), dt, 7)
        x = base[..., off:off + H * d].unflatten(2, (H, d))
        want = reference(host(x), pos, fh, False)
        check(host(mi.rope(x, f)), *want, dtype == "bf16")
        out = torch.empty((B, H, T, d), dtype=dt, device="cuda")
        mi.rope(x.transpose(1, 2), f, layout="bhtd", out=out)
        check(host(out.transpose(1, 2)), *want, dtype == "bf16")
        keep = base.clone()
        mi.rope(x, f, out=x)
        check(host(x), *want, dtype == "bf16")
        assert torch.equal(base[..., :off], keep[..., :off]) and torch.equal(base[..., off + H * d:], keep[..., off + H * d:])
    one = make((B, T, 1, d), dt, 8)  # a head that several share: read by stride 0
    check(host(mi.rope(one.expand(B, T, H, d), f)),
          *reference(host(one.expand(B, T, H, d)), pos, fh, False), dtype == "bf16")


@pytest.mark.parametrize("dtype,interleaved", [("bf16", False), ("bf16", True), ("f32", False)])
@pytest.mark.parametrize("B,T,nH,nKV,d", [(2, 65, 12, 12, 64), (1, 130, 16, 4, 128), (3, 1, 8, 1, 96), (1, 3, 2, 0, 64)])
def test_qkv_both_ways(mi, dev, dtype, interleaved, B, T, nH, nKV, d):
    import torch

    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    bf16 = dtype == "bf16"
    f, _ = mi.rope_frequencies(d)
    fh = f.cpu().numpy()
    qkv = make((B, T, (nH + 2 * nKV) * d), dt, 11)
    pos = torch.randint(0, 5000, (B, T), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    kw = dict(positions=pos.cuda(), interleaved=interleaved, scale=0.75)
    out = mi.rope_qkv(qkv, nH, nKV, f, **kw)
    x = host(qkv).reshape(B, T, nH + 2 * nKV, d)
    y, size = reference(x[:, :, :nH + nKV], pos.numpy(), fh, interleaved, 0.75)
    check(host(out[0]).transpose(0, 2, 1, 3), y[:, :, :nH], size[:, :, :nH], bf16)
    check(host(out[1]).transpose(0, 2, 1, 3), y[:, :, nH:], size[:, :, nH:], bf16)
    assert np.array_equal(host(out[2]).transpose(0, 2, 1, 3), x[:, :, nH + nKV:])
    assert all(o.is_contiguous() for o in out)
    grads = [make(o.shape, dt, 20 + i) for i, o in enumerate(out)]
    back = mi.rope_qkv_backward(*grads, f, **kw)
    g = np.concatenate([host(t).transpose(0, 2, 1, 3) for t in grads], 2)
    y, size = reference(g[:, :, :nH + nKV], pos.numpy(), fh, interleaved, 0.75, True)
    got = host(back).reshape(B, T, nH + 2 * nKV, d)
    check(got[:, :, :nH + nKV], y, size, bf16)
    assert np.array_equal(got[:, :, nH + nKV:], g[:, :, nH + nKV:])


def test_gradient_against_differences(mi, dev):
    """The map is linear, so (f(x + e) - f(x - e)) / 2 along a direction e is its derivative whatever
    e's size; against <g, .> it must give <back(g), e>. Sums of n products of values near 1, each
    value off by 2^-21 * 2: at most n * 2^-19 in all, and n * 2^-24 * n for the sum in fp32, here in 64 bits."""
    import torch

    B, T, nH, nKV, d = 2, 9, 4, 2, 32
    f, _ = mi.rope_frequencies(24)
    x, e = (make((B, T, (nH + 2 * nKV) * d), torch.float32, s) for s in (1, 2))
    up, down = mi.rope_qkv(x + e, nH, nKV, f), mi.rope_qkv(x - e, nH, nKV, f)
    g = [make(t.shape, torch.float32, 5 + i) for i, t in enumerate(up)]
    slope = sum(float(((a.double() - b.double()) / 2 * c.double()).sum()) for a, b, c in zip(up, down, g))
    back = mi.rope_qkv_backward(*g, f)
    mine = float((back.double() * e.double()).sum())
    size = float(sum((a.abs().double() * c.abs().double()).sum() for a, c in zip(up, g)))
    assert abs(slope - mine) <= 2.0 ** -19 * max(size, x.numel())


def test_frequencies(mi, dev):
    i = np.arange(32)
    plain = 10000.0 ** (-2.0 * i / 64)

    def get(*a, **k):
        f, s = mi.rope_frequencies(*a, **k)
        return f.cpu().numpy().astype(np.float64), s

    def same(a, b):  # one rounding to fp32, of a value computed in 64 bits
        assert (np.abs(a - b) <= 2.0 ** -24 * (1 + 2.0 ** -20) * np.abs(b)).all()

    same(get(64)[0], plain)
    same(get(64, 500000.0)[0], 500000.0 ** (-2.0 * i / 64))
    same(get(64, scaling=("linear", 4.0))[0], plain / 4)
    f, _ = get(64, scaling=("base", 8.0))
    same(f[:1], plain[:1])
    same(f[-1:], plain[-1:] / 8)
    f, s = get(64, scaling=("bands", 8.0, 1.0, 32.0, 4096, 1.2))
    assert s == 1.2
    turns = 4096 * plain / (2 * np.pi)
    same(f[turns >= 32], plain[turns >= 32])
    same(f[turns <= 1], plain[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (f[mid] < plain[mid]).all() and (f[mid] > plain[mid] / 8).all()
    for bad in (("linear", 0.0), ("what", 2.0), ("bands", 2.0), ("bands", 2.0, 3.0, 3.0, 100), ("linear",)):
        with pytest.raises(ValueError):
            mi.rope_frequencies(64, scaling=bad)
    with pytest.raises(ValueError):
        mi.rope_frequencies(63)


def test_streams_and_graph(mi, dev):
    import torch

    f, _ = mi.rope_frequencies(128)
    qkv = make((2, 50, 24 * 128), torch.bfloat16, 1)
    want = [t.clone() for t in mi.rope_qkv(qkv, 16, 4, f)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mi.rope_qkv(qkv, 16, 4, f, sync=False)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mi.rope_qkv(qkv, 16, 4, f, sync=False)
        back = mi.rope_qkv_backward(*out, f, sync=False)
    for seed in (2, 3, 4):
        qkv.copy_(make(qkv.shape, torch.bfloat16, seed))
        eager = mi.rope_qkv(qkv, 16, 4, f)
        eager_back = mi.rope_qkv_backward(*eager, f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)) and torch.equal(back, eager_back)


def test_training_attention_path(mi, dev):
    """QKV rows -> rope_qkv -> flash_attn_fwd -> flash_attn_bwd -> rope_qkv_backward, against the 64-bit
    chain from the same rows. Bounds: every bf16 rounding on the way (Q, K, P, O and the gradients, dS)
    moves a result by at most 2^-8 of the terms it sums; with unit-variance rows the ten of them stay
    within 10 * 2^-8 of the largest result."""
    import torch

    B, T, nH, nKV, d = 1, 96, 4, 2, 64
    f, _ = mi.rope_frequencies(d)
    qkv = make((B, T, (nH + 2 * nKV) * d), torch.bfloat16, 9)
    dO = make((B, T, nH * d), torch.bfloat16, 10)
    Q, K, V = mi.rope_qkv(qkv, nH, nKV, f)
    lse = torch.empty((B, nH, T), dtype=torch.float32, device="cuda")
    O = mi.flash_attn_fwd(Q, K, V, lse=lse)
    dqkv = mi.rope_qkv_backward(*mi.flash_attn_bwd(Q, K, V, O, dO, lse), f)

    x = qkv.double().cpu().requires_grad_()
    q, k, v = x.view(B, T, nH + 2 * nKV, d).split((nH, nKV, nKV), dim=2)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * f.double().cpu()
    c, s = ang.cos()[None, :, None], ang.sin()[None, :, None]

    def turn(t):
        a, b = t[..., :d // 2], t[..., d // 2:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q, k, v = (t.transpose(1, 2) for t in (turn(q), turn(k), v))
    k, v = (t.repeat_interleave(nH // nKV, 1) for t in (k, v))
    p = torch.matmul(q, k.transpose(-1, -2)) / d ** 0.5
    p = p.masked_fill(torch.ones(T, T).triu(1).bool(), -float("inf")).softmax(-1)
    o = torch.matmul(p, v).transpose(1, 2).reshape(B, T, nH * d)
    o.backward(dO.double().cpu())
    for got, ref in ((O, o.detach()), (dqkv, x.grad)):
        err = (got.double().cpu() - ref).abs().max() / ref.abs().max()
        assert err <= 10 * 2.0 ** -8, float(err)
