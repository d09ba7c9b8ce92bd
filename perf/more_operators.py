"""Performance cases of the K/V cache that is held in 8 or 4 bits.

A case is a dict of plain values; `op` says which operator it is:

* ``append``  new tokens enter the cache, K rotated, K and V quantised as they are written, Q rotated;
              what was written is read back;
* ``read``    the last tokens of each sequence are read back from the cache;
* ``attend``  attention of each sequence's new tokens over its pages (the new tokens are the
              sequence's last ones, each sees the keys up to its own).

The format: 32 neighbouring components of a head of a token are a group. With m their largest
magnitude, e is the least integer with m <= L 2^e, at least -100, L = 464 for 8 bits and 7 for 4;
held are the byte e + 127 and, for each component, x / 2^e rounded to the nearest number of e4m3 (8
bits) or e2m1 (4 bits: 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), ties to even, at most 448 or
6. Two 4-bit components share a byte, the even one in its low half. K's rotation is not rounded
before. Codes are [pages, nKV, page size, bytes], scales [pages, nKV, page size, d / 32]; sequence s
has its tokens in the pages that row s of the page table names, in order. Sequence lengths belong to
the case (`lens` draws them), values to the seed.
"""
import math
import os
import random
import sys

import torch

own = False

HEADS = ((12, 12, 64), (16, 4, 128))  # GPT-small block, 1.6B block


def listed():
    return [
        # token generation for 64 sequences: one new token each, 4 bits
        {"name": "append_e2m1_decode_s64", "op": "append", "bits": 4, "S": 64, "q_max": 1, "kv_max": 256, "nH": 16,
         "nKV": 4, "d": 128, "rot": 128, "interleaved": False, "page": 16, "lens": 3},
        # prompts of unequal length enter a 4-bit cache together
        {"name": "append_e2m1_prompts_s12", "op": "append", "bits": 4, "S": 12, "q_max": 1000, "kv_max": 1500,
         "nH": 16, "nKV": 4, "d": 128, "rot": 128, "interleaved": False, "page": 64, "lens": 4},
        # chunks and next tokens in one batch, 8 bits, 12 heads of 64 of which half turns, in neighbouring pairs
        {"name": "append_e4m3_mixed_s16", "op": "append", "bits": 8, "S": 16, "q_max": 333, "kv_max": 2500, "nH": 12,
         "nKV": 12, "d": 64, "rot": 32, "interleaved": True, "page": 32, "lens": 8},
        # a cached conversation of odd length, read back for another use of its prefix, 8 bits
        {"name": "read_e4m3_s1", "op": "read", "bits": 8, "S": 1, "q_max": 2047, "kv_max": 2047, "nH": 12, "nKV": 12,
         "d": 64, "page": 32, "lens": 1},
        # long contexts of several users read back, 4 bits
        {"name": "read_e2m1_s8", "op": "read", "bits": 4, "S": 8, "q_max": 16000, "kv_max": 16000, "nH": 16, "nKV": 4,
         "d": 128, "page": 64, "lens": 2},
        # one user's next token over 2047 cached ones, where latency counts
        {"name": "attend_e2m1_decode_s1", "op": "attend", "bits": 4, "S": 1, "q_max": 1, "kv_max": 2048, "nH": 16,
         "nKV": 4, "d": 128, "page": 64, "lens": 5},
        # next tokens of 64 sequences with 500 to 8000 cached tokens
        {"name": "attend_e2m1_decode_s64", "op": "attend", "bits": 4, "S": 64, "q_max": 1, "kv_max": 8000, "nH": 16,
         "nKV": 4, "d": 128, "page": 16, "lens": 6},
        # next tokens of long contexts, 8 bits
        {"name": "attend_e4m3_decode_s16", "op": "attend", "bits": 8, "S": 16, "q_max": 1, "kv_max": 32768, "nH": 16,
         "nKV": 4, "d": 128, "page": 64, "lens": 9},
        # up to four tokens a sequence checked at once, 12 heads of 64
        {"name": "attend_e2m1_few_s32", "op": "attend", "bits": 4, "S": 32, "q_max": 4, "kv_max": 3000, "nH": 12,
         "nKV": 12, "d": 64, "page": 32, "lens": 10},
        # chunks of up to 1024 prompt tokens of four sequences of 4095 tokens at most
        {"name": "attend_e2m1_chunk_s4", "op": "attend", "bits": 4, "S": 4, "q_max": 1024, "kv_max": 4095, "nH": 16,
         "nKV": 4, "d": 128, "page": 64, "lens": 7},
        # short chunks and next tokens in one batch, 12 heads of 64, 8 bits
        {"name": "attend_e4m3_mixed_s16", "op": "attend", "bits": 8, "S": 16, "q_max": 333, "kv_max": 2500, "nH": 12,
         "nKV": 12, "d": 64, "page": 32, "lens": 8},
    ]


# ---- drawn cases -------------------------------------------------------------------------

def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(("append", "read", "attend", "attend"))
    nH, nKV, d = rng.choice(HEADS + ((16, 16, 64), (8, 1, 128), (32, 8, 128), (8, 8, 96), (6, 2, 32)))
    c = {"op": op, "bits": rng.choice((8, 4)), "S": _log(rng, 1, 256), "q_max": 1, "kv_max": 1, "nH": nH, "nKV": nKV,
         "d": d, "page": rng.choice((16, 32, 64, 128)), "lens": rng.randrange(1 << 20)}
    if op == "read":
        c["q_max"] = _log(rng, 1, 16384)
        c["kv_max"] = c["q_max"] + rng.choice((0, _log(rng, 1, 2000)))
        return c
    if rng.random() >= 0.5:
        c["q_max"] = _log(rng, 2, 2048)
    c["kv_max"] = c["q_max"] + _log(rng, 1, 1000 if op == "append" else 65536)
    if op == "append":
        c.update(rot=rng.choice((d, d, d // 2, d // 4)), interleaved=rng.random() < 0.5)
    return c


def _cost(c):
    """(bytes that have to move, operations, values that the plain form holds at once)."""
    w = work(c)
    held = c["S"] * 2 * c["nKV"] * c["kv_max"] * c["d"]
    if c["op"] == "attend":
        held += c["S"] * c["nH"] * c["q_max"] * c["kv_max"]
    return w["bytes"], w["flops"], held


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = tuple(map(max, zip(_cost(c), most.get(c["op"], (0, 0, 0)))))
    while True:
        c = _draw(rng)
        if all(a <= b for a, b in zip(_cost(c), most[c["op"]])):
            return c


# ---- inputs ------------------------------------------------------------------------------

def _lens(c):
    """(new tokens, cached tokens with the new ones) of each sequence; the first has the largest of both."""
    r = random.Random(c["lens"])
    q = [c["q_max"]] + [_log(r, 1, c["q_max"]) for _ in range(c["S"] - 1)]
    before = c["kv_max"] - c["q_max"]
    return q, [n + (before if i == 0 else _log(r, max(1, before // 16), max(1, before)) if before else 0)
               for i, n in enumerate(q)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)

    q_len, kv_len = _lens(c)
    P, d, total = c["page"], c["d"], sum(q_len)
    n_pages = [-(-n // P) for n in kv_len]
    ids = torch.randperm(sum(n_pages), generator=g, device="cuda").to(torch.int32)
    width = max(n_pages)
    used = torch.arange(width, device="cuda") < torch.tensor(n_pages, device="cuda")[:, None]
    s = {"case": c}
    s["pages"] = torch.zeros((c["S"], width), dtype=torch.int32, device="cuda").masked_scatter_(used, ids)
    # cached values of unlike sizes from head to head and token to token, as a model's are
    for name in ("k", "v"):
        size = torch.exp(0.5 * torch.randn((sum(n_pages), c["nKV"], P, 1), generator=g, device="cuda"))
        s[name + "_codes"], s[name + "_scale"] = _quantised(normal(sum(n_pages), c["nKV"], P, d) * size, c["bits"])
    starts = torch.tensor([0] + q_len).cumsum(0)
    s["q_start"] = starts.to(torch.int32).cuda()
    s["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    s["max_q"], s["max_kv"] = max(q_len), max(kv_len)
    s["seq"] = torch.repeat_interleave(torch.arange(c["S"]), torch.tensor(q_len)).cuda()
    s["row"] = torch.arange(total).cuda() - starts.cuda()[s["seq"]]
    if c["op"] == "append":
        qkv = normal(total, c["nH"] + 2 * c["nKV"], d)
        s["q"], s["k"], s["v"] = qkv.split((c["nH"], c["nKV"], c["nKV"]), dim=1)
        i = torch.arange(0, c["rot"] // 2, dtype=torch.float64)
        s["freq"] = (10000.0 ** (-2.0 * i / c["rot"])).to(torch.float32).cuda()
    elif c["op"] == "attend":
        s["q"] = normal(total, c["nH"], d)
    return s


# ---- the framework's kernels ---------------------------------------------------------------

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "large-language-model_amd"))


def _run_own(s):
    import mi_gemm as mi

    c = s["case"]
    cache = mi.QuantCache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    # the start rows of the new tokens; None where every sequence has one, as a decode loop knows
    starts = None if s["max_q"] == 1 else s["q_start"]
    if c["op"] == "attend":
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
        o = mi.paged_attn_quant(s["q"], cache, s["pages"], s["kv_len"], q_start=starts, max_q_len=s["max_q"],
                                max_kv_len=s["max_kv"], lse=lse, sync=False)
        return o, lse
    if c["op"] == "read":
        return mi.kv_read_quant(cache, s["pages"], s["kv_len"], q_start=starts, rows=s["seq"].numel(), sync=False)
    q = mi.kv_append_quant(s["k"], s["v"], cache, s["pages"], s["kv_len"], q_start=starts, q=s["q"],
                           inv_freq=s["freq"], interleaved=c["interleaved"], sync=False)
    return (q,) + mi.kv_read_quant(cache, s["pages"], s["kv_len"], q_start=starts, rows=s["seq"].numel(), sync=False)


# ---- the plain forms -----------------------------------------------------------------------

def _power(e):
    """2^e, from its bits."""
    return (e.int() + 127 << 23).view(torch.float32)


def _quantised(x, bits):
    """Codes and scale bytes of x [..., d], d a multiple of 32."""
    x = x.unflatten(-1, (-1, 32))
    m = x.abs().amax(-1, keepdim=True)
    f, e = torch.frexp(m)  # m = f 2^e with f in [1/2, 1)
    top, below = (0.875, 3) if bits == 4 else (0.90625, 9)
    e = (e - below + (f > top)).masked_fill_(m == 0, -100).clamp_(min=-100)
    x = x * _power(-e)
    a = x.abs()
    if bits == 4:
        n = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
             + 8 * torch.signbit(x).byte())
        codes = n[..., 0::2] + 16 * n[..., 1::2]
    else:
        low = torch.frexp(a)[1].clamp_(min=-5) - 4  # the step between numbers of a's size is 2^low
        a = (torch.round(a * _power(-low)) * _power(low)).clamp_(max=448.0)
        codes = torch.copysign(a, x).float().to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.flatten(-2), (e + 127).squeeze(-1).byte()


def _values(codes, scale):
    """What codes [..., bytes] with scale bytes [..., groups] stand for, fp32 [..., 32 groups]."""
    if codes.shape[-1] == 16 * scale.shape[-1]:
        v = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0), device=codes.device)
        v = torch.cat((v, -v))
        pairs = torch.stack((v.repeat(16), v.repeat_interleave(16)), -1)  # of each byte
        v = pairs[codes.int()].flatten(-2)
    else:
        v = codes.view(torch.float8_e4m3fn).float()
    return (v.unflatten(-1, (-1, 32)) * _power(scale.int() - 127)[..., None]).flatten(-2)


def _slots(s):
    """Page and slot of each new token."""
    n = s["q_start"][1:] - s["q_start"][:-1]
    pos = (s["kv_len"] - n)[s["seq"]] + s["row"]
    return pos, s["pages"][s["seq"], pos // s["case"]["page"]].long(), pos % s["case"]["page"]


def _turn(x, cos, sin, interleaved):
    """x [..., d] with its first 2 * cos.shape[-1] components rotated pair by pair."""
    n = cos.shape[-1]
    r = x[..., : 2 * n]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :n], r[..., n:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, x[..., 2 * n:]), -1)


def _plain_append(s):
    c = s["case"]
    pos, page, slot = _slots(s)
    t = pos.double()[:, None, None] * s["freq"].double()
    cos, sin = t.cos(), t.sin()
    # in 64 bits up to the codes: a value next to the border of two of them could turn either way in 32
    k = _quantised(_turn(s["k"].double(), cos, sin, c["interleaved"]), c["bits"])
    v = _quantised(s["v"].float(), c["bits"])
    s["k_codes"][page, :, slot], s["k_scale"][page, :, slot] = k
    s["v_codes"][page, :, slot], s["v_scale"][page, :, slot] = v
    q = _turn(s["q"].float(), cos.float(), sin.float(), c["interleaved"]).to(s["q"].dtype)
    return (q,) + _plain_read(s)


def _plain_read(s):
    _, page, slot = _slots(s)
    return tuple(_values(s[n + "_codes"][page, :, slot], s[n + "_scale"][page, :, slot]).to(torch.bfloat16)
                 for n in ("k", "v"))


def _plain_attend(s):
    c = s["case"]
    S, nH, nKV, d, mq = c["S"], c["nH"], c["nKV"], c["d"], s["max_q"]
    n = s["q_start"][1:] - s["q_start"][:-1]

    def gathered(name):  # [S, nKV, keys, d]
        codes, scale = (s[name + x][s["pages"].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)
                        for x in ("_codes", "_scale"))
        return _values(codes, scale)

    k, v = gathered("k"), gathered("v")
    q = torch.zeros((S, mq, nH, d), device="cuda")
    q[s["seq"], s["row"]] = s["q"].float()
    q = q.permute(0, 2, 1, 3).reshape(S, nKV, nH // nKV * mq, d)
    x = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(S, nH, mq, -1)
    key = torch.arange(k.shape[2], device="cuda")
    last = (s["kv_len"] - n)[:, None] + torch.arange(mq, device="cuda")
    x.masked_fill_((key > last[..., None])[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x.sub_(m).exp_()
    t = x.sum(-1, keepdim=True)
    o = (x.view(S, nKV, -1, x.shape[-1]) @ v).view(S, nH, mq, d) / t
    at = (s["seq"], slice(None), s["row"])
    return o[at].to(s["q"].dtype), (m + t.log()).squeeze(-1)[at]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_append(state) if op == "append" else _plain_read(state) if op == "read" else _plain_attend(state)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    c = case
    q_len, kv_len = _lens(c)
    new, d = sum(q_len), c["d"]
    held = d * c["bits"] // 8 + d // 32  # bytes of a head of a cached token, K or V
    if c["op"] == "append":
        return {"bytes": new * (4 * c["nH"] * d + 2 * c["nKV"] * (2 * d + 2 * held + 2 * d)),
                "flops": new * (3 * c["nH"] * d + 9 * c["nKV"] * d)}
    if c["op"] == "read":
        return {"bytes": new * 2 * c["nKV"] * (held + 2 * d), "flops": new * 2 * c["nKV"] * d}
    seen = sum(n * k - n * (n - 1) // 2 for n, k in zip(q_len, kv_len))
    return {"bytes": 2 * c["nKV"] * held * sum(kv_len) + 4 * c["nH"] * (d + 1) * new, "flops": 4 * c["nH"] * d * seen}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _grid(bits):
    """The numbers of the type from 0 on, 64 bits: code n is the sign-less number n."""
    n = torch.arange(8 if bits == 4 else 127, device="cuda", dtype=torch.float64)
    m = 1 if bits == 4 else 3                 # bits behind the point
    low = 1 if bits == 4 else 7               # exponent bias
    e, f = (n / 2**m).floor(), n % 2**m
    return torch.where(e == 0, f / 2**m * 2.0 ** (1 - low), (1 + f / 2**m) * (e - low).exp2())


def _held(x, bits):
    """The values that stand for x [..., d] in the cache, by looking for the nearest number."""
    grid = _grid(bits)
    x = x.double().unflatten(-1, (-1, 32))
    m = x.abs().amax(-1, keepdim=True)
    most = 7.0 if bits == 4 else 464.0
    e = torch.log2(m / most).ceil()
    e = torch.where(m > most * e.exp2(), e + 1, torch.where(m <= most * (e - 1).exp2(), e - 1, e)).clamp(min=-100.0)
    a = x.abs() / e.exp2()
    above = torch.searchsorted(grid, a).clamp(1, grid.numel() - 1)  # first number >= a, the last if there is none
    up, down = grid[above] - a, a - grid[above - 1]
    n = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, above - 1)
    return (grid[n] * e.exp2() * x.sign()).flatten(-2)


def _meant(codes, scale, bits):
    """What codes and scale bytes stand for, from their bits."""
    n = codes.int()
    if bits == 4:
        n = torch.stack((n & 15, n >> 4), -1).flatten(-2)
    sign = 1.0 - 2.0 * (n >> (bits - 1)).double()
    v = _grid(bits)[n & ((1 << (bits - 1)) - 1)] * sign
    return v * (scale.double() - 127.0).exp2().repeat_interleave(32, -1)


def _rotated(x, pos, freq, interleaved):
    """x [tokens, heads, d] as complex pairs times exp(i pos freq), 64 bits."""
    n = freq.numel()
    x = x.double().clone()
    z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), pos.double()[:, None] * freq.double())
    re, im = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y = torch.complex(x[..., re], x[..., im]) * z[:, None]
    x[..., re], x[..., im] = y.real, y.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    g, d, P = c["nH"] // c["nKV"], c["d"], c["page"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    out = []
    for i in range(c["S"]):
        a, b, n = starts[i], starts[i + 1], lens[i]
        first = n - (b - a)
        if c["op"] == "append":
            pos = torch.arange(first, n, device="cuda")
            out.append((_rotated(s["q"][a:b], pos, s["freq"], c["interleaved"]),
                        _held(_rotated(s["k"][a:b], pos, s["freq"], c["interleaved"]), c["bits"]),
                        _held(s["v"][a:b], c["bits"])))
            continue
        ids = s["pages"][i, : -(-n // P)].long()
        heads = []
        for h in range(c["nKV"]):
            k, v = (_meant(s[x + "_codes"][ids, h].flatten(0, 1)[:n], s[x + "_scale"][ids, h].flatten(0, 1)[:n], c["bits"])
                    for x in ("k", "v"))
            if c["op"] == "read":
                heads.append((k[first:], v[first:]))
                continue
            hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(first, n, device="cuda")[:, None]
            for j in range(h * g, h * g + g):
                x = torch.mm(s["q"][a:b, j].double(), k.t()) / math.sqrt(d)
                x = torch.where(hidden, -math.inf, x)
                lse = torch.logsumexp(x, -1)
                heads.append((torch.mm((x - lse[:, None]).exp(), v), lse))
        out.append(tuple(torch.stack(x, 1) for x in zip(*heads)))
    return tuple(torch.cat(x) for x in zip(*out))
