"""Performance cases of the serving chain's operators and of rotary positions in training.

A case is a dict of plain values; `op` says which operator it is:

* ``rope``    rotary positions between the QKV projection and the attention: the product's rows
              [B, T, (nH + 2 nKV) d] become Q [B, nH, T, d], K and V [B, nKV, T, d] with Q and K
              rotated; with ``train`` also the way back, dQ, dK, dV to the product's gradient;
* ``append``  new tokens enter a paged cache: K rotated and V as it is into the pages, Q rotated;
* ``attend``  attention of each sequence's new tokens over its pages (the new tokens are the
              sequence's last ones, each sees the keys up to its own);
* ``sample``  a token for each row of logits by temperature, top-k, top-p and min-p.

A cache is [pages, nKV, page size, d]; sequence s has its tokens in the pages that row s of the page
table names, in order. Sequence lengths belong to the case (`lens` draws them), values to the seed.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

BF16, F32 = "bf16", "f32"
HEADS = ((12, 12, 64), (16, 4, 128))  # GPT-small block, 1.6B block


def listed():
    return [
        # the smallest call: the fp32 GPT-small block on one sequence of 128 tokens
        {"name": "rope_f32_t128", "op": "rope", "B": 1, "T": 128, "nH": 12, "nKV": 12, "d": 64,
         "rot": 64, "interleaved": False, "dtype": F32, "train": False, "pos": 0, "factor": 1.0},
        # a training step of the 1.6B block, 8 x 1024 tokens, both directions
        {"name": "rope_train_t1024", "op": "rope", "B": 8, "T": 1024, "nH": 16, "nKV": 4, "d": 128,
         "rot": 128, "interleaved": False, "dtype": BF16, "train": True, "pos": 0, "factor": 1.0},
        # a long prompt at far positions, half of each head rotated, neighbouring pairs, frequencies
        # scaled for a longer context, odd length
        {"name": "rope_long_t16381", "op": "rope", "B": 1, "T": 16381, "nH": 16, "nKV": 4, "d": 128,
         "rot": 64, "interleaved": True, "dtype": BF16, "train": False, "pos": 98304, "factor": 8.0},
        # token generation for 64 sequences: one new token each
        {"name": "append_decode_s64", "op": "append", "S": 64, "q_max": 1, "kv_max": 256, "nH": 16,
         "nKV": 4, "d": 128, "rot": 128, "interleaved": False, "page": 16, "lens": 3},
        # prompts of unequal length enter the cache together
        {"name": "append_prompts_s12", "op": "append", "S": 12, "q_max": 1000, "kv_max": 1500, "nH": 16,
         "nKV": 4, "d": 128, "rot": 128, "interleaved": False, "page": 64, "lens": 4},
        # one user's next token over 2047 cached ones, where latency counts
        {"name": "attend_decode_s1", "op": "attend", "S": 1, "q_max": 1, "kv_max": 2048, "nH": 16,
         "nKV": 4, "d": 128, "page": 64, "lens": 5},
        # next tokens of 64 sequences with 500 to 8000 cached tokens
        {"name": "attend_decode_s64", "op": "attend", "S": 64, "q_max": 1, "kv_max": 8000, "nH": 16,
         "nKV": 4, "d": 128, "page": 16, "lens": 6},
        # chunks of 1024 prompt tokens of four sequences of 4095 tokens at most
        {"name": "attend_chunk_s4", "op": "attend", "S": 4, "q_max": 1024, "kv_max": 4095, "nH": 16,
         "nKV": 4, "d": 128, "page": 64, "lens": 7},
        # short chunks and next tokens in one batch, 12 heads of 64
        {"name": "attend_mixed_s16", "op": "attend", "S": 16, "q_max": 333, "kv_max": 2500, "nH": 12,
         "nKV": 12, "d": 64, "page": 32, "lens": 8},
        # one user's token from bf16 logits
        {"name": "sample_s1_v32000", "op": "sample", "rows": 1, "vocab": 32000, "dtype": BF16,
         "ld": 32000, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # a serving batch, fp32 logits, vocabulary with one added token, each user's own settings
        {"name": "sample_s64_v32001", "op": "sample", "rows": 64, "vocab": 32001, "dtype": F32,
         "ld": 32064, "temperature": -1.0, "top_k": -1, "top_p": -1.0, "min_p": -1.0},
        # generation for a whole evaluation batch: the nucleus of the distribution as it is
        {"name": "sample_s512_v32000", "op": "sample", "rows": 512, "vocab": 32000, "dtype": BF16,
         "ld": 32000, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
    ]


# ---- drawn cases -------------------------------------------------------------------------

def _log(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(("rope", "append", "attend", "attend", "sample"))
    if op == "sample":
        vocab = _log(rng, 1000, 131072)
        mixed = rng.random() < 0.4
        return {"op": op, "rows": _log(rng, 1, 512), "vocab": vocab, "dtype": rng.choice((BF16, F32)),
                "ld": vocab + rng.choice((0, 0, 1, 64)),
                "temperature": -1.0 if mixed else rng.choice((0.0, 0.7, 1.0, 1.4)),
                "top_k": -1 if mixed else rng.choice((0, 1, 20, 200)),
                "top_p": -1.0 if mixed else rng.choice((1.0, 0.5, 0.9, 0.99)),
                "min_p": -1.0 if mixed else rng.choice((0.0, 0.0, 0.05))}
    nH, nKV, d = rng.choice(HEADS + ((16, 16, 64), (8, 1, 128), (32, 8, 128), (8, 8, 96)))
    rot = rng.choice((d, d, d // 2, d // 4))
    if op == "rope":
        return {"op": op, "B": _log(rng, 1, 16), "T": _log(rng, 1, 32768), "nH": nH, "nKV": nKV, "d": d,
                "rot": rot, "interleaved": rng.random() < 0.5, "dtype": rng.choice((BF16, F32)),
                "train": rng.random() < 0.5, "pos": rng.choice((0, 0, _log(rng, 1, 1000000))),
                "factor": rng.choice((1.0, 1.0, 4.0, 32.0))}
    q_max = 1 if rng.random() < 0.5 else _log(rng, 1, 2048)
    c = {"op": op, "S": _log(rng, 1, 256), "q_max": q_max, "kv_max": q_max + _log(rng, 1, 32768), "nH": nH,
         "nKV": nKV, "d": d, "page": rng.choice((16, 32, 64, 128)), "lens": rng.randrange(1 << 20)}
    if op == "append":
        c.update(kv_max=min(c["kv_max"], q_max + 1000), rot=rot, interleaved=rng.random() < 0.5)
    return c


def _cost(c):
    """(bytes that have to move, operations, values that the plain form holds at once)."""
    w = work(c)
    held = 0
    if c["op"] == "attend":
        held = c["S"] * (c["nH"] * c["q_max"] * c["kv_max"] + 2 * c["nKV"] * c["kv_max"] * c["d"])
    elif c["op"] == "append":
        held = 2 * c["S"] * c["nKV"] * c["kv_max"] * c["d"]
    elif c["op"] == "sample":
        held = 5 * c["rows"] * c["vocab"]
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


def _dtype(c):
    return torch.float32 if c.get("dtype", BF16) == F32 else torch.bfloat16


def _frequencies(c):
    """Rotary frequencies of base 10000; a context `factor` times as long stretches the slow half of them."""
    i = torch.arange(0, c["rot"] // 2, dtype=torch.float64)
    f = 10000.0 ** (-2.0 * i / c["rot"])
    f = torch.where(i < c["rot"] // 4, f, f / c.get("factor", 1.0))
    return f.to(torch.float32).cuda()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=_dtype(c), std=1.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    def uniform(n):
        return torch.rand((n,), generator=g, device="cuda", dtype=torch.float32)

    def pick(n, values, dtype):
        at = torch.randint(0, len(values), (n,), generator=g, device="cuda")
        return torch.tensor(values, dtype=dtype, device="cuda")[at]

    s = {"case": c}
    if c["op"] == "rope":
        heads = c["nH"] + 2 * c["nKV"]
        s["freq"] = _frequencies(c)
        s["qkv"] = normal(c["B"], c["T"], heads * c["d"])
        if c["pos"]:
            start = torch.randint(0, c["pos"], (c["B"], 1), generator=g, device="cuda")
            s["pos"] = (start + torch.arange(c["T"], device="cuda")).to(torch.int32)
        if c["train"]:
            s["dQ"] = normal(c["B"], c["nH"], c["T"], c["d"], std=1e-2)
            s["dK"] = normal(c["B"], c["nKV"], c["T"], c["d"], std=1e-2)
            s["dV"] = normal(c["B"], c["nKV"], c["T"], c["d"], std=1e-2)
        return s
    if c["op"] == "sample":
        rows, V = c["rows"], c["vocab"]
        x = normal(rows, c["ld"], std=2.5)
        x[:, 7::97] += 4.0    # a trained model's logits: some tokens well above the others,
        x[:, 5::1001] = -math.inf  # some ruled out
        s["logits"] = x[:, :V]
        s["u"] = uniform(rows)
        if c["top_k"] < 0:  # each row's own
            s["temperature"] = pick(rows, (0.0, 0.6, 0.8, 1.0, 1.3), torch.float32)
            s["top_k"] = pick(rows, (0, 1, 20, 50, 1000), torch.int32)
            s["top_p"] = pick(rows, (1.0, 0.5, 0.9, 0.98), torch.float32)
            s["min_p"] = pick(rows, (0.0, 0.0, 0.02, 0.1), torch.float32)
        else:
            for n in ("temperature", "top_k", "top_p", "min_p"):
                s[n] = c[n]
        return s
    q_len, kv_len = _lens(c)
    P = c["page"]
    n_pages = [-(-n // P) for n in kv_len]
    ids = torch.randperm(sum(n_pages), generator=g, device="cuda").to(torch.int32)
    width = max(n_pages)
    used = torch.arange(width, device="cuda") < torch.tensor(n_pages, device="cuda")[:, None]
    s["pages"] = torch.zeros((c["S"], width), dtype=torch.int32, device="cuda").masked_scatter_(used, ids)
    s["k_cache"] = normal(sum(n_pages), c["nKV"], P, c["d"])
    s["v_cache"] = normal(sum(n_pages), c["nKV"], P, c["d"])
    total = sum(q_len)
    s["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0] + q_len).cumsum(0)
    s["q_start"] = starts.to(torch.int32).cuda()
    s["max_q"], s["max_kv"] = max(q_len), max(kv_len)
    s["seq"] = torch.repeat_interleave(torch.arange(c["S"]), torch.tensor(q_len)).cuda()
    s["row"] = (torch.arange(total).cuda() - starts.cuda()[s["seq"]])
    qkv = normal(total, c["nH"] + 2 * c["nKV"], c["d"])
    s["q"], s["k"], s["v"] = qkv.split((c["nH"], c["nKV"], c["nKV"]), dim=1)
    if c["op"] == "append":
        s["freq"] = _frequencies(c)
    else:
        s["q"] = s["q"].contiguous()
    return s


# ---- the framework's kernels ---------------------------------------------------------------

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "large-language-model_amd"))


def _one_each(s):
    """The start rows of the new tokens; None where every sequence has one, as a decode loop knows."""
    return None if s["max_q"] == 1 else s["q_start"]


def _run_own(s):
    import mi_gemm as mi

    c = s["case"]
    if c["op"] == "rope":
        how = dict(positions=s.get("pos"), interleaved=c["interleaved"], sync=False)
        out = mi.rope_qkv(s["qkv"], c["nH"], c["nKV"], s["freq"], **how)
        if c["train"]:
            out += (mi.rope_qkv_backward(s["dQ"], s["dK"], s["dV"], s["freq"], **how),)
        return out
    if c["op"] == "append":
        q = mi.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["pages"], s["kv_len"],
                         q_start=_one_each(s), q=s["q"], inv_freq=s["freq"], interleaved=c["interleaved"],
                         sync=False)
        return q, s["k_cache"], s["v_cache"]
    if c["op"] == "attend":
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
        o = mi.paged_attn(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["kv_len"], q_start=_one_each(s),
                          max_q_len=s["max_q"], max_kv_len=s["max_kv"], lse=lse, sync=False)
        return o, lse
    prob = torch.empty((c["rows"],), dtype=torch.float32, device="cuda")
    token = mi.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                      min_p=s["min_p"], prob=prob, sync=False)
    return token, prob


# ---- the plain forms -----------------------------------------------------------------------

def _turn(x, cos, sin, interleaved):
    """x [..., d] with its first 2 * cos.shape[-1] components rotated pair by pair."""
    n = cos.shape[-1]
    r = x[..., : 2 * n]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :n], r[..., n:])
    a, b = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, x[..., 2 * n:]), -1)


def _angles(pos, freq):
    """cos and sin of pos * freq, the angle in 64 bits."""
    t = pos.double()[..., None] * freq.double()
    return t.cos().float(), t.sin().float()


def _plain_rope(s):
    c = s["case"]
    B, T, nH, nKV, d = (c[n] for n in ("B", "T", "nH", "nKV", "d"))
    dt = s["qkv"].dtype
    pos = s["pos"] if "pos" in s else torch.arange(T, device="cuda").expand(B, T)
    cos, sin = _angles(pos, s["freq"])
    cos, sin = cos[:, None], sin[:, None]
    q, k, v = s["qkv"].view(B, T, nH + 2 * nKV, d).permute(0, 2, 1, 3).split((nH, nKV, nKV), dim=1)
    out = (_turn(q.float(), cos, sin, c["interleaved"]).to(dt), _turn(k.float(), cos, sin, c["interleaved"]).to(dt),
           v.contiguous())
    if c["train"]:
        back = torch.cat((_turn(s["dQ"].float(), cos, -sin, c["interleaved"]),
                          _turn(s["dK"].float(), cos, -sin, c["interleaved"]), s["dV"].float()), 1)
        out += (back.permute(0, 2, 1, 3).reshape(B, T, -1).to(dt),)
    return out


def _plain_append(s):
    c = s["case"]
    n = s["q_start"][1:] - s["q_start"][:-1]
    pos = (s["kv_len"] - n)[s["seq"]] + s["row"]
    page = s["pages"][s["seq"], pos // c["page"]].long()
    cos, sin = _angles(pos, s["freq"])
    cos, sin = cos[:, None], sin[:, None]
    dt = s["k_cache"].dtype
    s["k_cache"][page, :, pos % c["page"]] = _turn(s["k"].float(), cos, sin, c["interleaved"]).to(dt)
    s["v_cache"][page, :, pos % c["page"]] = s["v"]
    return _turn(s["q"].float(), cos, sin, c["interleaved"]).to(dt), s["k_cache"], s["v_cache"]


def _plain_attend(s):
    c = s["case"]
    S, nH, nKV, d, mq = c["S"], c["nH"], c["nKV"], c["d"], s["max_q"]
    n = s["q_start"][1:] - s["q_start"][:-1]

    def gathered(cache):  # [S, nKV, keys, d]
        return cache[s["pages"].long()].permute(0, 2, 1, 3, 4).reshape(S, nKV, -1, d).float()

    k, v = gathered(s["k_cache"]), gathered(s["v_cache"])
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


def _plain_sample(s):
    c = s["case"]
    x = s["logits"].float()
    rows, V = x.shape

    def each(v):  # a row's setting, a 32-bit number
        return v[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), v, device="cuda")

    t, p, low = (each(s[n]).double() for n in ("temperature", "top_p", "min_p"))
    k = each(s["top_k"])
    x, order = x.sort(dim=-1, descending=True, stable=True)
    x = x.double()
    w = ((x - x[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    rank = torch.arange(V, device="cuda")
    w = w * (rank < torch.where(t > 0, torch.where(k > 0, k, V), 1))
    before = w.cumsum(-1) - w
    w = w * ((before < p * w.sum(-1, keepdim=True)) | (p >= 1) | (rank == 0)) * (w >= low)
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.sum(-1, keepdim=True)
    token = (w.cumsum(-1) <= s["u"].double()[:, None] * total).sum(-1, keepdim=True)
    return token.squeeze(1).to(torch.int32), (w.gather(1, token) / total).squeeze(1).float()


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "rope":
        return _plain_rope(state)
    if op == "append":
        return _plain_append(state)
    return _plain_attend(state) if op == "attend" else _plain_sample(state)


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    c = case
    size = 4 if c.get("dtype", BF16) == F32 else 2
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * size + 12), "flops": 4 * c["rows"] * c["vocab"]}
    heads = c["nH"] + 2 * c["nKV"]
    if c["op"] == "rope":
        n = c["B"] * c["T"] * heads * c["d"] * (2 if c["train"] else 1)
        return {"bytes": 2 * n * size, "flops": 3 * n}
    q_len, kv_len = _lens(c)
    if c["op"] == "append":
        n = sum(q_len) * heads * c["d"]
        return {"bytes": 2 * n * size, "flops": 3 * n}
    seen = sum(n * k - n * (n - 1) // 2 for n, k in zip(q_len, kv_len))
    return {"bytes": size * c["d"] * (2 * c["nKV"] * sum(kv_len) + 2 * c["nH"] * sum(q_len)) + 4 * c["nH"] * sum(q_len),
            "flops": 4 * c["nH"] * c["d"] * seen}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _rotated(x, pos, freq, interleaved, sign=1.0):
    """x [tokens, heads, d] as complex pairs times exp(i sign pos freq), 64 bits."""
    n = freq.numel()
    x = x.double().clone()
    z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), sign * pos.double()[:, None] * freq.double())
    re, im = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y = torch.complex(x[..., re], x[..., im]) * z[:, None]
    x[..., re], x[..., im] = y.real, y.imag
    return x


def _exact_rope(s):
    c = s["case"]
    B, T, nH, nKV, d = (c[n] for n in ("B", "T", "nH", "nKV", "d"))
    out = [[], [], [], []]
    for b in range(B):
        pos = s["pos"][b] if "pos" in s else torch.arange(T, device="cuda")
        x = s["qkv"][b].view(T, -1, d)
        y = _rotated(x[:, : nH + nKV], pos, s["freq"], c["interleaved"])
        out[0].append(y[:, :nH].transpose(0, 1))
        out[1].append(y[:, nH:].transpose(0, 1))
        out[2].append(x[:, nH + nKV:].transpose(0, 1).double())
        if c["train"]:
            y = torch.cat((s["dQ"][b], s["dK"][b])).transpose(0, 1)
            y = _rotated(y, pos, s["freq"], c["interleaved"], -1.0)
            out[3].append(torch.cat((y, s["dV"][b].transpose(0, 1).double()), 1).reshape(T, -1))
    return tuple(torch.stack(x) for x in out if x)


def _exact_append(s):
    c = s["case"]
    q, k, v = [], s["k_cache"].double(), s["v_cache"].double()
    starts, lens, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["pages"].tolist()
    for i in range(c["S"]):
        a, b = starts[i], starts[i + 1]
        first = lens[i] - (b - a)
        pos = torch.arange(first, lens[i], device="cuda")
        q.append(_rotated(s["q"][a:b], pos, s["freq"], c["interleaved"]))
        new = _rotated(s["k"][a:b], pos, s["freq"], c["interleaved"])
        for page in range(first // c["page"], (lens[i] - 1) // c["page"] + 1):
            lo, hi = max(first, page * c["page"]), min(lens[i], (page + 1) * c["page"])
            at = slice(lo - page * c["page"], hi - page * c["page"])
            k[table[i][page], :, at] = new[lo - first:hi - first].transpose(0, 1)
            v[table[i][page], :, at] = s["v"][a + lo - first:a + hi - first].transpose(0, 1).double()
    return torch.cat(q), k, v


def _exact_attend(s):
    c = s["case"]
    g, d = c["nH"] // c["nKV"], c["d"]
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    for i in range(c["S"]):
        a, b, n = starts[i], starts[i + 1], lens[i]
        ids = s["pages"][i, : -(-n // c["page"])].long()
        hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n - (b - a), n, device="cuda")[:, None]
        for h in range(c["nKV"]):
            k, v = (t[ids, h].reshape(-1, d)[:n].double() for t in (s["k_cache"], s["v_cache"]))
            for j in range(h * g, h * g + g):
                x = torch.mm(s["q"][a:b, j].double(), k.t()) / math.sqrt(d)
                x = torch.where(hidden, -math.inf, x)
                lse[a:b, j] = torch.logsumexp(x, -1)
                o[a:b, j] = torch.mm((x - lse[a:b, j, None]).exp(), v)
    return o, lse


def _exact_sample(s):
    x, u = s["logits"].double().cpu().numpy(), s["u"].tolist()
    rows, V = x.shape
    of = {n: (s[n].tolist() if isinstance(s[n], torch.Tensor) else [float(np.float32(s[n]))] * rows)
          for n in ("temperature", "top_k", "top_p", "min_p")}
    tokens, probs = [], []
    for r in range(rows):
        order = np.lexsort((np.arange(V), -x[r]))
        t, k = of["temperature"][r], int(of["top_k"][r])
        n = 1 if t <= 0 else min(k, V) if k > 0 else V
        w = np.exp((x[r, order[:n]] - x[r, order[0]]) / (t if t > 0 else 1.0))
        if of["top_p"][r] < 1:
            mass = np.cumsum(w)
            n = max(1, int(np.searchsorted(mass[:-1], of["top_p"][r] * mass[-1], side="left")) + 1)
        n = min(n, int((w[:n] >= of["min_p"][r]).sum()))
        kept = np.sort(order[:n])
        place = {int(v): i for i, v in enumerate(order[:n])}
        w = w[[place[int(v)] for v in kept]]
        mass = np.cumsum(w)
        at = min(n - 1, int(np.searchsorted(mass, u[r] * mass[-1], side="right")))
        tokens.append(int(kept[at]))
        probs.append(w[at] / mass[-1])
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _exact_rope(s)
    if op == "append":
        return _exact_append(s)
    return _exact_attend(s) if op == "attend" else _exact_sample(s)
