"""What mi_rope, mi_kv_append, mi_paged_attn and mi_sample refuse, on the host: no case reaches a GPU."""
import ctypes
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P16 = 1 << 20  # a fake device address


def _msg(mi):
    return mi.load_library().mi_last_error().decode()


def rotary(mi, **kw):
    r = mi.MiRotary()
    r.inv_freq, r.rot_dim, r.scale = P16, 64, 1.0
    for n, v in kw.items():
        setattr(r, n, v)
    return r


def part(mi, **kw):
    a = mi.MiRopePart()
    a.src, a.dst, a.heads, a.rotate = P16, 2 * P16, 4, 1
    a.src_b = a.dst_b = 1024
    a.src_t = a.dst_t = 256
    a.src_h = a.dst_h = 64
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def rope(mi, parts=None, n=None, B=2, T=4, d=64, rot=None, dtype=1, **kw):
    parts = parts if parts is not None else [part(mi, **kw)]
    arr = (mi.MiRopePart * max(1, len(parts)))(*parts)
    r = rot if rot is not None else rotary(mi)
    return mi.load_library().mi_rope(None, arr, len(parts) if n is None else n, B, T, d, ctypes.byref(r), 0, dtype)


def test_rope(mi):
    L = mi.load_library()
    assert rope(mi, B=0) == 0 and rope(mi, T=0) == 0 and rope(mi, d=0) == 0 and rope(mi, heads=0) == 0
    assert rope(mi, B=-1) == 1 and rope(mi, n=0) == 1 and rope(mi, n=5) == 1
    assert rope(mi, dtype=2) == 4
    assert rope(mi, B=1 << 20, T=1 << 20) == 1
    assert rope(mi, d=63) == 5 and rope(mi, d=2048) == 5
    assert rope(mi, src=0) == 3 and rope(mi, dst=0) == 3
    assert rope(mi, src=P16 + 1) == 5 and rope(mi, src=P16 + 2, dtype=0) == 5
    assert rope(mi, heads=-1) == 1 and "part 0" in _msg(mi)
    assert rope(mi, dst_t=0) == 2 and rope(mi, dst_h=0) == 2 and rope(mi, dst_b=0) == 2
    assert rope(mi, dst=P16, dst_t=512) == 5 and "in place" in _msg(mi)
    assert rope(mi, reserved=1) == 1
    assert rope(mi, parts=[part(mi), part(mi, src=0)]) == 3 and "part 1" in _msg(mi)
    for kw, st in ((dict(rot_dim=0), 1), (dict(rot_dim=63), 1), (dict(rot_dim=66), 1), (dict(inv_freq=0), 3),
                   (dict(inv_freq=P16 + 2), 5), (dict(positions=P16 + 1), 5), (dict(scale=float("inf")), 5),
                   (dict(scale=float("nan")), 5), (dict(interleaved=2), 1)):
        assert rope(mi, rot=rotary(mi, **kw)) == st, kw
    assert L.mi_rope(None, None, 1, 1, 1, 64, ctypes.byref(rotary(mi)), 0, 1) == 3
    assert L.mi_rope(None, (mi.MiRopePart * 1)(part(mi)), 1, 1, 1, 64, None, 0, 1) == 3


def cache(mi, **kw):
    c = mi.MiPagedCache()
    c.k, c.v, c.num_pages, c.page_size, c.n_kv, c.head_dim = P16, 2 * P16, 10, 16, 2, 64
    c.page_stride, c.head_stride, c.slot_stride = 2048, 1024, 64
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def seqs(mi, **kw):
    s = mi.MiPagedSeqs()
    s.n_seqs, s.total_q, s.q_start, s.kv_len, s.pages, s.max_pages, s.pages_ld = 3, 5, P16, P16, P16, 4, 4
    for n, v in kw.items():
        setattr(s, n, v)
    return s


def append(mi, c=None, s=None, r=None, q=P16, q_out=P16, k=P16, v=P16, nH=4, q_t=256, qo_t=256, qo_h=64):
    c, s = c or cache(mi), s or seqs(mi)
    return mi.load_library().mi_kv_append(None, q, q_t, 64, q_out, qo_t, qo_h, nH, k, 128, 64, v, 128, 64,
                                          ctypes.byref(c), ctypes.byref(s), ctypes.byref(r) if r else None)


def attend(mi, c=None, s=None, q=P16, o=P16, q_t=256, q_h=64, o_t=256, o_h=64, lse=None, nH=4, mq=5, mk=64, scale=0.1,
           ws=None, wsb=0):
    c, s = c or cache(mi), s or seqs(mi)
    return mi.load_library().mi_paged_attn(None, q, q_t, q_h, o, o_t, o_h, lse, nH, ctypes.byref(c), ctypes.byref(s), mq,
                                           mk, 1, scale, ws, wsb)


@pytest.mark.parametrize("call", [append, attend])
def test_paged_tables(mi, call):
    for kw in (dict(n_seqs=0), dict(total_q=0)):
        assert call(mi, s=seqs(mi, **kw)) == 0
    for kw, st in ((dict(n_seqs=-1), 1), (dict(total_q=-1), 1), (dict(total_q=1 << 31), 1), (dict(max_pages=-1), 1),
                   (dict(q_start=0), 1), (dict(pages_ld=3), 2), (dict(kv_len=0), 3), (dict(pages=0), 3),
                   (dict(kv_len=P16 + 2), 5), (dict(pages=P16 + 1), 5), (dict(q_start=P16 + 1), 5)):
        assert call(mi, s=seqs(mi, **kw)) == st, kw
    for kw, st in ((dict(page_size=0), 1), (dict(page_size=24), 1), (dict(page_size=1 << 21), 1), (dict(num_pages=-1), 1),
                   (dict(k=0), 3), (dict(v=0), 3), (dict(k=P16 + 8), 5), (dict(head_dim=60), 5), (dict(head_dim=0), 5),
                   (dict(slot_stride=60), 5), (dict(slot_stride=56), 2), (dict(head_stride=0), 2), (dict(page_stride=8), 2),
                   (dict(page_stride=-2048), 2)):
        assert call(mi, c=cache(mi, **kw)) == st, kw


def test_append(mi):
    assert append(mi, q_out=0) == 3 and append(mi, k=0) == 3 and append(mi, v=0) == 3
    assert append(mi, q=P16 + 1) == 5 and append(mi, nH=-1) == 1
    assert append(mi, qo_t=0) == 2 and append(mi, qo_h=0) == 2
    assert append(mi, qo_t=512) == 5 and "in place" in _msg(mi)
    assert append(mi, r=rotary(mi, rot_dim=66)) == 1


def test_attention(mi):
    assert attend(mi, nH=0) == 0
    assert attend(mi, mq=-1) == 1 and attend(mi, mk=-1) == 1
    assert attend(mi, nH=5) == 1 and attend(mi, c=cache(mi, n_kv=0)) == 1
    assert attend(mi, c=cache(mi, head_dim=136, slot_stride=136, head_stride=2176, page_stride=4352)) == 5
    assert attend(mi, q=0) == 3 and attend(mi, o=0) == 3
    assert attend(mi, q=P16 + 8) == 5 and attend(mi, o=P16 + 2) == 5 and attend(mi, lse=P16 + 2) == 5
    assert attend(mi, ws=P16 + 4, wsb=64) == 5
    assert attend(mi, q_t=260) == 5 and attend(mi, o_h=60) == 5
    assert attend(mi, o_t=0) == 2 and attend(mi, o_h=8) == 2
    assert attend(mi, o_t=512) == 5 and "in place" in _msg(mi)
    for scale in (0.0, -1.0, 3e38, float("inf"), float("nan")):
        assert attend(mi, scale=scale) == 5


def sample(mi, logits=P16, dtype=1, ld=100, rows=3, V=100, u=P16, tok=P16, prob=None, how=None):
    h = mi.MiSampling()
    for n, v in (how or {}).items():
        setattr(h, n, v)
    return mi.load_library().mi_sample(None, logits, dtype, ld, rows, V, ctypes.byref(h), u, tok, prob)


def test_sample(mi):
    assert sample(mi, rows=0) == 0
    assert sample(mi, rows=-1) == 1 and sample(mi, V=-1) == 1 and sample(mi, V=0) == 1
    assert sample(mi, V=(1 << 24) + 1, ld=1 << 25) == 1 and sample(mi, rows=1 << 31) == 1
    assert sample(mi, dtype=2) == 4
    assert sample(mi, ld=99) == 2
    assert sample(mi, logits=0) == 3 and sample(mi, u=0) == 3 and sample(mi, tok=0) == 3
    assert sample(mi, logits=P16 + 1) == 5 and sample(mi, logits=P16 + 2, dtype=0) == 5
    assert sample(mi, u=P16 + 2) == 5 and sample(mi, tok=P16 + 1) == 5 and sample(mi, prob=P16 + 3) == 5
    for n in ("temperature", "top_k", "top_p", "min_p"):
        assert sample(mi, how={n: P16 + 2}) == 5
    assert mi.load_library().mi_sample(None, P16, 1, 100, 3, 100, None, P16, P16, None) == 3


def test_no_device(mi):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the calls would run on the fake addresses")
    assert rope(mi) == 8 and append(mi, r=rotary(mi)) == 8 and attend(mi) == 8 and sample(mi) == 8


def test_workspace_query(mi):
    assert mi.paged_attn_workspace_size(16, 4, 128, 0, 0, 1, 100) == 0
    assert mi.paged_attn_workspace_size(16, 4, 128, 4, 4096, 1024, 4096) >= 0


@pytest.mark.parametrize("name,cls", [("mi_rotary", "MiRotary"), ("mi_rope_part", "MiRopePart"),
                                      ("mi_paged_cache", "MiPagedCache"), ("mi_paged_seqs", "MiPagedSeqs"),
                                      ("mi_sampling", "MiSampling")])
def test_struct_layouts(mi, name, cls):
    """The ctypes mirrors have the header's fields, in order, of the header's types."""
    hdr = open(os.path.join(ROOT, "include", "mi_gemm.h")).read()
    body = re.sub(r"/\*.*?\*/", "", hdr[hdr.index(f"typedef struct {name} {{") + len(f"typedef struct {name} {{"):
                                        hdr.index(f"}} {name};")], flags=re.S)
    want = []
    for line in body.split(";"):
        m = re.match(r"\s*(?:const )?(void|float|int32_t|int64_t)\s*(.*)", line.strip())
        if m:
            for n in m.group(2).split(","):
                ptr = "*" in n
                want.append((n.strip(" *"), ctypes.c_void_p if ptr else
                             {"float": ctypes.c_float, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64}[m.group(1)]))
    assert [(n, t) for n, t in getattr(mi, cls)._fields_] == want


def test_packed_structs_match_the_mirrors(mi):
    import struct

    for pack, cls in ((mi._PACK_PART, mi.MiRopePart), (mi._PACK_ROTARY, mi.MiRotary), (mi._PACK_CACHE, mi.MiPagedCache),
                      (mi._PACK_SEQS, mi.MiPagedSeqs), (mi._PACK_SAMPLING, mi.MiSampling)):
        kinds = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}
        fmt = "@" + "".join(kinds[t] for _, t in cls._fields_)
        assert pack.__self__.format == fmt and struct.calcsize(fmt) == ctypes.sizeof(cls)
        raw = pack(*range(1, len(fmt)))
        got = cls.from_buffer_copy(raw)
        assert [getattr(got, n) for n, _ in cls._fields_] == list(range(1, len(fmt)))


def test_python_refusals(mi):
    """The Python layer's own checks, on CPU tensors, which it refuses last."""
    import torch

    bf, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    f = torch.ones(32)
    x = torch.zeros(2, 3, 4, 64, dtype=bf)
    V = pytest.raises(ValueError)
    with V as e:
        mi.rope(x, f)
    assert "GPU" in str(e.value)
    for bad in (dict(layout="btdh"), dict(out=x[:1])):
        with pytest.raises(ValueError):
            mi.rope(x, f, **bad)
    with pytest.raises(ValueError):
        mi.rope_qkv(torch.zeros(1, 2, 100, dtype=bf), 3, 2, f)
    with pytest.raises(ValueError):
        mi.rope_qkv_backward(x, x, x[:1], f)
    k = torch.zeros(5, 2, 64, dtype=bf)
    c = torch.zeros(6, 2, 16, 64, dtype=bf)
    pages, n = torch.zeros(5, 3, dtype=i32), torch.ones(5, dtype=i32)
    q = torch.zeros(5, 4, 64, dtype=bf)
    good = dict(k=k, v=k, k_cache=c, v_cache=c, pages=pages, kv_len=n)
    for bad, word in ((dict(), "GPU"), (dict(v=k[:4]), "tokens"), (dict(k_cache=c.float(), v_cache=c.float()), "bf16"),
                      (dict(pages=pages.long()), "pages"), (dict(kv_len=n[:4]), "rows"), (dict(v_cache=c[:5]), "strides"),
                      (dict(q_start=n), "entries"), (dict(pages=pages[:, ::2]), "contiguous"),
                      (dict(pages=pages[:3], kv_len=n[:3]), "q_start is needed")):
        with pytest.raises(ValueError, match=word):
            mi.kv_append(**{**good, **bad})
    for args, kw, word in (((q[0], c, c, pages, n), {}, "tokens"), ((q, c, c, pages, n), {}, "GPU"),
                           ((q, c, c[:, :1], pages, n), {}, "strides")):
        with pytest.raises(ValueError, match=word):
            mi.paged_attn(*args, **kw)
    lg, u = torch.zeros(3, 10), torch.zeros(3)
    for args, kw, word in (((lg, u), {}, "GPU"), ((lg[0], u), {}, "rows"), ((lg.t(), u), {}, "contiguous"),
                           ((lg, u[:2]), {}, "u must"), ((lg, u), dict(top_k=u), "top_k"), ((lg, u.double()), {}, "u must"),
                           ((lg, u), dict(prob=u[:1]), "prob"), ((lg, u), dict(out=u), "out")):
        with pytest.raises(ValueError, match=word):
            mi.sample(*args, **kw)
