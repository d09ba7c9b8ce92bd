"""What the calls over a cache of 8 or 4 bits refuse, on the host, and their structs: no case reaches a GPU."""
import ctypes

import pytest
from test_serve_abi import P16, rotary, seqs, test_struct_layouts as check_layout
from test_serve_launches import ask  # noqa: F401  (a fixture)


def _msg(mi):
    return mi.load_library().mi_last_error().decode()


def cache(mi, **kw):
    c = mi.MiQuantCache()
    c.k, c.v, c.k_scale, c.v_scale = P16, 2 * P16, 3 * P16 + 1, 4 * P16 + 3
    c.num_pages, c.page_size, c.n_kv, c.head_dim, c.format = 10, 16, 2, 64, 1
    c.page_stride, c.head_stride, c.slot_stride = 1024, 512, 32
    c.scale_page_stride, c.scale_head_stride, c.scale_slot_stride = 66, 33, 2
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def append(mi, c=None, s=None, r=None, q=P16, q_out=P16, k=P16, v=P16, nH=4, q_t=256, qo_t=256, qo_h=64):
    c, s = c or cache(mi), s or seqs(mi)
    return mi.load_library().mi_kv_append_quant(None, q, q_t, 64, q_out, qo_t, qo_h, nH, k, 128, 64, v, 128, 64,
                                                ctypes.byref(c), ctypes.byref(s), ctypes.byref(r) if r else None)


def read(mi, c=None, s=None, k=P16, v=P16, k_t=128, k_h=64, v_t=128, v_h=64, dtype=1):
    c, s = c or cache(mi), s or seqs(mi)
    return mi.load_library().mi_kv_read_quant(None, k, k_t, k_h, v, v_t, v_h, dtype, ctypes.byref(c), ctypes.byref(s))


def attend(mi, c=None, s=None, q=P16, o=P16, q_t=256, q_h=64, o_t=256, o_h=64, lse=None, nH=4, mq=5, mk=64, scale=0.1,
           ws=None, wsb=0):
    c, s = c or cache(mi), s or seqs(mi)
    return mi.load_library().mi_paged_attn_quant(None, q, q_t, q_h, o, o_t, o_h, lse, nH, ctypes.byref(c), ctypes.byref(s),
                                                 mq, mk, 1, scale, ws, wsb)


@pytest.mark.parametrize("call", [append, read, attend])
def test_tables_and_cache(mi, call):
    for kw in (dict(n_seqs=0), dict(total_q=0)):
        assert call(mi, s=seqs(mi, **kw)) == 0
    for kw, st in ((dict(n_seqs=-1), 1), (dict(total_q=-1), 1), (dict(total_q=1 << 31), 1), (dict(max_pages=-1), 1),
                   (dict(q_start=0), 1), (dict(pages_ld=3), 2), (dict(kv_len=0), 3), (dict(pages=0), 3),
                   (dict(kv_len=P16 + 2), 5), (dict(pages=P16 + 1), 5), (dict(q_start=P16 + 1), 5)):
        assert call(mi, s=seqs(mi, **kw)) == st, kw
    for kw, st in ((dict(page_size=0), 1), (dict(page_size=24), 1), (dict(page_size=1 << 21), 1), (dict(num_pages=-1), 1),
                   (dict(k=0), 3), (dict(v=0), 3), (dict(k_scale=0), 3), (dict(v_scale=0), 3), (dict(k=P16 + 8), 5),
                   (dict(v=P16 + 4), 5), (dict(head_dim=48), 5), (dict(head_dim=0), 5), (dict(slot_stride=40), 5),
                   (dict(slot_stride=16), 2), (dict(slot_stride=-32), 2), (dict(head_stride=0), 2), (dict(page_stride=16), 2),
                   (dict(format=2), 4), (dict(format=-1), 4), (dict(reserved=1), 1), (dict(format=0), 2),
                   (dict(scale_slot_stride=1), 2), (dict(scale_head_stride=0), 2), (dict(scale_page_stride=-66), 2)):
        assert call(mi, c=cache(mi, **kw)) == st, kw
    lib = mi.load_library()
    assert lib.mi_kv_read_quant(None, P16, 128, 64, P16, 128, 64, 1, None, None) == 3


def test_append(mi):
    assert append(mi, q_out=0) == 3 and append(mi, k=0) == 3 and append(mi, v=0) == 3
    assert append(mi, q=P16 + 1) == 5 and append(mi, nH=-1) == 1 and append(mi, nH=65537) == 1
    assert append(mi, qo_t=0) == 2 and append(mi, qo_h=0) == 2
    assert append(mi, qo_t=512) == 5 and "in place" in _msg(mi)
    for kw, st in ((dict(rot_dim=66), 1), (dict(rot_dim=0), 1), (dict(rot_dim=63), 1), (dict(inv_freq=0), 3),
                   (dict(scale=float("nan")), 5), (dict(interleaved=2), 1), (dict(positions=P16 + 2), 5)):
        assert append(mi, r=rotary(mi, **kw)) == st, kw
    wide = dict(head_dim=1056, slot_stride=528, head_stride=16 * 528, page_stride=32 * 528, scale_slot_stride=33,
                scale_head_stride=16 * 33, scale_page_stride=32 * 33)
    assert append(mi, c=cache(mi, **wide)) == 5 and read(mi, c=cache(mi, **wide), k_t=4224, k_h=1056, v_t=4224, v_h=1056) == 5


def test_read(mi):
    assert read(mi, k=0, v=0) == 0
    assert read(mi, dtype=2) == 4 and read(mi, dtype=-1) == 4
    assert read(mi, k=P16 + 1) == 5 and read(mi, v=P16 + 2, dtype=0) == 5
    assert read(mi, k_t=63) == 2 and "of k" in _msg(mi)
    assert read(mi, v_h=32) == 2 and "of v" in _msg(mi)


def test_read_of_k_and_v_into_one_place(mi):
    import torch

    c = mi.quant_cache(6, 2, 16, 64, 4, device="cpu")
    tables = torch.zeros(5, 3, dtype=torch.int32), torch.ones(5, dtype=torch.int32)
    out = torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="same memory"):
        mi.kv_read_quant(c, *tables, k_out=out[:, :2], v_out=out[:, :2])
    with pytest.raises(ValueError, match="GPU"):
        mi.kv_read_quant(c, *tables, k_out=out[:, :2], v_out=out[:, 2:])


def test_attention(mi):
    assert attend(mi, nH=0) == 0
    assert attend(mi, mq=-1) == 1 and attend(mi, mk=-1) == 1
    assert attend(mi, nH=5) == 1 and attend(mi, c=cache(mi, n_kv=0)) == 1
    assert attend(mi, c=cache(mi, head_dim=160, slot_stride=80, head_stride=1280, page_stride=2560, scale_slot_stride=5,
                              scale_head_stride=80, scale_page_stride=160), q_t=1024, q_h=160, o_t=1024, o_h=160) == 5
    assert attend(mi, q=0) == 3 and attend(mi, o=0) == 3
    assert attend(mi, q=P16 + 8) == 5 and attend(mi, o=P16 + 2) == 5 and attend(mi, lse=P16 + 2) == 5
    assert attend(mi, ws=P16 + 4, wsb=64) == 5
    assert attend(mi, q_t=260) == 5 and attend(mi, o_h=60) == 5
    assert attend(mi, o_t=0) == 2 and attend(mi, o_h=8) == 2
    assert attend(mi, o_t=512) == 5 and "in place" in _msg(mi)
    for scale in (0.0, -1.0, 3e38, float("inf"), float("nan")):
        assert attend(mi, scale=scale) == 5


def test_a_stride_that_no_step_takes_may_be_anything(mi):
    """One page, one head or one slot: nothing is stepped over."""
    for kw in (dict(num_pages=1, page_stride=5), dict(n_kv=1, head_stride=7), dict(page_size=1, slot_stride=3),
               dict(num_pages=1, scale_page_stride=0), dict(n_kv=1, scale_head_stride=0),
               dict(page_size=1, scale_slot_stride=-1)):
        assert read(mi, c=cache(mi, **kw), k=0, v=0) == 0, kw


def test_no_device(mi):
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the calls would run on the fake addresses")
    assert append(mi, r=rotary(mi)) == 8 and read(mi) == 8 and attend(mi) == 8


def test_struct(mi):
    check_layout(mi, "mi_quant_cache", "MiQuantCache")
    kinds = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i"}
    fmt = "@" + "".join(kinds[t] for _, t in mi.MiQuantCache._fields_)
    assert mi._PACK_QUANT.__self__.format == fmt
    got = mi.MiQuantCache.from_buffer_copy(mi._PACK_QUANT(*range(1, len(fmt))))
    assert [getattr(got, n) for n, _ in mi.MiQuantCache._fields_] == list(range(1, len(fmt)))


def test_workspace_query(mi):
    f = mi.paged_attn_quant_workspace_size
    assert f(16, 4, 128, 0, 0, 1, 100) == 0 and f(16, 3, 128, 4, 4, 1, 100) == 0
    assert f(16, 4, 128, 1, 1, 1, 64) == 0  # one piece, nothing to join
    assert f(16, 4, 128, 1, 1, 1, 32768) > 0 and f(16, 4, 128, 4, 4096, 1024, 4096) >= 0


@pytest.mark.parametrize("tokens", [1, 300, 2 ** 28 + 5, 2 ** 31 - 1])
@pytest.mark.parametrize("call", ["append", "read"])
def test_launches_of_many_tokens(ask, call, tokens):  # noqa: F811
    """A launch counts its threads in 32 bits: calls of more go out in several."""
    st, got = ask(f"__import__('test_quant_abi').{call}(mi, s=t.seqs(mi, n_seqs=3, total_q={tokens})), launches()")
    assert st == 0 and len(got) >= 1
    assert all(g * b < 2 ** 32 for g, b, _ in got)
    if tokens == 1:
        assert [g for g, _, _ in got] == [1]
    else:
        each = -(-tokens // sum(g for g, _, _ in got))
        assert 1 <= each <= 64 and len(got) == -(-(-(-tokens // each)) // (2 ** 24 - 1))


def test_python_refusals(mi):
    """The Python layer's own checks, on CPU tensors, which it refuses last."""
    import torch

    bf, i32 = torch.bfloat16, torch.int32
    k, q = torch.zeros(5, 2, 64, dtype=bf), torch.zeros(5, 4, 64, dtype=bf)
    pages, n = torch.zeros(5, 3, dtype=i32), torch.ones(5, dtype=i32)
    c = mi.quant_cache(6, 2, 16, 64, 4, device="cpu")
    assert c.k.shape == (6, 2, 16, 32) and c.v_scale.shape == (6, 2, 16, 2)
    assert mi.quant_cache(6, 2, 16, 64, device="cpu").v.shape == (6, 2, 16, 64)
    for bits, d in ((5, 64), (4, 48), (8, 0)):
        with pytest.raises(ValueError, match="bits"):
            mi.quant_cache(1, 1, 1, d, bits, device="cpu")
    good = dict(k=k, v=k, cache=c, pages=pages, kv_len=n)
    f = torch.ones(32)
    for bad, word in ((dict(), "GPU"), (dict(v=k[:4]), "tokens"), (dict(k=k.float(), v=k.float()), "bf16"),
                      (dict(pages=pages.long()), "pages"), (dict(kv_len=n[:4]), "rows"),
                      (dict(cache=c._replace(v=c.v[:5])), "strides"), (dict(cache=c._replace(k_scale=c.k_scale[:, :1])), "strides"),
                      (dict(cache=c._replace(k=c.k.view(torch.int8), v=c.v.view(torch.int8))), "uint8"),
                      (dict(cache=mi.QuantCache(c.k[..., :16], c.v[..., :16], c.k_scale, c.v_scale)), "groups"),
                      (dict(cache=mi.quant_cache(6, 2, 16, 32, 4, device="cpu")), "heads"),
                      (dict(q_start=n), "entries"), (dict(pages=pages[:, ::2]), "contiguous"),
                      (dict(pages=pages[:3], kv_len=n[:3]), "q_start is needed"), (dict(q=q[:3]), "q must"),
                      (dict(q=q, q_out=q.float()), "q_out"), (dict(inv_freq=f.double()), "GPU"),
                      (dict(positions=n), "GPU")):
        with pytest.raises(ValueError, match=word):
            mi.kv_append_quant(**{**good, **bad})
    args = (c, pages, n)
    start = torch.zeros(6, dtype=i32)
    for kw, word in ((dict(), "GPU"), (dict(parts="q"), "parts"), (dict(q_start=start), "rows"), (dict(rows=4), "q_start is needed"),
                     (dict(dtype=torch.float16), "."), (dict(k_out=k.float()), "v_out|GPU"), (dict(k_out=k, dtype=torch.float32), "k_out"),
                     (dict(k_out=k[:, :1]), "k_out"), (dict(k_out=k, v_out=k.float()), "v_out"),
                     (dict(k_out=k.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous")):
        with pytest.raises((ValueError, KeyError, TypeError), match=word):
            mi.kv_read_quant(*args, **kw)
    for a, kw, word in (((q[0], *args), {}, "tokens"), ((q, *args), {}, "GPU"), ((q[..., :32], *args), {}, "heads of"),
                        ((q, *args), dict(lse=torch.zeros(5, 3)), "lse"), ((q, *args), dict(out=q.float()), "out"),
                        ((q, *args), dict(workspace=torch.zeros(64)[::2]), "workspace")):
        with pytest.raises(ValueError, match=word):
            mi.paged_attn_quant(*a, **kw)
