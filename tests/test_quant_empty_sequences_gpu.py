"""Batches of which most sequences have no new token, as a padded batch of a serving loop: the append and the reading
back over a cache of 8 or 4 bits."""
import numpy as np
import pytest
from quant_numbers import pack, quantise, values

pytestmark = pytest.mark.gpu


def i32(x):
    import torch

    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def batch(q, P=16):
    """(pages, kv_len, q_start, page, slot): sequences of q new tokens and none before, of pages of their own."""
    q = np.asarray(q)
    need = -(-q // P)
    first = np.concatenate([[0], np.cumsum(need)])
    width = int(need.max())
    table = np.where(np.arange(width) < need[:, None], first[:-1, None] + np.arange(width), -1)
    starts = np.concatenate([[0], np.cumsum(q)])
    seq = np.repeat(np.arange(len(q)), q)
    pos = np.arange(len(seq)) - starts[seq]
    return i32(table), i32(q), i32(starts), table[seq, pos // P], pos % P, int(first[-1])


def rows(n, seed):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((n, 2, 64), generator=g, device="cuda").to(torch.bfloat16)


# workgroups take several tokens each where there are a thousand and more, up to 16 and 64 of them
LENGTHS = {
    "front": [0] * 5000 + [3, 4000],
    "between": [1999] + [0] * 4000 + [2003],
    "many gaps": ([37] + [0] * 67) * 270 + [5],
    "gaps of all sizes": sum(([29] + [0] * n for n in range(130)), []),
    "behind": [2000, 1501] + [0] * 3000,
    "powers": sum(([61] + [0] * (2 ** n + d) for n in range(1, 12) for d in (-1, 0, 1)), []),
    "several in one workgroup": sum(([1, 0, 2] + [0] * (n % 70) + [1, 1] for n in range(2500)), []),
    "few tokens": [7] + [0] * 4000 + [3, 1],
}


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("name", LENGTHS)
def test_tokens_find_their_sequences(mi, dev, bits, name):
    import torch

    pages, kv, start, page, slot, num = batch(LENGTHS[name])
    n = len(slot)
    c = mi.quant_cache(num, 2, 16, 64, bits)
    k, v = rows(n + 2, 1), rows(n + 2, 2)
    mi.kv_append_quant(k, v, c, pages, kv, q_start=start)
    for x, codes, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want, byte = quantise(x[:n].double().cpu().numpy(), bits)
        assert np.array_equal(codes.cpu().numpy()[page, :, slot], pack(want, bits))
        assert np.array_equal(scale.cpu().numpy()[page, :, slot], byte)
    out = [torch.full((n + 2, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    mi.kv_read_quant(c, pages, kv, q_start=start, k_out=out[0], v_out=out[1])
    for o, x in zip(out, (k, v)):
        assert np.array_equal(o[:n].double().cpu().numpy(), values(*quantise(x[:n].double().cpu().numpy(), bits), bits))
        assert (o[n:] == 3.0).all()


def test_empty_sequences_cost_no_walk(mi, dev):
    """A hundred thousand of them between two prompts: less than twenty times what the prompts alone take, where a step
    for each would take thousands of times as long."""
    import torch

    def time_of(q):
        pages, kv, start, _, _, num = batch(q)
        n = sum(q)
        c, k = mi.quant_cache(num, 2, 16, 64, 4), rows(n, 1)
        outs = [torch.empty_like(k) for _ in "kv"]

        def step():
            mi.kv_append_quant(k, k, c, pages, kv, q_start=start, sync=False)
            mi.kv_read_quant(c, pages, kv, q_start=start, k_out=outs[0], v_out=outs[1], sync=False)

        step()
        torch.cuda.synchronize()
        took = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                step()
            b.record()
            b.synchronize()
            took.append(a.elapsed_time(b))
        return min(took)

    assert time_of([2001] + [0] * 100000 + [2002]) < 20 * time_of([2001, 2002])
