"""Reading a cache of 8 or 4 bits back into tensors that the caller gives: what the Python layer refuses, without a GPU."""
import pytest


@pytest.fixture
def args(mi):
    import torch

    cache = mi.quant_cache(6, 2, 16, 64, 4, device="cpu")
    return cache, torch.zeros(5, 3, dtype=torch.int32), torch.ones(5, dtype=torch.int32)


def outs(views):
    """K and V views of one buffer: (strides, offset) each."""
    import torch

    base = torch.zeros(20000, dtype=torch.bfloat16)
    return [torch.as_strided(base, (5, 2, 64), (t, h, 1), at) for t, h, at in views]


@pytest.mark.parametrize("views", [
    ((128, 64, 0), (128, 64, 0)),      # one place
    ((128, 64, 0), (128, 64, 64)),     # a token and a head further on, half of it shared
    ((256, 64, 0), (256, 64, 64)),     # out[:, :2] and out[:, 1:3]
    ((256, 64, 64), (256, 64, 0)),
    ((256, 64, 0), (256, 64, 1)),
    ((256, 64, 0), (256, 64, 127)),
    ((256, 64, 0), (256, 64, 256 * 4 + 64 + 63)),  # the last element of the one is the first of the other
    ((64, 320, 0), (64, 320, 256)),    # heads outermost
    ((128, 64, 0), (256, 64, 0)),      # unlike strides
    ((128, 64, 0), (64, 320, 320)),
    ((300, 64, 0), (200, 100, 1299)),
])
def test_overlapping_outputs_are_refused(mi, args, views):
    k, v = outs(views)
    with pytest.raises(ValueError, match="memory"):
        mi.kv_read_quant(*args, k_out=k, v_out=v)


@pytest.mark.parametrize("views", [
    ((256, 64, 0), (256, 64, 128)),    # out[:, :2] and out[:, 2:]
    ((256, 64, 128), (256, 64, 0)),
    ((256, 128, 0), (256, 128, 64)),   # K and V of a head side by side
    ((128, 64, 0), (128, 64, 640)),    # one behind the other
    ((64, 320, 0), (64, 320, 640)),
    ((64, 640, 0), (64, 640, 320)),
    ((256, 64, 0), (256, 64, 256 * 4 + 128)),
    ((300, 64, 0), (600, 64, 128)),    # unlike strides, rows between each other's
    ((300, 64, 0), (300, 100, 128)),
])
def test_outputs_side_by_side_are_taken(mi, args, views):
    """As far as the refusal of tensors that are not on a GPU."""
    k, v = outs(views)
    with pytest.raises(ValueError, match="GPU"):
        mi.kv_read_quant(*args, k_out=k, v_out=v)


def test_against_all_places(mi):
    """Random strides: refused where, and only where, an element of the one is one of the other."""
    import random

    r = random.Random(5)
    both = [0, 0]
    for _ in range(3000):
        rows, heads, d = r.randint(1, 4), r.randint(1, 3), r.randint(1, 4)
        strides = [(r.choice((d * heads, d, d + 1, 17, 2 * d * heads)), r.choice((d, d + 1, 2 * d, rows * d))) for _ in "kv"]
        if r.random() < 0.7:
            strides[1] = strides[0]
        at = [100, 100 + r.randint(-60, 60)]
        places = [{at[i] + t * strides[i][0] + h * strides[i][1] + c for t in range(rows) for h in range(heads) for c in range(d)}
                  for i in range(2)]
        want = bool(places[0] & places[1])
        both[want] += 1
        assert mi._rows_meet(at[1] - at[0], strides[0], strides[1], rows, heads, d) == want, (rows, heads, d, strides, at)
    assert min(both) > 300


@pytest.mark.parametrize("parts,other", [("k", "v_out"), ("v", "k_out")])
def test_a_tensor_for_the_part_not_read_is_refused(mi, args, parts, other):
    import torch

    out = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=other):
        mi.kv_read_quant(*args, parts=parts, **{other: out})
    with pytest.raises(ValueError, match=other):
        mi.kv_read_quant(*args, parts=parts, k_out=out, v_out=torch.zeros_like(out))
