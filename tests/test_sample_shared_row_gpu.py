"""Several tokens from one row of logits, read in place (row stride 0): the same as from copies of it, to the bit."""
import pytest


def test_a_pitch_of_zero_is_taken(mi):
    """Without a GPU: pitches from 1 to V - 1 and negative ones stay refused, 0 gets as far as the device."""
    import torch
    from test_serve_abi import sample

    assert sample(mi, ld=99) == 2 and sample(mi, ld=1) == 2 and sample(mi, ld=-100) == 2
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the call would run on the fake addresses")
    assert sample(mi, ld=0) == 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("V", [1, 7, 5000, 32001])
@pytest.mark.parametrize("how", [dict(), dict(k=50, p=0.9), dict(p=0.9), dict(T=0.0), dict(k=1000, low=0.01)])
def test_one_row_for_all(mi, dev, dtype, rows, V, how):
    import torch
    from test_sample_gpu import check, make

    x, _ = make(1, V, dtype, V)
    u = torch.rand((rows,), generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda")
    got = check(mi, x.expand(rows, V), u, **how)
    want = mi.sample(x.expand(rows, V).contiguous(), u, temperature=how.get("T", 1.0), top_k=how.get("k", 0),
                     top_p=how.get("p", 1.0), min_p=how.get("low", 0.0))
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_one_row_with_settings_of_each(mi, dev):
    import torch
    from test_sample_gpu import check, make

    x, u = make(64, 10007, "bf16", 4)
    t = torch.linspace(0.0, 2.0, 64, device="cuda")
    k = torch.arange(64, dtype=torch.int32, device="cuda") * 40
    p = torch.linspace(0.1, 1.0, 64, device="cuda")
    check(mi, x[:1].expand(64, 10007), u, T=t, k=k, p=p)
