"""Calls of more workgroups than one launch can have: more than 2^28 tokens in a rotation, more than 2^23 rows in
a sampling call."""
import pytest

pytestmark = pytest.mark.gpu


def test_rotation_of_2_28_tokens(mi, dev):
    """One call against two of half the tokens each, at their positions."""
    import torch

    T, half = 2 ** 28 + 5, 2 ** 27 + 3
    x = torch.randint(-2 ** 15, 2 ** 15, (T * 2,), dtype=torch.int16, device="cuda") & 0x3fff  # finite, positive
    x = x.view(torch.bfloat16).view(1, T, 1, 2)
    f, _ = mi.rope_frequencies(2)
    got = mi.rope(x, f)
    for a, b in ((0, half), (half, T)):
        assert torch.equal(got[:, a:b], mi.rope(x[:, a:b], f, pos0=a))


def test_tokens_of_2_23_rows(mi, dev):
    import torch

    rows = 2 ** 23 + 77
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((rows, 3), generator=g, device="cuda")
    u = torch.rand((rows,), generator=g, device="cuda")
    t = (torch.rand((rows,), generator=g, device="cuda") < 0.5).float()  # half of the rows greedy
    k = torch.full((rows,), 2, dtype=torch.int32, device="cuda")
    p, low = torch.ones((rows,), device="cuda"), torch.zeros((rows,), device="cuda")
    prob = torch.full((rows,), -1.0, device="cuda")
    got = mi.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=low, prob=prob)
    top = x.max(1, keepdim=True).values
    assert torch.equal(got[t == 0].long(), (x == top).int().argmax(1)[t == 0])
    assert (prob[t == 0] == 1).all() and (prob > 0).all()
    assert (got.long() != x.argmin(1)).all()  # never the third
    for a in (0, 2 ** 22, 2 ** 23 - 10, 2 ** 23 - 1, rows - 40):
        s = slice(a, a + 40)
        assert torch.equal(got[s], mi.sample(x[s], u[s], temperature=t[s], top_k=k[s], top_p=p[s], min_p=low[s]))
