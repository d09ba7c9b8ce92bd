"""Arguments of the Python calls of the paged cache and the sampler, on CPU tensors: a call whose arguments
are all right is refused last, for its device."""
import pytest


def test_a_workspace_with_gaps_is_refused(mi):
    """The call writes as many bytes as the workspace has elements for, from its first one on: with gaps or
    repeated elements these are not its own."""
    import torch

    bf, i32 = torch.bfloat16, torch.int32
    q, c = torch.zeros(5, 4, 64, dtype=bf), torch.zeros(6, 2, 16, 64, dtype=bf)
    pages, n = torch.zeros(5, 3, dtype=i32), torch.ones(5, dtype=i32)
    ws = torch.zeros(4096, dtype=torch.uint8)
    for bad in (ws[::2], ws[:1].expand(4096), ws.view(64, 64).t(), ws.view(64, 64)[:, :32]):
        with pytest.raises(ValueError, match="workspace"):
            mi.paged_attn(q, c, c, pages, n, workspace=bad)
    for good in (ws, ws[16:], ws.view(64, 64), ws.view(torch.float32), None, "auto"):
        with pytest.raises(ValueError, match="GPU"):
            mi.paged_attn(q, c, c, pages, n, workspace=good)


@pytest.mark.parametrize("top_k", [2 ** 31, 10 ** 12, -(2 ** 40), 2 ** 31 - 1, -(2 ** 31), 50, 50.0])
def test_a_top_k_of_any_size_is_taken(mi, top_k):
    """A number larger than the vocabulary, as a caller writes for "no limit", is off; so is a negative one."""
    import torch

    with pytest.raises(ValueError, match="GPU"):
        mi.sample(torch.zeros(3, 10), torch.zeros(3), top_k=top_k)


@pytest.mark.gpu
def test_a_large_top_k_is_off(mi, dev):
    import torch

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((9, 5003), generator=g, device="cuda")
    u = torch.rand((9,), generator=g, device="cuda")
    want = mi.sample(x, u, top_p=0.9)
    for k in (2 ** 31, 10 ** 12, -(2 ** 40), 5003):
        assert torch.equal(mi.sample(x, u, top_k=k, top_p=0.9), want)
    assert torch.equal(mi.sample(x, u, top_k=50.0), mi.sample(x, u, top_k=50))
