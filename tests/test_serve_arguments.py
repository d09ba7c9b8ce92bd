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
