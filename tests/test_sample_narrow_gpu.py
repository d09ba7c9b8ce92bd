"""Sampling from rows whose logits lie so close together, next to the temperature, that all of them weigh about 1.
Tokens against the definition in 64 bits, without tolerance, as in the tests of mi_sample."""
import pytest
from test_sample_gpu import check

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("T,width", [(1e38, 1e-6), (3e38, 1e-4), (3.4e38, 1e-37), (1e30, 1e-12), (1e10, 1e-35), (INF, 1.0),
                                     (3e38, 3e38), (1.0, 1e-44)])
@pytest.mark.parametrize("how", [dict(p=0.5), dict(k=-50), dict(k=-50, p=0.99), dict(k=30, p=0.9), dict(low=1.0)])
def test_narrow_rows(mi, dev, rows, T, width, how):
    """Borders in the middle of the row and in its tail; k counted from the row's end where negative."""
    import torch

    V = 5003
    g = torch.Generator(device="cuda").manual_seed(7)
    x = (torch.rand((rows, V), generator=g, device="cuda") - 0.5) * width
    u = torch.rand((rows,), generator=g, device="cuda")
    how = dict(how)
    if how.get("k", 0) < 0:
        how["k"] += V
    check(mi, x, u, T=T, **how)
    check(mi, x.bfloat16(), u, T=T, **how)


@pytest.mark.parametrize("T", [1e38, 3e38])
def test_settings_of_each_row(mi, dev, T):
    import torch

    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.rand((64, 32001), generator=g, device="cuda") * torch.logspace(-12, 1, 64, device="cuda")[:, None]
    u = torch.rand((64,), generator=g, device="cuda")
    k = torch.tensor([0, 31990, 200, 20000], dtype=torch.int32, device="cuda").repeat(16)
    p = torch.tensor([0.9, 1.0, 0.5, 0.999], device="cuda").repeat_interleave(16)
    check(mi, x, u, T=torch.full((64,), T, device="cuda"), k=k, p=p)
