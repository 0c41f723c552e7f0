"""Distillation of more rows than one grid has threads for."""
import pytest
import torch

from pcp_amd import distill

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("S,T", [(16_800_000, 1), (1, 67_300_000)])
@pytest.mark.parametrize("want_dlogits", [True, False])
def test_more_preparation_than_a_grid_holds(S, T, want_dlogits):
    """Two tokens, one of them the teacher's only entry, renormalised: l = log(1 + exp(d)) of the logits'
    difference d, and c sigmoid(d) for the other token's gradient."""
    n = S * T
    z = torch.zeros((S, T, 2), device=DEV)
    z.view(n, 2)[:, 1] = (torch.arange(n, device=DEV) % 1000).float() / 250 - 2
    ids = torch.zeros((S, T, 1), dtype=torch.int32, device=DEV)
    val = torch.ones((S, T, 1), device=DEV)
    out = distill.distill_fwd_bwd(z, ids, val, want_dlogits=want_dlogits)
    d = z.view(n, 2)[:, 1].double()
    want = torch.log1p(torch.exp(d))
    assert bool(((out.token_loss.view(n).double() - want).abs() <= 2e-5 * (1 + want)).all())
    if want_dlogits:
        c = 1.0 / (S * T)
        other = c * torch.sigmoid(d)
        g = out.dlogits.view(n, 2).double()
        assert bool(((g[:, 1] - other).abs() <= 4e-5 * c).all()) and bool(((g[:, 0] + other).abs() <= 4e-5 * c).all())
