"""Distillation at its largest: more rows than one grid has threads for, and 2^24 tokens."""
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("divergence", ["forward", "reverse"])
@pytest.mark.parametrize("offset", [0, 1])
def test_largest_vocabulary(dtype, divergence, offset):
    """2^24 tokens, in 2,048 parts and more, against the formulas in 64 bits (distill_ref.REL is for up to
    160 terms in a lane's chain, which a part of 64 stays below)."""
    V, k, T = 1 << 24, 256, 2
    g = torch.Generator(device=DEV).manual_seed(5)
    buf = torch.empty(T * V + offset, dtype=dtype, device=DEV).normal_(0, 2, generator=g)
    x = buf[offset:].view(1, T, V)
    t = x.float() + torch.empty_like(x, dtype=torch.float32).normal_(0, 0.5, generator=g)
    top = distill.top_logits(t, k)
    out = distill.distill_fwd_bwd(x, top.ids, top.values, top.lse, divergence=divergence, dlogits_dtype=torch.float32)
    for r in range(T):
        z = x[0, r].double()
        ids = top.ids[0, r].long()
        lq = torch.logsumexp(z, 0)
        q = torch.exp(z - lq)
        log_p = top.values[0, r].double() - top.lse[0, r].double()
        p = log_p.exp()
        pt = (1 - p.sum()).clamp_min(2.0 ** -24)
        inside = torch.zeros(V, dtype=torch.bool, device=DEV)
        inside[ids] = True
        qt = q[~inside].sum()
        log_q = z[ids] - lq
        if divergence == "forward":
            l = (p * (log_p - log_q)).sum() + pt * (pt.log() - qt.log())
            size = (p * (log_p - log_q)).abs().sum() + (pt * (pt.log() - qt.log())).abs()
            grad = q * (p.sum() + pt) - pt * q / qt
            mag = q * (p.sum() + pt) + pt * q / qt
            grad[ids], mag[ids] = q[ids] * (p.sum() + pt) - p, q[ids] * (p.sum() + pt) + p
        else:
            f, ft = log_q - log_p, qt.log() - pt.log()
            l = (q[ids] * f).sum() + qt * ft
            size = (q[ids] * f).abs().sum() + (qt * ft).abs()
            grad, mag = q * (ft - l), q * (1 + ft.abs() + size)
            grad[ids], mag[ids] = q[ids] * (f - l), q[ids] * (1 + f.abs() + size)
        assert abs(float(out.token_loss[0, r]) - float(l)) <= 2e-5 * (1 + float(size)) + 2.0 ** -24 * abs(float(l))
        off = (out.dlogits[0, r].double() - grad / T).abs()
        assert bool((off <= (2e-5 * mag + 2.0 ** -24 * grad.abs()) / T + 2.0 ** -126).all())
