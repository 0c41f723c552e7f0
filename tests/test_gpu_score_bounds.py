"""Token scores where the definition bounds them: signs of peaked rows, the smallest vocabularies."""
import numpy as np
import pytest
import torch

from pcp_amd import scores
from score_ref import bars, close, score_ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("R,V,k", [(4096, 1000, 4), (4096, 1000, 0), (512, 20000, 64), (24, 151936, 3), (200, 50257, 0), (4096, 1, 1)])
@pytest.mark.parametrize("tau", [1.0, 0.7])
@pytest.mark.parametrize("second", [200.0, 30.0, 16.0])
def test_signs_of_peaked_rows(dtype, R, V, k, tau, second):
    """One token has nearly all of the mass, its logit anywhere: a log-prob is never
    above 0, an entropy and a log-sum against the largest logit never below, so that sqrt(entropy) and
    log1p(-exp(logp)) are numbers."""
    g = torch.Generator(device=DEV).manual_seed(R + V)
    top = (torch.rand((R, 1), generator=g, device=DEV) * 25 + 3).to(DT[dtype])
    x = (top.float() - second - torch.rand((R, V), generator=g, device=DEV)).to(DT[dtype])
    ids = torch.randint(0, V, (R, 1), generator=g, device=DEV)
    x.scatter_(1, ids, top)
    out = scores.token_scores(x[:, None], ids, k=k, temperature=tau)
    # log(1 + rest) <= rest, the other terms' share; a logit of at most 229 moves by half a step, 0.5 in bf16, and so does the
    # largest (0.0625): less than 1 in all. The sum and the results are off by a few f32 roundings of numbers up to 1.
    rest = V * np.exp(-(second - 1) / float(np.float32(tau))) + 2.0 ** -21
    assert (out.logp <= 0).all() and (out.logp >= -rest).all(), (out.logp.max(), out.logp.min())
    assert (out.log_sum >= 0).all() and (out.log_sum <= rest).all(), (out.log_sum.min(), out.log_sum.max())
    assert (out.entropy >= 0).all(), out.entropy.min()
    assert torch.isfinite(out.entropy.sqrt()).all() and not torch.isnan(torch.log1p(-out.logp.exp())).any()
    if k:
        assert (out.top_logp <= 0).all() and torch.equal(out.top_ids[:, 0, 0].long(), ids[:, 0])


@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("R", [1, 300])
def test_smallest_vocabularies(dtype, offset, R):
    """Rows without a whole 16-byte vector, or with one or two: every k there is."""
    rng = np.random.default_rng(R)
    for V in range(1, 19):
        host = torch.from_numpy(rng.standard_normal((R, V)) * 3).to(DT[dtype])
        buf = torch.empty(R * V + offset, dtype=DT[dtype], device=DEV)
        x = buf[offset:].view(R, V)
        x.copy_(host)
        ids = rng.integers(0, V, R)
        for k in range(V + 1):
            out = scores.token_scores(x[:, None], torch.from_numpy(ids[:, None]).to(DEV), k=k)
            logp, h, m, log_sum, tlp, tid = score_ref(host.double().numpy(), ids, 1.0, k)
            for got, want, bar in ((out.logp, logp, bars(h)), (out.entropy, h, bars(h)), (out.log_sum, log_sum, bars(h)),
                                   (out.row_max, m, 0.0)):
                close(got.cpu().numpy()[:, 0], want, bar)
            if k:
                assert np.array_equal(out.top_ids.cpu().numpy()[:, 0], tid), (V, k)
                close(out.top_logp.cpu().numpy()[:, 0], tlp, bars(h)[:, None])
