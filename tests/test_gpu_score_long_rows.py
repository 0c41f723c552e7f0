"""Long rows of the token scores against each output's own bar (tests/score_bars.py), with the mass where a lost or
doubled element shows."""
import numpy as np
import pytest
import torch

from pcp_amd import scores
from score_bars import edge_row, sharp_bars
from score_ref import close, score_ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def check(x, ids, out, tau, k, elem):
    h64 = x.double().cpu().numpy()
    logp, h, m, log_sum, tlp, tid = score_ref(h64, ids, tau, k)
    bar, ebar = sharp_bars(h64, tau, elem)
    got = {n: None if (t := getattr(out, n)) is None else t.double().cpu().numpy().reshape(len(h64), -1)
           for n in ("logp", "entropy", "row_max", "log_sum", "top_logp", "top_ids")}
    assert np.array_equal(got["row_max"][:, 0], m)
    close(got["log_sum"][:, 0], log_sum, bar)
    close(got["logp"][:, 0], logp, bar)
    close(got["entropy"][:, 0], h, ebar)
    if k:
        assert np.array_equal(got["top_ids"], tid)
        close(got["top_logp"], tlp, bar[:, None])


SIZES = [("bf16", 1), ("bf16", 3), ("bf16", 300), ("f32", 1), ("f32", 5), ("f32", 260), ("f16", 2), ("f16", 257)]


@pytest.mark.parametrize("dtype,R", SIZES)
@pytest.mark.parametrize("V", [50257, 16383, 151936])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("k", [0, 20])
def test_mass_at_the_edges(dtype, R, V, offset, k):
    elem = DT[dtype].itemsize
    buf = torch.empty(R * V + offset, dtype=DT[dtype], device=DEV)
    x = buf[offset:].view(R, V)
    rng = np.random.default_rng(V + offset)
    ids = np.zeros(R, np.int64)
    picked = sorted({0, 1, R // 2, R - 1} & set(range(R)))
    x.normal_()
    for r in picked:
        row, at = edge_row(V, elem, (offset + r * V) % (16 // elem))
        x[r] = torch.from_numpy(row).to(DT[dtype]).to(DEV)
        ids[r] = rng.choice(at)
    out = scores.token_scores(x[:, None], torch.from_numpy(ids[:, None]).to(DEV), k=k)
    part = scores.TokenScores(*(None if t is None else t[picked] for t in (
        out.logp, out.entropy, out.row_max, out.log_sum, out.top_logp, out.top_ids)))
    check(x[picked], ids[picked], part, 1.0, k, elem)


@pytest.mark.parametrize("dtype,R", SIZES)
@pytest.mark.parametrize("V", [50257, 151936])
@pytest.mark.parametrize("tau", [1.0, 0.75])
def test_rows_like_a_models(dtype, R, V, tau):
    g = torch.Generator(device=DEV).manual_seed(R + V)
    x = torch.randn((R, V), generator=g, device=DEV) * 3
    at = torch.randint(0, V, (R, 12), generator=g, device=DEV)
    x.scatter_add_(1, at, torch.rand(at.shape, generator=g, device=DEV) * 12)
    x = x.to(DT[dtype])
    ids = torch.randint(0, V, (R, 1), generator=g, device=DEV)
    out = scores.token_scores(x[:, None], ids, k=9, temperature=tau)
    picked = sorted({0, 1, R // 2, R - 1} & set(range(R)))
    part = scores.TokenScores(*(t[picked] for t in (out.logp, out.entropy, out.row_max, out.log_sum, out.top_logp, out.top_ids)))
    check(x[picked], ids[picked, 0].cpu().numpy(), part, tau, 9, DT[dtype].itemsize)
