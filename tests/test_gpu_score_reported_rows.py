"""Token scores of rows that are reported because a logit is NaN: what is written for them, and that the rows beside
them are as they would be."""
import numpy as np
import pytest
import torch

from pcp_amd import grpo, scores
from pcp_amd._lib import PcpError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
QUIET = {"bf16": torch.tensor([0x7fc0, -0x40], dtype=torch.int16), "f16": torch.tensor([0x7e00, -0x200], dtype=torch.int16),
         "f32": torch.tensor([0x7fc00000, -0x400000], dtype=torch.int32)}
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("R,V,k", [(300, 20003, 5), (300, 20003, 256), (3, 20003, 5), (3, 151936, 77), (1, 151936, 20), (100, 50257, 33),
                                   (2, 1003, 256), (3, 262144, 256), (4, 7, 7)])
@pytest.mark.parametrize("numbers", [0, 3, "masked", "half"])
def test_every_alternative_of_a_row_of_nan_is_written(dtype, R, V, k, numbers):
    """Rows of NaN with no or few numbers among them, in one part and in several: k ids of the vocabulary, each once,
    the numbers first (NaN ranks below every number), whatever the buffers held."""
    rng = np.random.default_rng(R + V + k)
    x = rng.standard_normal((R, V)).astype(np.float32) * 3
    bad = np.arange(R) % 3 == 0
    for r in np.flatnonzero(bad):
        if numbers == "half":
            x[r, rng.random(V) < 0.5] = np.nan
            x[r, 0] = np.nan
            continue
        x[r] = np.nan
        n = 0 if numbers == 0 else min(3, V - 1)
        x[r, rng.choice(V, n, replace=False)] = [2.0, -1.0, 0.5][:n]
        if numbers == "masked":   # and masks among the numbers, of two values
            at = rng.choice(V, min(4, V), replace=False)
            x[r, at] = np.array([-np.inf, -1e9 if dtype != "f16" else -60000.0] * 2)[:len(at)]
            x[r, rng.integers(0, V)] = np.nan
    x = torch.from_numpy(x).to(DT[dtype]).to(DEV)
    ids = torch.zeros((R, 1), dtype=torch.int64, device=DEV)
    ctx = grpo.Context(0)
    fill = lambda *shape: torch.full(shape, 7.0, device=DEV)  # noqa: E731
    out = scores.TokenScores(fill(R, 1), fill(R, 1), fill(R, 1), fill(R, 1), fill(R, 1, k),
                             torch.full((R, 1, k), -77, dtype=torch.int32, device=DEV))
    scores.token_scores(x[:, None], ids, k=k, outputs=out, sync=False, ctx=ctx)
    with pytest.raises(PcpError) as e:
        ctx.sync()
    assert e.value.code == -4
    top = out.top_ids[:, 0].cpu().numpy()
    assert (top >= 0).all() and (top < V).all(), (top.min(), top.max())
    assert all(len(set(t)) == k for t in top)
    lp = out.top_logp[:, 0].cpu().numpy()
    assert np.isnan(lp[bad]).all() and not np.isnan(lp[~bad]).any()
    host = x.double().cpu().numpy()[bad]
    order = np.lexsort((np.broadcast_to(np.arange(V), host.shape), -np.nan_to_num(host, nan=0.0, posinf=np.inf, neginf=-np.inf),
                        np.isnan(host)))[:, :k]
    assert np.array_equal(top[bad], order)
    good = torch.from_numpy(~bad).to(DEV)
    if good.any():
        want = scores.token_scores(x[good][:, None], ids[good], k=k)
        assert torch.equal(out.top_ids[good], want.top_ids)


@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("R,V,k", [(300, 20003, 5), (300, 20003, 100), (3, 20003, 5), (2, 151936, 77), (20, 50257, 0), (4, 8192, 9)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_nan_hides_no_number(dtype, R, V, k, sign):
    """A NaN of either sign a few elements from the largest logits, which mostly are the same lane's: they are found all the same."""
    rng = np.random.default_rng(R + V + k)
    x = rng.standard_normal((R, V)).astype(np.float32) * 3
    rows = np.arange(R)
    at = rng.integers(0, V - 32, R)
    for step in (2, 4, 6):             # distinct logits, all above the rest, at places of the same parity
        x[rows, at + step] = 40 + step
    d = torch.from_numpy(x).to(DT[dtype])
    for i in (at, at + 12):            # by their bits: a conversion may give any NaN
        d[rows, i] = QUIET[dtype][0 if sign > 0 else 1].view(DT[dtype])
    assert torch.isnan(d[rows, at]).all()
    d = d.to(DEV)
    ctx = grpo.Context(0)
    out = scores.token_scores(d[:, None], torch.zeros((R, 1), dtype=torch.int64, device=DEV), k=k, sync=False, ctx=ctx)
    with pytest.raises(PcpError) as e:
        ctx.sync()
    assert e.value.code == -4
    assert torch.isnan(out.entropy).all() and torch.isnan(out.log_sum).all()
    if k:
        host = d.double().cpu().numpy()
        order = np.lexsort((np.broadcast_to(np.arange(V), host.shape), -np.nan_to_num(host, nan=0.0), np.isnan(host)))[:, :k]
        assert np.array_equal(out.top_ids[:, 0].cpu().numpy(), order)
