"""The loss head and the log-probs on logits masked by large finite values: the same bits as with -inf."""
import numpy as np
import pytest
import torch

from pcp_amd import grpo
from pcp_amd._lib import LossMode

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def masked(dtype, S, T, V, pattern, low, seed):
    """Policy and reference logits, and tokens among those that are left."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    pol = torch.randn((S, T, V), device=DEV, generator=g).mul_(3)
    ref = pol + 0.1 * torch.randn((S, T, V), device=DEV, generator=g)
    out = torch.zeros(V, dtype=torch.bool, device=DEV)
    if pattern == "run":
        out[V // 5:4 * V // 5] = True
    elif pattern == "tail":
        out[V - V // 3:] = True
    elif pattern == "scattered":
        out = torch.rand(V, device=DEV, generator=g) < 0.98
    else:
        out[:] = True
    out[V // 7], out[V // 2], out[0] = False, False, False
    for x in (pol, ref):
        x[..., out] = low
    left = torch.nonzero(~out)[:, 0]
    ids = left[torch.randint(0, len(left), (S, T), device=DEV, generator=g)]
    return pol.to(DT[dtype]), ref.to(DT[dtype]), ids


@pytest.mark.parametrize("pattern", ["run", "tail", "scattered", "three"])
@pytest.mark.parametrize("dtype,low", [("f32", -1e10), ("f32", -1e20), ("f32", -1e30), ("f32", -3.4e38), ("bf16", -1e10),
                                       ("bf16", -1e20), ("bf16", -1e30), ("bf16", -1e12), ("f16", -65504.0)])
@pytest.mark.parametrize("S,T,V", [(4, 50, 3001), (2, 3, 40000), (2, 200, 33000), (2, 60, 151936)])
def test_as_with_infinite_masks(dtype, low, pattern, S, T, V):
    got, want = (masked(dtype, S, T, V, pattern, v, V) for v in (low, -float("inf")))
    lens = np.random.default_rng(V).integers(1, T + 1, (S, 1))
    mask = torch.from_numpy((np.arange(T)[None] < lens).astype(np.float32)).to(DEV)
    adv = torch.linspace(-1, 1, S, device=DEV)
    old = grpo.logprob_fwd(want[0], want[2])[0] + 0.01
    kinds = [{}, dict(exact_bf16=True)] + ([dict(force_streaming=True)] if V <= 33000 else [])
    kinds += [dict(dlogits_dtype=torch.float32)] if dtype != "f32" else []
    for kw in kinds:
        a, b = (grpo.grpo_loss_fwd_bwd(p, i, mask, advantages=adv, ref_logits=r, old_logp=old,
                                       loss_mode=LossMode.GRPO_CLIP_KL, **kw) for p, r, i in (got, want))
        for name in ("loss", "dlogits", "logp", "ref_logp", "token_loss"):
            assert torch.equal(getattr(a, name), getattr(b, name)), (kw, name)
        assert bool(torch.isfinite(a.loss))
    for kw in ({}, dict(force_streaming=True)):
        for x, y in zip(grpo.logprob_fwd(got[0], got[2], got[1], **kw), grpo.logprob_fwd(want[0], want[2], want[1], **kw)):
            assert torch.equal(x, y)
