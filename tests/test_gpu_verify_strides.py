"""Draft verification of logits as a model leaves them: the last positions of longer rows of
positions, drafting steps stacked one after another, windows that share rows."""
import numpy as np
import pytest
import torch

from pcp_amd import step

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def equal(a, b):
    assert torch.equal(a.tokens, b.tokens) and torch.equal(a.accepted, b.accepted) and torch.equal(a.logp, b.logp)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("S,n,L,V", [(1, 3, 9, 1000), (3, 2, 8, 1003), (6, 4, 5, 9001), (40, 1, 7, 257), (5, 0, 4, 33)])
@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_views_are_read_in_place(dtype, S, n, L, V, temperature):
    g = torch.Generator(device=DEV).manual_seed(V)
    long = torch.full((S, L, V), float("nan"), device=DEV, dtype=DT[dtype])
    long[:, -(n + 1):] = torch.randn((S, n + 1, V), device=DEV, generator=g).mul_(2).to(DT[dtype])
    steps = (long[:, -(n + 1):][:, :n].transpose(0, 1).float()
             + 0.4 * torch.randn((n, S, V), device=DEV, generator=g)).to(DT[dtype])
    target, draft = long[:, -(n + 1):], steps.transpose(0, 1)
    ids = draft.float().add(torch.rand(draft.shape, device=DEV, generator=g)).argmax(-1)
    kw = dict(temperature=temperature, uniforms=torch.rand((S, n + 1), device=DEV, generator=g))
    want = step.verify_drafts(target.contiguous(), ids, draft.contiguous(), **kw)
    equal(step.verify_drafts(target, ids, draft, **kw), want)
    equal(step.verify_drafts(target, ids, draft.contiguous(), **kw), want)
    equal(step.verify_drafts(target.contiguous(), ids, draft, **kw), want)
    equal(step.verify_drafts(target, ids, **kw), step.verify_drafts(target.contiguous(), ids, **kw))


def test_windows_that_share_rows():
    """Sequence s scored by rows s .. s + n of one long text: sequence and row strides of one row."""
    S, n, V = 6, 3, 5000
    text = torch.randn((S + n, V), device=DEV)
    target = text.as_strided((S, n + 1, V), (V, V, 1))
    ids = target[:, :n].argmax(-1)
    kw = dict(uniforms=torch.rand((S, n + 1), device=DEV))
    equal(step.verify_drafts(target, ids, **kw), step.verify_drafts(target.contiguous(), ids, **kw))


def test_sequences_past_32_bits():
    """Sequences 1.1e9 elements apart, the draft's steps 1.3e9."""
    S, n, V = 3, 2, 3000
    far = torch.empty(2 * 1_100_000_000 + (n + 1) * V, dtype=torch.bfloat16, device=DEV)
    target = far.as_strided((S, n + 1, V), (1_100_000_000, V, 1))
    target.copy_(torch.randn((S, n + 1, V), device=DEV))
    wide = torch.empty(1_300_000_000 + S * V, dtype=torch.bfloat16, device=DEV)
    draft = wide.as_strided((S, n, V), (V, 1_300_000_000, 1))
    draft.copy_(target[:, :n])
    ids = draft.argmax(-1)
    kw = dict(uniforms=torch.rand((S, n + 1), device=DEV))
    equal(step.verify_drafts(target, ids, draft, **kw), step.verify_drafts(target.contiguous(), ids, draft.contiguous(), **kw))
