"""Arguments that contradict each other in the calls of a draft model are refused before any work
(no GPU needed); those that go together do what each says."""
import ctypes

import pytest
import torch

from pcp_amd import _lib, distill, step
from pcp_amd._lib import PcpError

X = torch.zeros((2, 3, 50))
IDS, VAL, LSE = torch.zeros((2, 3, 4), dtype=torch.int32), torch.zeros((2, 3, 4)), torch.zeros((2, 3))


def outputs(dlogits):
    return distill.DistillOutputs(torch.empty(()), torch.empty((2, 3)), dlogits)


@pytest.mark.parametrize("kw,code,text", [
    (dict(dlogits=torch.empty_like(X), want_dlogits=False), -1, "want_dlogits"),
    (dict(dlogits=torch.empty_like(X), outputs=outputs(torch.empty_like(X))), -1, "twice"),
    (dict(dlogits=torch.empty_like(X), outputs=outputs(None)), -1, "twice"),
    (dict(dlogits=torch.empty_like(X), dlogits_dtype=torch.bfloat16), -2, "bfloat16"),
    (dict(outputs=outputs(torch.empty_like(X)), dlogits_dtype=torch.bfloat16), -2, "bfloat16"),
    (dict(outputs=outputs(None), dlogits_dtype=torch.float32), -1, "no dlogits"),
])
def test_dlogits_given_in_two_ways(kw, code, text):
    with pytest.raises(PcpError, match=text) as e:
        distill.distill_fwd_bwd(X, IDS, VAL, LSE, **kw)
    assert e.value.code == code


@pytest.mark.parametrize("kw", [
    dict(mask=torch.ones((2, 0))), dict(mask=torch.ones((2, 0), dtype=torch.bool), rows=1), dict(tokens=0),
    dict(tokens=2), dict(mask=torch.ones((2, 3)), tok_offset=1), dict(rows=-1), dict(tok_offset=-1, rows=2),
    dict(rows=1 << 40),
])
def test_rows_that_no_token_belongs_to(kw):
    with pytest.raises(PcpError, match="do not fit"):
        distill.distill_fwd_bwd(X, IDS, VAL, LSE, **kw)


@pytest.mark.parametrize("k", [0, -1, 51, 257, (1 << 32) + 5])
def test_numbers_of_entries(k):
    with pytest.raises(PcpError, match="k must be"):
        distill.top_logits(X if k != 257 else torch.zeros((2, 400)), k)
    with pytest.raises(PcpError, match="k must be"):
        distill.distill_fwd_bwd(X, IDS[..., :1].expand(2, 3, 257), VAL[..., :1].expand(2, 3, 257), LSE)
    with pytest.raises(PcpError, match="k must be"):
        distill.distill_fwd_bwd(X, IDS[..., :0], VAL[..., :0], LSE)


@pytest.mark.parametrize("kw,code,text", [
    (dict(target_seq_stride=99), -1, "sequence strides"),
    (dict(target_seq_stride=-400), -1, "sequence strides"),
    (dict(draft_seq_stride=99, draft_logits=0x1000), -1, "sequence strides"),
    (dict(target_seq_stride=1 << 62), -9, "overflows"),
    (dict(target_row_stride=1 << 62), -9, "overflows"),
    (dict(draft_seq_stride=1 << 61), -9, "overflows"),
    (dict(draft_row_stride=1 << 60), -9, "overflows"),
    (dict(target_row_stride=200, target_seq_stride=100), -1, "context is NULL"),
    (dict(n_draft=0, draft_ids=None), -1, "context is NULL"),
])
def test_strides_of_the_verification(kw, code, text):
    L, a = _lib.lib(), _lib.VerifyArgs()
    L.pcp_verify_args_init(ctypes.byref(a))
    for k, v in {**dict(n_seq=2, n_draft=3, vocab=100, target_logits=0x1000, draft_ids=0x2000, uniforms=0x3000,
                        tokens=0x4000, accepted=0x5000), **kw}.items():
        setattr(a, k, v)
    assert L.pcp_verify_drafts(None, ctypes.byref(a)) == code
    assert text in L.pcp_last_error(None).decode()


def test_strides_of_views():
    x = torch.zeros((4, 9, 50))
    assert (step._row_stride(x[:, -3:]), step._seq_stride(x[:, -3:])) == (50, 450)
    t = torch.zeros((3, 4, 50)).transpose(0, 1)
    assert (step._row_stride(t), step._seq_stride(t)) == (200, 50)
    assert step._seq_stride(x[:1]) == 0 and step._seq_stride(x[:, :0]) == 0
    for bad in (x.transpose(1, 2), x[..., ::2]):
        with pytest.raises(PcpError, match="contiguous"):
            step._row_stride(bad)


@pytest.mark.gpu
def test_loss_alone_into_outputs_that_have_dlogits():
    dev = torch.device("cuda:0")
    x = torch.randn((2, 3, 700), device=dev)
    top = distill.top_logits(torch.randn((2, 3, 700), device=dev), 9)
    out = distill.distill_fwd_bwd(x, top.ids, top.values, top.lse)
    want, kept = float(out.loss), out.dlogits.fill_(7.0)
    out.loss.zero_()
    again = distill.distill_fwd_bwd(x, top.ids, top.values, top.lse, outputs=out, want_dlogits=False)
    assert again is out and abs(float(out.loss) - want) <= 4e-5 * (1 + abs(want))
    assert out.dlogits is kept and bool((kept == 7.0).all())
    distill.distill_fwd_bwd(x, top.ids, top.values, top.lse, outputs=out, dlogits=kept, dlogits_dtype=torch.float32)
    assert not bool((kept == 7.0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("V,want_dlogits", [(700, True), (40000, True), (40000, False)])
@pytest.mark.parametrize("weight", [float("nan"), float("inf")])
def test_weights_that_are_not_finite_are_reported(V, want_dlogits, weight):
    dev = torch.device("cuda:0")
    x, t = torch.randn((2, 3, V), device=dev), torch.randn((2, 3, V), device=dev)
    top, mask = distill.top_logits(t, 9), torch.ones((2, 3), device=dev)
    distill.distill_fwd_bwd(x, top.ids, top.values, top.lse, mask, want_dlogits=want_dlogits)
    mask[1, 2] = weight
    with pytest.raises(PcpError) as e:
        distill.distill_fwd_bwd(x, top.ids, top.values, top.lse, mask, want_dlogits=want_dlogits)
    assert e.value.code == -4
    top.ids[1, 2] = -100                       # a row without entries has no loss, whatever its weight
    distill.distill_fwd_bwd(x, top.ids, top.values, top.lse, mask, want_dlogits=want_dlogits)
