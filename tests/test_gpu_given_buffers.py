"""Result buffers of the caller's in top logits, distillation and draft verification: kept by the
allocator while another stream writes them, and refused off the context's device."""
import pytest
import torch

from pcp_amd import distill, grpo, step
from pcp_amd._lib import PcpError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
S, T, V, K = 2, 3, 5000, 8


def calls():
    """name -> (a call with `outputs`, the tensors of its outputs)."""
    x = torch.randn((S, T, V), device=DEV)
    ids = torch.arange(K, dtype=torch.int32, device=DEV).expand(S, T, K).contiguous()
    val, lse = torch.randn((S, T, K), device=DEV), torch.full((S, T), 5.0, device=DEV)
    draft, u = torch.zeros((S, T - 1), dtype=torch.int64, device=DEV), torch.rand((S, T), device=DEV)
    return {
        "top": (lambda outputs=None, **kw: distill.top_logits(x, K, outputs=outputs, **kw),
                lambda o: [o.values, o.ids, o.lse]),
        "distill": (lambda outputs=None, **kw: distill.distill_fwd_bwd(x, ids, val, lse, outputs=outputs, **kw),
                    lambda o: [o.loss, o.token_loss, o.dlogits]),
        "dlogits": (lambda outputs=None, **kw: distill.distill_fwd_bwd(
            x, ids, val, lse, dlogits=None if outputs is None else outputs.dlogits, **kw), lambda o: [o.dlogits]),
        "verify": (lambda outputs=None, **kw: step.verify_drafts(x, draft, uniforms=u, outputs=outputs, **kw),
                   lambda o: [o.tokens, o.accepted, o.logp]),
    }


@pytest.mark.parametrize("name", ["top", "distill", "dlogits", "verify"])
def test_buffers_dropped_while_another_stream_writes_them(name):
    """The caller's own stream does not get a dropped buffer's memory before the other stream is done."""
    call, tensors = calls()[name]
    ctx, s = grpo.Context(0), torch.cuda.Stream()
    call(ctx=ctx)                                          # the work buffer has its size
    out = call(ctx=ctx)
    torch.cuda.synchronize()
    at = [t.data_ptr() for t in tensors(out)]
    shapes = [(t.shape, t.dtype) for t in tensors(out)]
    done = torch.cuda.Event()
    with torch.cuda.stream(s):
        busy = torch.randn((4096, 4096), device=DEV)
        for _ in range(200):
            busy = busy @ busy
            busy /= busy.norm()
    again = call(out, ctx=ctx, stream=s, sync=False)
    done.record(s)
    del out, again
    fresh = [torch.empty(sh, dtype=dt, device=DEV) for sh, dt in shapes]
    assert not done.query(), "the other stream ended too early for this test to see anything"
    assert not set(t.data_ptr() for t in fresh) & set(at)
    s.synchronize()
    ctx.sync()


@pytest.mark.parametrize("name", ["top", "distill", "dlogits", "verify"])
def test_buffers_elsewhere_are_refused(name):
    call, tensors = calls()[name]
    n = len(tensors(call()))
    for i in range(n):
        out = call()
        fields = {"top": ["values", "ids", "lse"], "distill": ["loss", "token_loss", "dlogits"], "dlogits": ["dlogits"],
                  "verify": ["tokens", "accepted", "logp"]}[name]
        setattr(out, fields[i], getattr(out, fields[i]).cpu())
        with pytest.raises(PcpError, match="cpu"):
            call(out)
