"""A context whose work buffer grows after a call on it was captured: the graph's replays keep theirs."""
import pytest
import torch

from pcp_amd import distill, grpo, step

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def inputs(V):
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn((2, 4, V), device=DEV, generator=g)
    return dict(x=x, t=x + torch.randn(x.shape, device=DEV, generator=g),
                ids=torch.randint(0, V, (2, 3), device=DEV, generator=g), u=torch.rand((2, 4), device=DEV, generator=g))


def run(a, ctx, top=None, dist=None, ver=None):
    top = distill.top_logits(a["t"], 12, outputs=top, sync=False, ctx=ctx)
    dist = distill.distill_fwd_bwd(a["x"], top.ids, top.values, top.lse, outputs=dist, sync=False, ctx=ctx)
    ver = step.verify_drafts(a["t"], a["ids"], a["x"][:, :3], uniforms=a["u"], outputs=ver, sync=False, ctx=ctx)
    return top, dist, ver


def flat(outs):
    return [t for o in outs for t in vars(o).values()]


@pytest.mark.parametrize("how", ["verify", "distill", "top", "loss"])
def test_replays_after_the_work_buffer_has_grown(how):
    a, ctx, s = inputs(30000), grpo.Context(0), torch.cuda.Stream()
    outs = run(a, ctx)
    ctx.sync()
    held = ctx.workspace_bytes()
    g = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        run(a, ctx, *outs)
    big = torch.randn((64, 300, 2048), device=DEV)
    for i in range(3):
        if how == "verify":
            step.verify_drafts(big[:, :33].repeat(60, 1, 1), torch.zeros((3840, 32), dtype=torch.int64, device=DEV),
                               uniforms=torch.rand((3840, 33), device=DEV), ctx=ctx)
        elif how == "top":
            distill.top_logits(torch.randn((400, 300000), device=DEV), 256, ctx=ctx)
        elif how == "distill":
            top = distill.top_logits(big, 64, ctx=grpo.default_context())
            distill.distill_fwd_bwd(big, top.ids, top.values, top.lse, ctx=ctx)
        else:
            grpo.grpo_loss_fwd_bwd(torch.zeros((300, 8192, 2), device=DEV), torch.zeros((300, 8192), dtype=torch.int64, device=DEV),
                                   advantages=torch.zeros(300, device=DEV), ctx=ctx)
        other = [torch.full((1 << 18,), 3.0e38, device=DEV) for _ in range(64)]   # whatever was freed is another's now
        for o in flat(outs):
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
        for got, want in zip(flat(outs), flat(run(a, grpo.Context(0)))):
            assert torch.equal(got, want)
        del other
        a["x"].mul_(0.9)
        a["u"].copy_(1 - a["u"])
    if how in ("verify", "top", "distill"):
        assert ctx.workspace_bytes() > 2 * held
    ctx.sync()
    del g
    ctx.release_workspace()
    assert ctx.workspace_bytes() == 0
