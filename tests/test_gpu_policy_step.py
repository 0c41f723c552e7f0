"""Token scores, their gradient, clipping and the update of many tensors together, as a training step uses them: a
small language model's rollouts are scored, the loss head's dlogits take an entropy bonus, and the clipped step
is checked against torch's autograd in 64 bits."""
import numpy as np
import pytest
import torch

from pcp_amd import grpo, scores, step

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("V,H,S,T", [(1024, 64, 4, 17), (5004, 32, 2, 9)])
def test_policy_step(V, H, S, T):
    torch.manual_seed(V)
    emb = torch.randn(V, H, device=DEV) * 0.3
    head = torch.randn(V, H, device=DEV) * 0.3
    params = [emb, head]
    vel = [torch.zeros_like(x) for x in params]
    # Rollouts: every token drawn from the model, scored as it is drawn.
    ids = torch.zeros(S, T, dtype=torch.int64, device=DEV)
    ids[:, 0] = torch.randint(0, V, (S,), device=DEV)
    behaviour = torch.zeros(S, T, device=DEV)
    for t in range(1, T):
        logits = emb[ids[:, t - 1]] @ head.t()
        drawn = step.sample_tokens(logits, 1.0, torch.rand(S, device=DEV))
        ids[:, t] = drawn
        sc = scores.token_scores(logits[:, None], drawn[:, None], k=3)
        behaviour[:, t] = sc.logp[:, 0]
        assert (sc.top_logp[:, 0, :-1] >= sc.top_logp[:, 0, 1:]).all()
    mask = (torch.arange(T, device=DEV) < torch.randint(T // 2, T + 1, (S, 1), device=DEV)).float()
    adv = torch.randn(S, device=DEV)
    # The step: loss head on the shifted logits, entropy bonus added, backward through the model, clipped update.
    logits = emb[ids] @ head.t()
    out = grpo.grpo_loss_fwd_bwd(logits, ids, mask, advantages=adv, rows=T - 1, tok_offset=1)
    sc = scores.token_scores(logits, ids, mask, rows=T - 1, tok_offset=1)
    assert torch.allclose(sc.logp[:, 1:], behaviour[:, 1:] * mask[:, 1:], atol=1e-4)
    assert torch.allclose(sc.logp[:, 1:], out.logp[:, 1:] * mask[:, 1:], atol=1e-5)
    beta = 0.05
    w = mask / (S * mask[:, 1:].sum(1, keepdim=True).clamp(min=1))
    scores.token_scores_bwd(logits, ids, sc.row_max, sc.log_sum, sc.entropy, dentropy=-beta * w, mask=mask, rows=T - 1,
                            tok_offset=1, dlogits=out.dlogits, accumulate=True)
    d = out.dlogits.reshape(-1, V)
    g_head = (d.t() @ emb[ids].reshape(-1, H)).to(torch.bfloat16)       # mixed types, as an autocast model leaves them
    g_emb = torch.zeros_like(emb).index_add_(0, ids.reshape(-1), d @ head)
    most = 0.5 * float(step.grad_norm([g_emb, g_head]).norm)
    norm = step.grad_norm([g_emb, g_head], most, sync=False)
    before = [x.clone() for x in params]
    step.nesterov_update_many(params, vel, [g_emb, g_head], coef=norm.coef, learning_rate=0.1, momentum=0.9, sync=False)
    grpo.default_context(0).sync()
    # The same in 64 bits by autograd.
    e, h = before[0].double().cpu().requires_grad_(), before[1].double().cpu().requires_grad_()
    i, m = ids.cpu(), mask.double().cpu()
    log_p = torch.log_softmax(e[i] @ h.t(), -1)[:, :-1]
    lp = log_p.gather(2, i[:, 1:, None])[..., 0]
    ent = -(log_p.exp() * log_p).sum(-1)
    n = m[:, 1:].sum(1).clamp(min=1)
    loss = ((-(adv.double().cpu()[:, None]) * lp - beta * ent) * m[:, 1:]).sum(1).div(n).mean()
    ge, gh = torch.autograd.grad(loss, (e, h))
    full = float(torch.sqrt((ge * ge).sum() + (gh * gh).sum()))
    # bf16 head gradients: half a step, 2^-8, of each at most, and so of their norm.
    assert abs(float(norm.norm) - full) <= (2.0 ** -8 + 1e-4) * full
    c = min(1.0, most / full)
    for p, b, g in zip(params, before, (ge, gh)):
        moved = b.double().cpu() - p.double().cpu()
        want = 0.1 * (c * g + 0.9 * c * g)
        # Of the step: 2^-8 twice (the gradients' and the norm's rounding) and the products' f32; of the weights 2^-24.
        lim = (2.0 ** -7 + 2e-4) * want.abs() + 2.0 ** -22 * b.double().cpu().abs() + 1e-5 * want.abs().max()
        assert ((moved - want).abs() <= lim).all()
