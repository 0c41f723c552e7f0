"""Draft verification on the GPU: tokens and counts equal to the definition in 64 bits
(tests/distill_ref.py), log-probs to f32 rounding."""
import numpy as np
import pytest
import torch

from distill_ref import IGNORE, verify_ref
from pcp_amd import grpo, step
from pcp_amd._lib import PcpError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def dev_as(x, dtype, offset=0):
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(DT[dtype])
    buf = torch.empty(t.numel() + offset, dtype=t.dtype, device=DEV)
    v = buf[offset:].view(t.shape)
    v.copy_(t)
    return v


def host64(t):
    return t.detach().double().cpu().numpy()


def make(rng, S, n, V, near=0.7, temperature=1.0):
    x = rng.standard_normal((S, n + 1, V)).astype(np.float32) * 3
    for r in x.reshape(-1, V):
        r[rng.integers(0, V, 5)] += 8
    y = x[:, :n] + near * rng.standard_normal((S, n, V)).astype(np.float32)
    d = np.zeros((S, n), np.int64)
    for s in range(S):
        for i in range(n):
            z = y[s, i].astype(np.float64) / max(temperature, 1e-3)
            d[s, i] = np.argmax(z + rng.gumbel(size=V)) if temperature > 0 else np.argmax(z)
    return x, y, d, rng.random((S, n + 1)).astype(np.float32)


def check(out, x, y, d, lens, u, T):
    V = x.shape[-1]
    S, n = d.shape
    want = verify_ref(host64(x), None if y is None else host64(y), d, lens, u, T, V)
    assert np.array_equal(out.accepted.cpu().numpy(), want[1])
    assert np.array_equal(out.tokens.cpu().numpy(), want[0])
    lp = host64(out.logp)
    # log p rounded once to f32 from 64-bit sums
    assert (np.abs(lp - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 1e-12).all()


CASES = [("f32", 1, 0, 1), ("f32", 3, 1, 2), ("bf16", 4, 3, 7), ("f16", 5, 4, 100), ("bf16", 6, 2, 1003),
         ("f32", 9, 5, 1000), ("bf16", 40, 6, 4096), ("f32", 7, 64, 300), ("bf16", 8, 4, 50257), ("f16", 3, 2, 50257),
         ("f32", 2, 3, 151936), ("bf16", 5, 8, 151936), ("bf16", 1, 1, 8193)]


@pytest.mark.parametrize("dtype,S,n,V", CASES)
@pytest.mark.parametrize("temperature", [1.0, 0.7, 0.0])
@pytest.mark.parametrize("lookup", [False, True])
def test_verify(dtype, S, n, V, temperature, lookup):
    rng = np.random.default_rng(S * V + n)
    x, y, d, u = make(rng, S, n, V, temperature=temperature)
    xd, yd = dev_as(x, dtype), None if lookup else dev_as(y, dtype)
    lens = np.full(S, n, np.int32)
    kw = dict(temperature=temperature, uniforms=torch.from_numpy(u).to(DEV))
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, **kw)
    check(out, xd, yd, d, lens, u, np.float64(np.float32(temperature)))
    lens = rng.integers(0, n + 1, S).astype(np.int32)
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, draft_lens=torch.from_numpy(lens).to(DEV), **kw)
    check(out, xd, yd, d, lens, u, np.float64(np.float32(temperature)))


@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("S,n,V", [(700, 6, 64), (90, 64, 33), (4200, 1, 40), (8300, 0, 16)])
def test_verify_many_rows(S, n, V, lookup):
    """Calls whose rows go in two launches, the second without the sequences that have ended."""
    rng = np.random.default_rng(S)
    x, y, d, u = make(rng, S, n, V, near=0.3)
    xd, yd = dev_as(x, "bf16"), None if lookup else dev_as(y, "bf16")
    lens = rng.integers(0, n + 1, S).astype(np.int32)
    for _ in range(2):
        out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV),
                                 draft_lens=torch.from_numpy(lens).to(DEV))
        check(out, xd, yd, d, lens, u, np.float64(1.0))


@pytest.mark.parametrize("xo,yo", [(1, 0), (0, 1), (3, 5)])
@pytest.mark.parametrize("dtype,V", [("bf16", 1000), ("f32", 4097), ("f16", 20001), ("bf16", 5)])
def test_verify_rows_off_16_bytes(xo, yo, dtype, V):
    rng = np.random.default_rng(V)
    x, y, d, u = make(rng, 12, 3, V)
    xd, yd = dev_as(x, dtype, xo), dev_as(y, dtype, yo)
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV))
    check(out, xd, yd, d, np.full(12, 3), u, 1.0)


def test_verify_rows_apart():
    rng = np.random.default_rng(3)
    x, y, d, u = make(rng, 6, 2, 900)
    wide = torch.full((6, 3, 1001), float("nan"), device=DEV)
    wide[..., 5:905] = dev_as(x, "f32")
    narrow = torch.full((6, 2, 950), float("nan"), device=DEV)
    narrow[..., :900] = dev_as(y, "f32")
    xd, yd = wide[..., 5:905], narrow[..., :900]
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV))
    check(out, xd, yd, d, np.full(6, 2), u, 1.0)


def test_verify_draws_at_the_borders():
    """Draws of 0 and just below 1, and thresholds placed on the ratio p/q itself: the nearest
    f32 values around it fall on their own sides."""
    rng = np.random.default_rng(5)
    S, n, V = 64, 1, 2000
    x, y, d, u = make(rng, S, n, V)
    x[:, :, :7] = -np.inf                    # a draw of 0 passes over tokens without probability
    xd, yd = dev_as(x, "f32"), dev_as(y, "f32")
    a, b = host64(xd), host64(yd)
    for s in range(S):
        p = np.exp(a[s, 0] - a[s, 0].max())
        q = np.exp(b[s, 0] - b[s, 0].max())
        ratio = np.float32((p / p.sum())[d[s, 0]] / (q / q.sum())[d[s, 0]])
        u[s, 0] = min(np.float32(0.99999994), [ratio, np.nextafter(ratio, np.float32(0)),
                                               np.nextafter(ratio, np.float32(2))][s % 3])
    u[:, 1] = np.where(np.arange(S) % 2, 0.0, 0.99999994)
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV))
    check(out, xd, yd, d, np.full(S, n), u, 1.0)


def test_verify_equal_models_masks_and_certain_tokens():
    rng = np.random.default_rng(6)
    S, n, V = 20, 4, 3000
    x, _, d, u = make(rng, S, n, V)
    x[:, :, 100:] = -np.inf                   # a masked vocabulary
    d %= 100
    x[3, :, :] = -np.inf
    x[3, :, 42] = 0.0                         # one token has everything
    d[3] = 42
    low = x.copy()
    low[low == -np.inf] = np.finfo(np.float32).min
    for z in (x, low):
        xd = dev_as(z, "f32")
        yd = xd[:, :n].contiguous()           # the draft is the target: everything is accepted
        out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV))
        assert (out.accepted.cpu().numpy() == n).all()
        check(out, xd, yd, d, np.full(S, n), u, 1.0)
        out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), uniforms=torch.from_numpy(u).to(DEV))
        check(out, xd, None, d, np.full(S, n), u, 1.0)
    d[:, 1] = 2999                            # a drafted token that the target rules out
    xd, yd = dev_as(x, "f32"), dev_as(rng.standard_normal((S, n, V)), "f32")
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV))
    check(out, xd, yd, d, np.full(S, n), u, 1.0)
    assert (out.accepted.cpu().numpy() <= 1).all()


def test_verify_text_follows_the_target():
    """65,000 sequences from one pair of rows: the first token's counts follow the target's
    probabilities whatever the draft (binomial, 5.5 standard deviations for 16 tokens)."""
    rng = np.random.default_rng(7)
    S, V = 65000, 16
    x, y = rng.standard_normal((1, 2, V)) * 1.5, rng.standard_normal((1, 1, V)) * 1.5
    xd = dev_as(np.repeat(x, S, 0), "f32")
    yd = dev_as(np.repeat(y, S, 0), "f32")
    q = np.exp(host64(yd)[0, 0])
    d = rng.choice(V, size=(S, 1), p=q / q.sum())
    u = rng.random((S, 2), dtype=np.float32)
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV))
    p = np.exp(host64(xd)[0, 0])
    p /= p.sum()
    got = np.bincount(out.tokens[:, 0].cpu().numpy(), minlength=V)
    assert (np.abs(got - S * p) <= 5.5 * np.sqrt(S * p * (1 - p))).all()


def test_verify_reports_bad_input_and_leaves_the_other_sequences():
    rng = np.random.default_rng(8)
    S, n, V = 5, 3, 1200
    x, y, d, u = make(rng, S, n, V)
    u[:, :n] = 0.0                            # everything is accepted
    ud = torch.from_numpy(u).to(DEV)
    clean = step.verify_drafts(dev_as(x, "f32"), torch.from_numpy(d).to(DEV), dev_as(y, "f32"), uniforms=ud)
    assert (clean.accepted.cpu().numpy() == n).all()

    def bad(code, change, lens=None):
        x2, y2, d2 = x.copy(), y.copy(), d.copy()
        change(x2, y2, d2)
        ctx = grpo.Context(0)
        out = step.verify_drafts(dev_as(x2, "f32"), torch.from_numpy(d2).to(DEV), dev_as(y2, "f32"), uniforms=ud,
                                 draft_lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV),
                                 sync=False, ctx=ctx)
        with pytest.raises(PcpError) as e:
            ctx.sync()
        assert e.value.code == code
        for s in (0, 1, 3, 4):
            assert torch.equal(out.tokens[s], clean.tokens[s]) and torch.equal(out.logp[s], clean.logp[s])
        return out.tokens[2].cpu().numpy(), int(out.accepted[2])

    t, j = bad(-3, lambda x2, y2, d2: d2.__setitem__((2, 1), V))
    assert j == 1 and t[0] == d[2, 0] and 0 <= t[1] < V and (t[2:] == IGNORE).all()
    _, j = bad(-3, lambda x2, y2, d2: d2.__setitem__((2, 0), -100))
    assert j == 0
    t, j = bad(-4, lambda x2, y2, d2: x2.__setitem__((2, 1, 5), np.nan))
    assert j == 1 and t[1] == V - 1
    t, j = bad(-4, lambda x2, y2, d2: x2.__setitem__((2, 3, 5), np.inf))
    assert j == 3 and t[3] == V - 1
    t, j = bad(-4, lambda x2, y2, d2: y2.__setitem__((2, 2), -np.inf))
    assert j == 2 and 0 <= t[2] < V
    _, j = bad(-1, lambda x2, y2, d2: None, lens=[n, n, n + 4, n, n])
    assert j == n
    _, j = bad(-1, lambda x2, y2, d2: None, lens=[n, n, -2, n, n])
    assert j == 0
    # A row past the end of the text is not looked at.
    x2 = x.copy()
    x2[2, 3] = np.nan
    u2 = u.copy()
    d2 = d.copy()
    x2[2, 1, d[2, 1]] = -np.inf
    out = step.verify_drafts(dev_as(x2, "f32"), torch.from_numpy(d2).to(DEV), dev_as(y, "f32"),
                             uniforms=torch.from_numpy(u2).to(DEV))
    assert int(out.accepted[2]) == 1


def test_verify_offsets_past_32_bits():
    """2.2e9 target logits, rows apart: the last sequence reads its own."""
    rng = np.random.default_rng(9)
    V, S, n = 60000, 3, 2
    x, y, d, u = make(rng, S, n, V)
    apart = 240_000_000
    wide = torch.empty(9 * apart, dtype=torch.bfloat16, device=DEV)
    wide.fill_(float("nan"))
    xd = wide.view(3, 3, apart)[..., :V]
    xd.copy_(dev_as(x, "bf16"))
    yd = dev_as(y, "bf16")
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, uniforms=torch.from_numpy(u).to(DEV))
    check(out, xd, yd, d, np.full(S, n), u, 1.0)


def test_verify_captured_and_repeated():
    rng = np.random.default_rng(10)
    S, n, V = 6, 4, 20000
    ctx = grpo.Context(0)
    x, y, d, u = make(rng, S, n, V)
    xd, yd, dd, ud = dev_as(x, "bf16"), dev_as(y, "bf16"), torch.from_numpy(d).to(DEV), torch.from_numpy(u).to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = step.verify_drafts(xd, dd, yd, uniforms=ud, stream=s, sync=False, ctx=ctx)
    s.synchronize()
    cold = grpo.Context(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step.verify_drafts(xd, dd, yd, uniforms=ud, outputs=out, sync=False, ctx=ctx)
        with pytest.raises(PcpError) as e:
            step.verify_drafts(xd, dd, yd, uniforms=ud, outputs=out, sync=False, ctx=cold)
    assert e.value.code == -1 and "captured" in str(e.value)
    for _ in range(4):
        x, y, d, u = make(rng, S, n, V)
        xd.copy_(dev_as(x, "bf16")); yd.copy_(dev_as(y, "bf16"))
        dd.copy_(torch.from_numpy(d)); ud.copy_(torch.from_numpy(u))
        g.replay()
        torch.cuda.synchronize()
        check(out, xd, yd, d, np.full(S, n), u, 1.0)
        again = step.verify_drafts(xd, dd, yd, uniforms=ud)
        assert torch.equal(again.tokens, out.tokens) and torch.equal(again.logp, out.logp)
    ctx.sync()


def test_verified_log_probs_are_the_loss_heads():
    """As the calls are used together: the verified tokens with their log-probs are what the
    loss takes as ids and old_logp, and the policy's own log-probs agree with them."""
    rng = np.random.default_rng(11)
    S, n, V = 4, 5, 5000
    x, y, d, u = make(rng, S, n, V)
    xd = dev_as(x, "f32")
    out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), dev_as(y, "f32"), uniforms=torch.from_numpy(u).to(DEV))
    logp, _ = grpo.logprob_fwd(xd, out.tokens)
    assert (np.abs(host64(logp) - host64(out.logp)) <= 1e-5 * 12).all()
    mask = (out.tokens >= 0).float()
    loss = grpo.grpo_loss_fwd_bwd(xd, out.tokens, mask, advantages=torch.ones(S, device=DEV), ref_logits=xd.clone(),
                                  old_logp=out.logp, loss_mode=grpo.LossMode.GRPO_CLIP_KL)
    assert abs(float(loss.loss) + 1.0) <= 1e-4          # every ratio is 1 and the policy its own reference
