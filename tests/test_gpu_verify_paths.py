"""Draft verification by number of sequences: with few the last workgroup of a sequence's residual
picks its token, by counters that are zero again after each call; with many the rows go in two
launches. Captured and replayed, with bad rows and clean calls after them, and with every one of
64 drafted tokens accepted."""
import numpy as np
import pytest
import torch

from distill_ref import IGNORE, verify_ref
from pcp_amd import grpo, step
from pcp_amd._lib import PcpError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def make(rng, S, n, V):
    x = rng.standard_normal((S, n + 1, V)).astype(np.float32) * 3
    y = x[:, :n] + 0.7 * rng.standard_normal((S, n, V)).astype(np.float32)
    d = np.argmax(y.astype(np.float64) + rng.gumbel(size=y.shape), -1).astype(np.int64).reshape(S, n)
    return x, y, d, rng.random((S, n + 1)).astype(np.float32)


def on_gpu(*arrays):
    return [torch.from_numpy(a).to(DEV) for a in arrays]


def check(out, x, y, d, u, rows=slice(None)):
    S, n = d.shape
    want = verify_ref(x.astype(np.float64), None if y is None else y.astype(np.float64), d, np.full(S, n), u, 1.0, x.shape[-1])
    assert np.array_equal(out.accepted.cpu().numpy()[rows], want[1][rows])
    assert np.array_equal(out.tokens.cpu().numpy()[rows], want[0][rows])
    lp = out.logp.double().cpu().numpy()
    assert (np.abs(lp - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 1e-12)[rows].all()


@pytest.mark.parametrize("S,V", [(1, 20000), (2, 20000), (4, 20000), (5, 20000), (6, 20000), (16, 20000), (17, 20000),
                                 (96, 500), (97, 500), (12, 8000), (13, 8000)])
@pytest.mark.parametrize("lookup", [False, True])
def test_captured_and_replayed(S, V, lookup):
    rng = np.random.default_rng(S)
    n = 3
    ctx, cold = grpo.Context(0), grpo.Context(0)
    x, y, d, u = on_gpu(*make(rng, S, n, V))
    draft = None if lookup else y
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = step.verify_drafts(x, d, draft, uniforms=u, stream=s, sync=False, ctx=ctx)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step.verify_drafts(x, d, draft, uniforms=u, outputs=out, sync=False, ctx=ctx)
        with pytest.raises(PcpError, match="captured"):
            step.verify_drafts(x, d, draft, uniforms=u, outputs=out, sync=False, ctx=cold)
    for _ in range(4):
        new = make(rng, S, n, V)
        for t, a in zip((x, y, d, u), new):
            t.copy_(torch.from_numpy(a))
        g.replay()
        torch.cuda.synchronize()
        check(out, new[0], None if lookup else new[1], new[2], new[3])
        again = step.verify_drafts(x, d, draft, uniforms=u, ctx=ctx)     # eager, by the same counters
        assert torch.equal(again.tokens, out.tokens) and torch.equal(again.logp, out.logp)
    ctx.sync()


def test_counters_made_under_capture_are_refused():
    """A context that has run only calls of many sequences has no counters yet."""
    rng = np.random.default_rng(1)
    n, V = 2, 3000
    many = 40
    ctx, s, g = grpo.Context(0), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    x, y, d, u = on_gpu(*make(rng, many, n, V))
    out = step.verify_drafts(x, d, y, uniforms=u, ctx=ctx)
    few = step.verify_drafts(x[:2], d[:2], y[:2], uniforms=u[:2])
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        step.verify_drafts(x, d, y, uniforms=u, outputs=out, sync=False, ctx=ctx)
        with pytest.raises(PcpError, match="captured"):
            step.verify_drafts(x[:2], d[:2], y[:2], uniforms=u[:2], outputs=few, sync=False, ctx=ctx)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(few.tokens, out.tokens[:2]) and torch.equal(few.logp, out.logp[:2])


@pytest.mark.parametrize("S", [1, 4, 10, 11])
@pytest.mark.parametrize("bad_row", ["target", "draft", "after", "token"])
def test_clean_calls_after_bad_ones(S, bad_row):
    """A bad row ends its sequence before the counters; the calls after it on the same context are right."""
    rng = np.random.default_rng(S)
    n, V = 3, 9000
    ctx = grpo.Context(0)
    x, y, d, u = make(rng, S, n, V)
    u[:, :n] = 0.0                              # all accepted
    bx, by, bd = x.copy(), y.copy(), d.copy()
    at = S - 1
    if bad_row == "target":
        bx[at, 1, 77] = np.nan
    elif bad_row == "draft":
        by[at, 1] = -np.inf
    elif bad_row == "after":
        bx[at, n, 5] = np.inf
    else:
        bd[at, 2] = V
    for _ in range(3):
        ax, ay, ad, au = on_gpu(bx, by, bd, u)
        out = step.verify_drafts(ax, ad, ay, uniforms=au, sync=False, ctx=ctx)
        with pytest.raises(PcpError) as e:
            ctx.sync()
        assert e.value.code == (-3 if bad_row == "token" else -4)
        j = {"target": 1, "draft": 1, "after": n, "token": 2}[bad_row]
        t = out.tokens[at].cpu().numpy()
        assert int(out.accepted[at]) == j and np.array_equal(t[:j], d[at, :j]) and (t[j + 1:] == IGNORE).all()
        assert t[j] == V - 1 if bad_row in ("target", "after") else 0 <= t[j] < V
        if S > 1:
            check(out, x, y, d, u, slice(0, S - 1))
        cx, cy, cd, cu = on_gpu(x, y, d, u)
        check(step.verify_drafts(cx, cd, cy, uniforms=cu, ctx=ctx), x, y, d, u)


@pytest.mark.parametrize("S", [1, 5])
@pytest.mark.parametrize("kind", ["model", "lookup", "greedy"])
def test_all_of_64_accepted(S, kind):
    rng = np.random.default_rng(64)
    n, V = 64, 700
    x, y, _, u = make(rng, S, n, V)
    d = np.argmax(x[:, :n], -1).astype(np.int64)
    u[:, :n] = 0.0
    xd, yd, dd, ud = on_gpu(x, y, d, u)
    if kind == "greedy":
        out = step.verify_drafts(xd, dd, temperature=0.0)
        assert np.array_equal(out.tokens[:, n].cpu().numpy(), np.argmax(x[:, n], -1)) and not out.logp.any()
    else:
        out = step.verify_drafts(xd, dd, yd if kind == "model" else None, uniforms=ud)
        check(out, x, y if kind == "model" else None, d, u)
    assert (out.accepted.cpu().numpy() == n).all() and np.array_equal(out.tokens[:, :n].cpu().numpy(), d)
    # The last one refused: 63 accepted.
    d[:, n - 1] = np.argmin(x[:, n - 1], -1)
    u[:, n - 1] = 0.999
    dd, ud = on_gpu(d, u)
    out = (step.verify_drafts(xd, dd, temperature=0.0) if kind == "greedy" else
           step.verify_drafts(xd, dd, yd if kind == "model" else None, uniforms=ud))
    if kind == "greedy":
        assert (out.accepted.cpu().numpy() == n - 1).all()
        assert np.array_equal(out.tokens[:, n - 1].cpu().numpy(), np.argmax(x[:, n - 1], -1))
        assert (out.tokens[:, n] == IGNORE).all()
    else:
        check(out, x, y if kind == "model" else None, d, u)


@pytest.mark.parametrize("lookup", [False, True])
@pytest.mark.parametrize("S,n,V", [(1300, 6, 64), (130, 64, 33), (5500, 1, 40), (300, 6, 9000), (3, 2, 700)])
def test_rows_in_two_launches(S, n, V, lookup):
    """Calls on both sides of the number of rows from which those of ended sequences are left out."""
    rng = np.random.default_rng(S)
    x, y, d, u = make(rng, S, n, V)
    xd, yd, dd, ud = on_gpu(x, y, d, u)
    for _ in range(2):
        check(step.verify_drafts(xd, dd, None if lookup else yd, uniforms=ud), x, None if lookup else y, d, u)
