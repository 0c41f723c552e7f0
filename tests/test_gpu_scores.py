"""Token scores and their gradient on the GPU against their definitions in 64 bits (tests/score_ref.py, which also
derives the bars)."""
import numpy as np
import pytest
import torch

from pcp_amd import grpo, scores
from pcp_amd._lib import PcpError
from score_ref import IGNORE, bars, close, grad_ref, half_step, score_ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def to_dev(x, dtype, offset=0):
    """x in `dtype` on the GPU, its first element `offset` elements past an aligned address."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(DT[dtype])
    buf = torch.empty(t.numel() + offset, dtype=t.dtype, device=DEV)
    v = buf[offset:].view(t.shape)
    v.copy_(t)
    return v


def dev(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).to(DEV)


def host64(t):
    return t.detach().double().cpu().numpy()


def rows_like_a_model(rng, shape, scale=3.0):
    x = rng.standard_normal(shape).astype(np.float32) * scale
    for r in x.reshape(-1, shape[-1]):
        n = min(6, shape[-1])
        r[rng.choice(shape[-1], n, replace=False)] += rng.random(n).astype(np.float32) * 12
    return x


def check_scores(x, ids, out, tau, k, live=None):
    """x [R, V] device logits, out's arrays flattened to [R, ...]."""
    R = len(x)
    live = np.ones(R, bool) if live is None else live
    logp, h, m, log_sum, tlp, tid = score_ref(host64(x)[live], None if ids is None else np.asarray(ids)[live], tau, k)
    got = {n: getattr(out, n) for n in ("logp", "entropy", "row_max", "log_sum", "top_logp", "top_ids")}
    got = {n: None if t is None else host64(t).reshape(R, -1) for n, t in got.items()}
    bar = bars(h)
    if ids is not None:
        close(got["logp"][live, 0], logp, bar)
    close(got["entropy"][live, 0], h, bar)
    assert np.array_equal(got["row_max"][live, 0], m)
    close(got["log_sum"][live, 0], log_sum, bar)
    if k:
        assert np.array_equal(got["top_ids"][live], tid)
        close(got["top_logp"][live], tlp, bar[:, None])
        assert (got["top_ids"][~live] == IGNORE).all()
    for n, t in got.items():
        if t is not None and n != "top_ids":
            assert (t[~live] == 0).all(), n


SHAPES = [("f32", 1, 1, 1), ("bf16", 3, 7, 7), ("f16", 5, 64, 64), ("f32", 4, 255, 20), ("bf16", 6, 1000, 256),
          ("bf16", 2, 1003, 65), ("f32", 3, 8191, 128), ("bf16", 5, 16385, 256), ("f16", 2, 50257, 33),
          ("f32", 2, 50257, 256), ("bf16", 1, 151936, 20), ("bf16", 300, 16000, 8), ("f32", 511, 9000, 3),
          ("f32", 512, 9000, 3), ("bf16", 513, 20000, 1), ("bf16", 2, 262144, 256), ("f16", 2049, 4096, 64), ("f32", 515, 151936, 30), ("f32", 64, 151936, 5), ("bf16", 100, 151936, 33),
          ("f16", 255, 50257, 17), ("bf16", 128, 32768, 0), ("f32", 3, 600000, 77)]


@pytest.mark.parametrize("dtype,R,V,k", SHAPES)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("top", [False, True])
def test_scores(dtype, R, V, k, offset, top):
    rng = np.random.default_rng(R * V + k)
    x = to_dev(rows_like_a_model(rng, (R, V)), dtype, offset)
    ids = rng.integers(0, V, R)
    tau = 1.0 if top else 0.75
    k = k if top else 0
    out = scores.token_scores(x[None], dev(ids[None], torch.int64), k=k, temperature=tau)
    check_scores(x, ids, out, tau, k)


KINDS = ["equal", "rising", "falling", "two_values", "one_left", "few_left", "zeros", "peaked", "lowest", "far", "far_below"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("R,V,k", [(2, 40000, 12), (2, 40000, 0), (600, 5000, 40), (600, 5000, 0)])
@pytest.mark.parametrize("tau", [1.0, 0.3])
def test_scores_of_odd_rows(kind, dtype, R, V, k, tau):
    """Rows of equal values, of masks and nearly nothing else, peaked so that the entropy is next to 0, and far from zero."""
    rng = np.random.default_rng(7)
    x = np.zeros((R, V), np.float32)
    low = float(torch.finfo(DT[dtype]).min)
    if kind == "equal":
        x[:] = -1.5
    elif kind == "rising":
        x[:] = np.linspace(-20, 20, V)
    elif kind == "falling":
        x[:] = np.linspace(20, -20, V)
    elif kind == "two_values":
        x[:] = rng.integers(0, 2, (R, V))
    elif kind in ("one_left", "few_left"):
        x[:] = -np.inf
        n = 1 if kind == "one_left" else 7
        for r in range(R):
            x[r, rng.choice(V, n, replace=False)] = rng.standard_normal(n)
    elif kind == "zeros":
        x[:] = np.where(rng.random((R, V)) < 0.5, 0.0, -0.0)   # both zeros are one value
    elif kind == "peaked":
        x[:] = rng.standard_normal((R, V)) * 0.1 - 20
        x[np.arange(R), rng.integers(0, V, R)] = 3.0
    elif kind == "lowest":
        x[:] = low                                             # nothing but masks: uniform
        x[1::2] = rows_like_a_model(rng, x[1::2].shape)
        x[1::2, V // 3:] = low
    elif kind == "far":
        x[:] = rng.standard_normal((R, V)) * 2 + (30000 if dtype != "f16" else 3000)
    else:
        x[:] = rng.standard_normal((R, V)) * 2 - (1e30 if dtype != "f16" else 60000)
    x = to_dev(x, dtype)
    ids = rng.integers(0, V, R)
    ids[0] = int(x[0].argmax())
    out = scores.token_scores(x[:, None], dev(ids[:, None], torch.int32), k=k, temperature=tau, top_ids_dtype=torch.int64)
    check_scores(x, ids, out, tau, k)


@pytest.mark.parametrize("R,V,k,left", [(2, 40000, 20, 3), (600, 5000, 9, 2), (1, 151936, 64, 64), (520, 20000, 5, 0), (3, 300, 256, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_fewer_tokens_left_than_alternatives(dtype, R, V, k, left):
    """Rows of two kinds of masks, of one, and with the unmasked ones spread over every part."""
    rng = np.random.default_rng(V + left)
    x = np.full((R, V), -1e30, np.float32)
    x[::2][rng.random(x[::2].shape) < 0.5] = -np.inf
    if R == 1:
        x[:] = -np.inf
    for r in range(R):
        n = max(left, 1)
        x[r, rng.choice(V, n, replace=False)] = rng.standard_normal(n)
    x = to_dev(x, dtype, 1)
    ids = rng.integers(0, V, R)
    out = scores.token_scores(x[:, None], dev(ids[:, None], torch.int64), k=k)
    check_scores(x, ids, out, 1.0, k)


@pytest.mark.parametrize("mask_dtype", [torch.float32, torch.bool])
@pytest.mark.parametrize("S,T,V,k,shift", [(3, 9, 1003, 5, 1), (2, 5, 70000, 3, 0), (40, 20, 333, 0, 1), (64, 1, 30000, 2, 0)])
def test_layout_masks_and_ignored_tokens(mask_dtype, S, T, V, k, shift):
    """The shifted layout in padded rows; masked, ignored and unaddressed tokens; buffers given keep what no row addresses."""
    rng = np.random.default_rng(S + T)
    TS, rows = T + 2, T - shift
    wide = to_dev(rows_like_a_model(rng, (S, T + 3, V + 5)), "bf16")
    x = wide[:, 3:, 2:V + 2]
    ids = rng.integers(0, V, (S, TS))
    ids[rng.random((S, TS)) < 0.2] = IGNORE
    mask = rng.random((S, TS)) < 0.7
    ids[~mask & (rng.random((S, TS)) < 0.3)] = V + 3           # out of range, but weighs nothing
    mask[0] = False
    kept = scores.TokenScores(*(torch.full((S, TS), 7.0, device=DEV) for _ in range(4)),
                              torch.full((S, TS, k), 7.0, device=DEV) if k else None,
                              torch.full((S, TS, k), 7, dtype=torch.int32, device=DEV) if k else None)
    off = 1 + shift
    out = scores.token_scores(x, dev(ids, torch.int64), dev(mask, mask_dtype), k=k, rows=rows, tok_offset=off, outputs=kept)
    assert out is kept
    sel = slice(off, off + rows)
    part = scores.TokenScores(*(None if t is None else t[:, sel].reshape(S * rows, -1) for t in (
        out.logp, out.entropy, out.row_max, out.log_sum, out.top_logp, out.top_ids)))
    live = (mask & (ids != IGNORE))[:, sel].reshape(-1)
    check_scores(x[:, :rows].reshape(S * rows, V), ids[:, sel].reshape(-1), part, 1.0, k, live)
    for t in (out.logp, out.entropy, out.row_max, out.log_sum) + ((out.top_logp, out.top_ids) if k else ()):
        assert (t[:, :off] == 7).all() and (t[:, off + rows:] == 7).all()


@pytest.mark.parametrize("dtype,R,V,k", [("bf16", 1, 1 << 24, 40), ("f32", 520, 600000, 70), ("f16", 3, 5000001, 256)])
def test_long_rows(dtype, R, V, k):
    """Groups of several batches a lane, and the largest vocabulary; a few rows are checked."""
    g = torch.Generator(device=DEV).manual_seed(R)
    x = torch.empty((R, V), dtype=DT[dtype], device=DEV)
    for r in range(R):
        x[r] = (torch.randn(V, generator=g, device=DEV) * 2).to(DT[dtype])
    x[:, V // 3] = 11.0
    x[:, V - 1] = 10.5
    ids = torch.randint(0, V, (R, 1), generator=g, device=DEV)
    out = scores.token_scores(x[:, None], ids, k=k)
    picked = sorted({0, R // 2, R - 1})
    check_scores(x[picked], ids[picked, 0].cpu().numpy(), scores.TokenScores(*(t[picked] for t in (
        out.logp, out.entropy, out.row_max, out.log_sum, out.top_logp, out.top_ids))), 1.0, k)


def test_views_and_entropy_alone():
    """A stack of decode steps, transposed; the last rows of longer ones; no tokens; no rows at all."""
    rng = np.random.default_rng(2)
    steps = to_dev(rows_like_a_model(rng, (5, 3, 777)), "f16")
    ids = rng.integers(0, 777, (3, 5))
    x = steps.transpose(0, 1)
    out = scores.token_scores(x, dev(ids, torch.int64), k=4)
    check_scores(x.reshape(15, 777), ids.reshape(-1), out, 1.0, 4)
    out = scores.token_scores(x[:, -2:], k=0)
    assert out.logp is None
    check_scores(x[:, -2:].reshape(6, 777), None, out, 1.0, 0)
    assert scores.token_scores(x[:, :0], dev(ids[:, :0], torch.int64), k=3).top_ids.shape == (3, 0, 3)
    assert scores.token_scores(x[:0], dev(ids[:0], torch.int64)).entropy.shape == (0, 5)


def test_offsets_past_32_bits():
    R, V = 14500, 151936                      # 2.2e9 elements
    rng = np.random.default_rng(1)
    x = torch.empty((R, V), dtype=torch.bfloat16, device=DEV)
    x.fill_(-3.0)
    last = to_dev(rows_like_a_model(rng, (2, V)), "bf16")
    x[-2:] = last
    ids = torch.zeros((1, R), dtype=torch.int64, device=DEV)
    for k in (0, 3):
        out = scores.token_scores(x[None], ids, k=k)
        check_scores(last, [0, 0], scores.TokenScores(*(None if t is None else t[0, -2:] for t in (
            out.logp, out.entropy, out.row_max, out.log_sum, out.top_logp, out.top_ids))), 1.0, k)
        assert (out.entropy[0, :-2] - np.log(V)).abs().max() < 1e-4
    scores.token_scores_bwd(x[None], ids, out.row_max, out.log_sum, out.entropy, dlogp=torch.ones_like(out.logp),
                            dentropy=torch.ones_like(out.logp), dlogits=x[None])   # in place
    g, bar = grad_ref(host64(last), [0, 0], [1, 1], [1, 1])
    got = host64(x[-2:])
    assert (np.abs(got - g) <= bar + half_step(np.abs(g) + bar, "bf16")).all()
    first = host64(x[0])
    assert abs(first[0] - (1 - 1 / V)) < 2.0 ** -8 and np.abs(first[1:] + 1 / V).max() < 2.0 ** -8 / V + 1e-9


def test_more_rows_than_a_grid_dimension():
    rng = np.random.default_rng(4)
    R, V = 70001, 9
    x = to_dev(rng.standard_normal((R, V)) * 3, "f32")
    ids = rng.integers(0, V, R)
    out = scores.token_scores(x.view(R, 1, V), dev(ids[:, None], torch.int64), k=2)
    check_scores(x, ids, out, 1.0, 2)


def bad_calls():
    x = torch.randn(4, 6, 500, device=DEV)
    ids = torch.randint(0, 500, (4, 6), device=DEV)
    return x, ids


@pytest.mark.parametrize("k", [0, 5])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), "all"])
def test_rows_without_a_finite_sum_are_reported(k, bad):
    x, ids = bad_calls()
    want = scores.token_scores(x, ids, k=k)
    y = x.clone()
    if bad == "all":
        y[2, 3] = -float("inf")
    else:
        y[2, 3, 77] = bad
    ctx = grpo.Context(0)
    out = scores.token_scores(y, ids, k=k, sync=False, ctx=ctx)
    with pytest.raises(PcpError) as e:
        ctx.sync()
    assert e.value.code == -4
    other = torch.ones(4, 6, dtype=torch.bool, device=DEV)
    other[2, 3] = False
    assert torch.equal(out.entropy[other], want.entropy[other]) and torch.equal(out.logp[other], want.logp[other])
    g = scores.token_scores_bwd(y, ids, out.row_max, out.log_sum, out.entropy, dlogp=other.float(), mask=other, ctx=ctx)
    assert torch.isfinite(g).all()                      # the row is not read
    with pytest.raises(PcpError) as e:
        scores.token_scores_bwd(y, ids, out.row_max, out.log_sum, out.entropy, dentropy=torch.ones(4, 6, device=DEV), ctx=ctx)
    assert e.value.code == -4
    scores.token_scores(x, ids, k=k, ctx=ctx)           # nothing is left behind


def test_a_bad_token_is_reported_and_its_row_left_out():
    x, ids = bad_calls()
    ids[1, 2] = 500
    ctx = grpo.Context(0)
    out = scores.token_scores(x, ids, k=2, sync=False, ctx=ctx)
    with pytest.raises(PcpError) as e:
        ctx.sync()
    assert e.value.code == -3 and out.entropy[1, 2] == 0 and (out.top_ids[1, 2] == IGNORE).all()
    w = torch.ones(4, 6, device=DEV)
    g = scores.token_scores_bwd(x, ids, out.row_max, out.log_sum, out.entropy, dlogp=w, sync=False, ctx=ctx)
    with pytest.raises(PcpError) as e:
        ctx.sync()
    assert e.value.code == -3 and (g[1, 2] == 0).all() and (g[1, 1] != 0).any()


GRADS = [("f32", "f32", 2, 3, 1, 0), ("bf16", "bf16", 3, 4, 7, 0), ("f16", "f32", 2, 5, 1003, 1), ("bf16", "f32", 4, 6, 50257, 1),
         ("f16", "f16", 3, 3, 4099, 0), ("f32", "f32", 2, 2, 151936, 0), ("bf16", "bf16", 2, 33, 20000, 1),
         ("bf16", "bf16", 1, 1, 151937, 0), ("bf16", "f32", 3, 7, 33, 1)]


@pytest.mark.parametrize("dtype,out,S,T,V,shift", GRADS)
@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("tau", [1.0, 0.6])
def test_gradient(dtype, out, S, T, V, shift, offset, accumulate, tau):
    rng = np.random.default_rng(S * T * V + shift)
    host = rows_like_a_model(rng, (S, T, V))
    host[rng.random(host.shape) < 0.1] = -np.inf
    host[..., V // 2] = 1.0
    x = to_dev(host, dtype, offset)
    rows = T - shift
    ids = rng.integers(0, V, (S, T))
    ids[rng.random((S, T)) < 0.15] = IGNORE
    mask = rng.random((S, T)) < 0.8
    d_ids, d_mask = dev(ids, torch.int64), dev(mask, torch.float32)
    sc = scores.token_scores(x, d_ids, d_mask, temperature=tau, rows=rows, tok_offset=shift)
    gl, gh = rng.standard_normal((S, T)).astype(np.float32), rng.standard_normal((S, T)).astype(np.float32)
    gl[rng.random((S, T)) < 0.3] = 0
    gh[rng.random((S, T)) < 0.3] = 0
    base = to_dev(rng.standard_normal((S, T, V)) * 0.01, out, 5)
    had = host64(base)
    got = scores.token_scores_bwd(x, d_ids, sc.row_max, sc.log_sum, sc.entropy, dlogp=dev(gl, torch.float32),
                                  dentropy=dev(gh, torch.float32), mask=d_mask, temperature=tau, rows=rows, tok_offset=shift,
                                  dlogits=base, accumulate=accumulate)
    assert got is base
    got = host64(got)
    live = (mask & (ids != IGNORE) & ((gl != 0) | (gh != 0)))[:, shift:]
    want = had.copy() if accumulate else np.zeros_like(had)
    lim = np.zeros_like(had)
    for s in range(S):
        r = np.flatnonzero(live[s])
        if len(r) == 0:
            continue
        g, bar = grad_ref(host64(x[s])[r], ids[s, shift + r], gl[s, shift + r], gh[s, shift + r], tau)
        want[s, r] += g
        if accumulate:
            bar = bar + 2.0 ** -24 * (np.abs(want[s, r]) + bar)
        lim[s, r] = bar + half_step(np.abs(want[s, r]) + bar, out)
    err = np.abs(got - want)
    assert (err <= lim).all(), (err - lim).max()


def test_gradient_in_place_and_strided():
    """Over the logits, in rows of a padded vocabulary; into rows of another stride; entropy alone, log-probs alone."""
    rng = np.random.default_rng(9)
    S, T, V = 3, 4, 1001
    wide = to_dev(rows_like_a_model(rng, (S, T, V + 7)), "bf16")
    x = wide[..., :V]
    keep = wide.clone()
    ids = dev(rng.integers(0, V, (S, T)), torch.int32)
    sc = scores.token_scores(x, ids)
    w = dev(rng.standard_normal((S, T)), torch.float32)
    plain = scores.token_scores_bwd(x, ids, sc.row_max, sc.log_sum, sc.entropy, dlogp=w, dentropy=w)
    apart = torch.full((T, S, V + 2), 5.0, dtype=torch.bfloat16, device=DEV)
    scores.token_scores_bwd(x, ids, sc.row_max, sc.log_sum, sc.entropy, dlogp=w, dentropy=w,
                            dlogits=apart.transpose(0, 1)[..., 1:V + 1])
    assert torch.equal(apart.transpose(0, 1)[..., 1:V + 1], plain)
    assert (apart[..., 0] == 5).all() and (apart[..., V + 1] == 5).all()
    a = scores.token_scores_bwd(x, ids, sc.row_max, sc.log_sum, dlogp=w, dlogits_dtype=torch.float32)
    b = scores.token_scores_bwd(x, None, sc.row_max, sc.log_sum, sc.entropy, dentropy=w, dlogits_dtype=torch.float32)
    g, bar = grad_ref(host64(x).reshape(-1, V), ids.cpu().numpy().reshape(-1), host64(w).reshape(-1), 0 * host64(w).reshape(-1))
    assert (np.abs(host64(a).reshape(-1, V) - g) <= bar + half_step(np.abs(g) + bar, "f32")).all()
    g, bar = grad_ref(host64(x).reshape(-1, V), None, 0 * host64(w).reshape(-1), host64(w).reshape(-1))
    assert (np.abs(host64(b).reshape(-1, V) - g) <= bar + half_step(np.abs(g) + bar, "f32")).all()
    scores.token_scores_bwd(x, ids, sc.row_max, sc.log_sum, sc.entropy, dlogp=w, dentropy=w, dlogits=x)
    assert torch.equal(x, plain) and torch.equal(wide[..., V:], keep[..., V:])
    with pytest.raises(PcpError):
        scores.token_scores_bwd(x, ids, sc.row_max, sc.log_sum, dlogp=w, dlogits=wide[..., 7:])


@pytest.mark.parametrize("k,S,V", [(0, 3, 151936), (9, 3, 151936), (4, 700, 5000)])
def test_the_same_call_gives_the_same_bits(k, S, V):
    torch.manual_seed(0)
    x = (torch.randn(S, 1, V, device=DEV) * 3).to(torch.bfloat16)
    ids = torch.randint(0, V, (S, 1), device=DEV)
    a = scores.token_scores(x, ids, k=k)
    for _ in range(5):
        b = scores.token_scores(x, ids, k=k)
        for n in ("logp", "entropy", "row_max", "log_sum", "top_logp", "top_ids"):
            if getattr(a, n) is not None:
                assert torch.equal(getattr(a, n), getattr(b, n)), n


def test_rows_beside_the_number_of_tickets():
    """As many rows as may be dealt to several workgroups, and one more; the context's other buffers stay as they are."""
    from pcp_amd import step
    ctx = grpo.Context(0)
    g = torch.randn(1 << 20, device=DEV)
    want = step.grad_norm(g, ctx=ctx)
    torch.manual_seed(1)
    for rows in (1, 100, 255, 256, 257, 511, 512, 4096):
        x = torch.randn(rows, 1, 20000, device=DEV).to(torch.bfloat16)
        ids = torch.randint(0, 20000, (rows, 1), device=DEV)
        for _ in range(3):
            out = scores.token_scores(x, ids, k=3, ctx=ctx)
        picked = [0, rows // 2, rows - 1]
        check_scores(x[picked, 0], ids[picked, 0].cpu().numpy(), scores.TokenScores(*(t[picked] for t in (
            out.logp, out.entropy, out.row_max, out.log_sum, out.top_logp, out.top_ids))), 1.0, 3)
        got = step.grad_norm(g, ctx=ctx)
        assert torch.equal(got.norm, want.norm)


@pytest.mark.parametrize("which", ["dlogp", "dentropy", "row_max", "entropy"])
def test_a_gradient_or_statistic_that_is_not_finite_is_reported(which):
    x, ids = bad_calls()
    ctx = grpo.Context(0)
    sc = scores.token_scores(x, ids, ctx=ctx)
    a = dict(row_max=sc.row_max, log_sum=sc.log_sum, entropy=sc.entropy, dlogp=torch.ones(4, 6, device=DEV),
             dentropy=torch.ones(4, 6, device=DEV))
    a[which] = a[which].clone()
    a[which][2, 1] = float("nan")
    d = torch.zeros_like(x)
    with pytest.raises(PcpError) as e:
        scores.token_scores_bwd(x, ids, dlogits=d, ctx=ctx, **a)
    assert e.value.code == -4 and torch.isnan(d[2, 1]).all()
    d[2, 1] = 0
    assert torch.isfinite(d).all()


def test_captured_calls_and_other_streams():
    """Forward and gradient in one graph, replayed on new inputs with eager work of another size between; a stream of its
    own; two contexts whose graphs overlap."""
    V, S = 60000, 5
    ctxs = [grpo.Context(0), grpo.Context(0)]
    sets = []
    for i, ctx in enumerate(ctxs):
        torch.manual_seed(i)
        x = torch.randn(S, 2, V, device=DEV)
        ids = torch.randint(0, V, (S, 2), device=DEV)
        w = torch.randn(S, 2, device=DEV)
        out = scores.token_scores(x, ids, k=6, ctx=ctx)
        d = scores.token_scores_bwd(x, ids, out.row_max, out.log_sum, out.entropy, dlogp=w, dentropy=w, ctx=ctx)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            scores.token_scores(x, ids, k=6, outputs=out, sync=False, ctx=ctx)
            scores.token_scores_bwd(x, ids, out.row_max, out.log_sum, out.entropy, dlogp=w, dentropy=w, dlogits=d, sync=False,
                                    ctx=ctx)
        sets.append((x, ids, w, out, d, g))
    streams = [torch.cuda.Stream() for _ in sets]
    for turn in range(4):
        for i, (x, ids, w, out, d, g) in enumerate(sets):
            x.copy_(torch.randn(S, 2, V, device=DEV) * (turn + 1))
            out.entropy.fill_(-1)
            d.fill_(-1)
        torch.cuda.synchronize()
        for st, (x, ids, w, out, d, g) in zip(streams, sets):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for ctx, (x, ids, w, out, d, g) in zip(ctxs, sets):
            want = scores.token_scores(x, ids, k=6)
            for n in ("logp", "entropy", "row_max", "log_sum", "top_logp", "top_ids"):
                assert torch.equal(getattr(out, n), getattr(want, n)), (turn, n)
            assert torch.equal(d, scores.token_scores_bwd(x, ids, want.row_max, want.log_sum, want.entropy, dlogp=w, dentropy=w))
            scores.token_scores(x[:, :1], ids[:, :1].contiguous(), k=200, ctx=ctx)     # a larger work buffer
    st = torch.cuda.Stream()
    x, ids = sets[0][:2]
    st.wait_stream(torch.cuda.current_stream())
    out = scores.token_scores(x, ids, k=6, stream=st)
    want = scores.token_scores(x, ids, k=6)
    assert torch.equal(out.top_logp, want.top_logp)


def test_refused_while_captured_if_the_buffer_would_grow():
    ctx = grpo.Context(0)
    x, ids = torch.randn(2, 1, 100000, device=DEV), torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    out = scores.token_scores(x, ids, k=200, ctx=grpo.Context(0))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = x * 2
        with pytest.raises(PcpError, match="work buffer"):
            scores.token_scores(x, ids, k=200, outputs=out, sync=False, ctx=ctx)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x * 2)


def test_given_buffers_that_do_not_fit():
    x, ids = torch.randn(2, 3, 50, device=DEV), torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    out = scores.token_scores(x, ids, k=2)
    for kw in (dict(k=3), dict(k=2, top_ids_dtype=torch.int64)):
        with pytest.raises(PcpError):
            scores.token_scores(x, ids, outputs=out, **kw)
    with pytest.raises(PcpError):
        scores.token_scores(x[:1], ids[:1], outputs=out)
    with pytest.raises(PcpError):
        scores.token_scores(x, ids.cpu())
