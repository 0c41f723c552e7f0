"""Finite masks of any size (-1e9 .. a type's lowest value) at several temperatures: top logits,
distillation and draft verification against their definitions in 64 bits (tests/distill_ref.py,
which also derives the distillation's bars).

A finite mask differs from -inf in that a lane, a part or a row may hold nothing else: sums are
then against the mask itself, whose product with log2(e) / temperature is rounded by far more
than the whole range of an exponential.
"""
import numpy as np
import pytest
import torch

from distill_ref import IGNORE, REL, half_step, lse_ref, row_ref, top_ref, verify_ref
from pcp_amd import distill, grpo, step
from pcp_amd._lib import PcpError

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MASKS = {"f32": [-1e9, -1e10, -1e20, -1e30, "lowest"], "bf16": [-1e9, -1e10, -1e20, -1e30, "lowest"],
         "f16": [-3e4, "lowest"]}
CASES = [(d, m) for d in MASKS for m in MASKS[d]]
TEMPERATURES = [0.7, 1.0, 1.5, 2.0, 3.0, 4.0]
PATTERNS = ["run", "scattered", "tail", "alone"]


def mask_value(dtype, mask):
    return float(torch.finfo(DT[dtype]).min) if mask == "lowest" else float(torch.tensor(mask).to(DT[dtype]))


def to_dev(x, dtype, offset=0):
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(DT[dtype])
    buf = torch.empty(t.numel() + offset, dtype=t.dtype, device=DEV)
    v = buf[offset:].view(t.shape)
    v.copy_(t)
    return v


def host64(t):
    return t.detach().double().cpu().numpy()


def where_masked(rng, pattern, R, V):
    """[R, V] of booleans: a run through the middle, most of the row, the row's end, all but one token."""
    m = np.zeros((R, V), bool)
    if pattern == "run":
        m[:, V // 5:4 * V // 5] = True
    elif pattern == "scattered":
        m[:] = rng.random((R, V)) < 0.97
        m[:, rng.integers(0, V, 3)] = False
    elif pattern == "tail":
        m[:, V - V // 3:] = True
    else:
        m[:] = True
        m[np.arange(R), rng.integers(0, V, R)] = False
    return m


# ---- top logits ------------------------------------------------------------------------


def lse_bar(z):
    """Bar of an f32 log-sum-exp of z = x / temperature [R, V]. A lane adds up to 64 terms in f32
    (63 roundings of 2^-24), its batches in f64, rounded once; the trees over lanes, waves and
    parts add 6 + 2 + 6. A term 2^y, y below the largest by |y|, has the roundings of
    the exponent, of k and of the two of each rescaling: 5 * 2^-24 |y| ln 2; v_exp_f32 once for the
    term and once for each rescaling (lane, wave, part, the reference's residue), 5 * 2^-23; the
    batch's product 2^-24, log2f 2^-23. Then half a step of the result."""
    z = z.astype(np.float64)
    lse = lse_ref(z)
    q = np.exp(z - lse[:, None])
    far = (q * np.minimum(z.max(1)[:, None] - z, 1e4)).sum(1)     # |y| ln 2; q is 0 beyond
    return 2.0 ** -24 * (63 + 1 + 14 + 10 + 1 + 2 + 5 * far) * 1.01 + 2.0 ** -24 * np.abs(lse)


def check_top(x, k, temperature, out):
    v, i, lse = top_ref(host64(x), k, float(np.float32(temperature)))
    assert np.array_equal(out.ids.cpu().numpy(), i)
    assert np.array_equal(host64(out.values), v)
    off = np.abs(host64(out.lse) - lse)
    assert (off <= lse_bar(host64(x) / float(np.float32(temperature)))).all(), off.max()


@pytest.mark.parametrize("dtype,mask", CASES)
@pytest.mark.parametrize("pattern", PATTERNS)
@pytest.mark.parametrize("R,V,k", [(3, 40000, 30), (700, 21000, 5), (2, 300, 7)])
def test_top_logits(dtype, mask, pattern, R, V, k):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((R, V)).astype(np.float32) * 3
    x[where_masked(rng, pattern, R, V)] = mask_value(dtype, mask)
    for offset in (0, 3):
        xd = to_dev(x, dtype, offset)
        for t in TEMPERATURES:
            check_top(xd if R < 100 else xd[:4], k, t, distill.top_logits(xd, k, temperature=t) if R < 100 else
                      first_rows(distill.top_logits(xd, k, temperature=t), 4))


def first_rows(out, n):
    return distill.TopLogits(out.values[:n], out.ids[:n], out.lse[:n])


@pytest.mark.parametrize("dtype,mask", CASES)
@pytest.mark.parametrize("R,V", [(2, 40000), (600, 20000)])
def test_top_logits_of_rows_with_nothing_else(dtype, mask, R, V):
    """Every logit the mask: a uniform distribution, whose log-sum-exp is reported only where it
    leaves f32's range."""
    low = mask_value(dtype, mask)
    x = torch.full((R, V), low, dtype=DT[dtype], device=DEV)
    for t in TEMPERATURES:
        if low / t < -float(torch.finfo(torch.float32).max):
            with pytest.raises(PcpError):
                distill.top_logits(x, 9, temperature=t)
            continue
        out = distill.top_logits(x, 9, temperature=t)
        assert torch.equal(out.ids.cpu(), torch.arange(9, dtype=torch.int32).expand(R, 9))
        assert bool((out.values == low).all())
        want = low / float(np.float32(t)) + np.log(V)
        assert (np.abs(host64(out.lse) - want) <= 2.0 ** -23 * abs(want)).all()


@pytest.mark.parametrize("dtype,R,V", [("bf16", 2, 151936), ("f32", 5, 50257), ("f16", 600, 32000), ("bf16", 520, 1 << 24)])
def test_log_sum_exp_to_its_rounding(dtype, R, V):
    """Ordinary rows, up to the largest vocabulary in one workgroup, to the bar that the sums
    leave (the rest of the probability, 1 - sum p, is taken from this number)."""
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.empty((R, V), dtype=DT[dtype], device=DEV).normal_(0, 3, generator=g)
    for t in (1.0, 0.6):
        out = distill.top_logits(x, 4, temperature=t)
        for r in (0, R // 2, R - 1):
            z = (x[r].double() / float(np.float32(t)))[None].cpu().numpy()
            assert abs(float(out.lse[r]) - lse_ref(z)[0]) <= lse_bar(z)[0]


# ---- distillation ----------------------------------------------------------------------


def masked_rows(rng, V, k, low, huge_teacher):
    """Student rows [8, V] with teacher ids and logits [8, k]: a masked run outside the entries; nothing
    else outside them; all entries masked; all but one; the whole row; the entries and most of the
    rest; all but one entry; an ordinary row (or one whose teacher has the mask at every entry)."""
    R = 8
    x = rng.standard_normal((R, V)).astype(np.float32) * 3
    ids = np.stack([rng.choice(V, k, replace=False) for _ in range(R)]).astype(np.int32)
    t = (np.take_along_axis(x, ids, 1) + rng.standard_normal((R, k))).astype(np.float32)
    lse = np.zeros(R, np.float32)
    for r in range(R):
        lse[r] = lse_ref(t[r].astype(np.float64)[None])[0] + rng.random() * 0.2
    outside = np.ones((R, V), bool)
    np.put_along_axis(outside, ids, False, 1)
    run = np.zeros(V, bool)
    run[V // 5:4 * V // 5] = True
    x[0, outside[0] & run] = low
    x[1, outside[1]] = low
    x[2, ids[2]] = low
    x[3, ids[3, 1:]] = low
    x[3, outside[3] & run] = low
    x[4] = low
    x[5, ids[5]] = low
    x[5, outside[5] & (rng.random(V) < 0.99)] = low
    x[5, np.flatnonzero(outside[5])[:2]] = 1.0
    x[6] = low
    x[6, ids[6, 0]] = 0.5
    if huge_teacher:
        t[7] = low
    return x, ids, t, lse


@pytest.mark.parametrize("dtype,mask", CASES)
@pytest.mark.parametrize("mode", ["forward", "renormalised", "reverse"])
@pytest.mark.parametrize("N,V", [(8, 701), (8, 40000), (900, 40000)])
def test_distill(dtype, mask, mode, N, V):
    """Rows in parts and rows kept by a workgroup, against the definition of each row shifted by
    its largest logit (in 64 bits -1e30 + log q would lose the second)."""
    rng = np.random.default_rng(V + N)
    k = 20
    x, ids, t, lse = masked_rows(rng, V, k, mask_value(dtype, mask), mode == "renormalised")
    xs = torch.zeros((1, N, V), dtype=DT[dtype], device=DEV)
    xs[0, -8:] = to_dev(x, dtype)

    def all_rows(a, fill):
        out = torch.full((1, N) + a.shape[1:], fill, dtype=torch.from_numpy(a).dtype)
        out[0, -8:] = torch.from_numpy(a)
        return out.to(DEV)

    weight = torch.zeros((1, N), device=DEV)
    weight[0, -8:] = 1.0
    args = (all_rows(ids, IGNORE), all_rows(t, 0.0), None if mode == "renormalised" else all_rows(lse, 0.0), weight)
    kw = dict(divergence="reverse" if mode == "reverse" else "forward", sync=False)
    x64 = host64(xs[0, -8:])
    ctx = grpo.Context(0)
    for tau in (0.7, 1.0, 1.5, 2.0, 4.0):
        out = distill.distill_fwd_bwd(xs, *args, temperature=tau, ctx=ctx, **kw)
        alone = distill.distill_fwd_bwd(xs, *args, temperature=tau, ctx=ctx, want_dlogits=False, **kw)
        wide = None
        if dtype != "f32":
            wide = distill.distill_fwd_bwd(xs, *args, temperature=tau, ctx=ctx, dlogits_dtype=torch.float32, **kw)
        ctx.sync()
        tau64 = float(np.float32(tau))
        for r in range(8):
            t64 = t[r].astype(np.float64)
            l, grad, mag, lb = row_ref(x64[r] - x64[r].max(), ids[r], t64 - t64.max() if mode == "renormalised" else t64,
                                       None if mode == "renormalised" else float(lse[r]), tau64, mode != "reverse")
            for o in (out, alone):
                got = float(o.token_loss[0, N - 8 + r])
                if abs(l) < 3.3e38:
                    assert abs(got - l) <= lb + 2.0 ** -24 * abs(l), (tau, r, got, l)
                else:
                    assert not np.isnan(got) and got > 3e38
            c = 1.0 / (8 * tau64)
            bar = c * REL * mag
            flushed = 2.0 ** -42 * np.abs(c * grad).max() + 2.0 ** -126
            for o, kind in ((out, dtype), (wide, "f32")):
                if o is None:
                    continue
                off = np.abs(host64(o.dlogits[0, N - 8 + r]) - c * grad)
                worst = off - bar - half_step(kind, c * grad) - 2.0 ** -8 * bar - flushed
                assert worst.max() <= 0, (tau, r, kind, worst.argmax(), off[worst.argmax()])
        assert not out.dlogits[0, :-8].any()


# ---- draft verification ----------------------------------------------------------------


@pytest.mark.parametrize("dtype,mask", CASES)
@pytest.mark.parametrize("pattern", PATTERNS + ["everything"])
@pytest.mark.parametrize("S", [2, 6])
@pytest.mark.parametrize("lookup", [False, True])
def test_verify(dtype, mask, pattern, S, lookup):
    """Tokens and counts equal to the definition's, log-probs to f32 rounding. The second sequence's
    target is masked throughout, so that every token is as probable as any other."""
    rng = np.random.default_rng(S)
    n, V = 2, 40000
    low = mask_value(dtype, mask)
    x = rng.standard_normal((S, n + 1, V)).astype(np.float32) * 3
    y = x[:, :n] + 0.5 * rng.standard_normal((S, n, V)).astype(np.float32)
    out_of = np.ones((S, V), bool) if pattern == "everything" else where_masked(rng, pattern, S, V)
    for s in range(S):
        x[s, :, out_of[s]] = low
        y[s, :, out_of[s]] = low
    x[1] = low
    d = np.zeros((S, n), np.int64)
    for s in range(S):
        for i in range(n):
            z = y[s, i].astype(np.float64)
            d[s, i] = np.argmax(np.where(out_of[s] & ~out_of[s].all(), -np.inf, z - z.max()) + rng.gumbel(size=V))
    xd, yd = to_dev(x, dtype, 1), None if lookup else to_dev(y, dtype)
    for t in (0.7, 1.0, 1.5, 2.0, 4.0):
        u = rng.random((S, n + 1)).astype(np.float32)
        u[0, 0] = 0.0                         # accepted if the token has any probability
        out = step.verify_drafts(xd, torch.from_numpy(d).to(DEV), yd, temperature=t, uniforms=torch.from_numpy(u).to(DEV))
        want = verify_ref(host64(xd), None if lookup else host64(yd), d, np.full(S, n), u, float(np.float32(t)), V)
        assert np.array_equal(out.accepted.cpu().numpy(), want[1]), t
        assert np.array_equal(out.tokens.cpu().numpy(), want[0]), t
        assert (np.abs(host64(out.logp) - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 1e-12).all(), t


# ---- rows with one large offset ---------------------------------------------------------

OFFSETS = [1e3, -1e4, 1e5, -1e6, 1e7, -3e7, 2e8, -1e9, 1.4e9, -1.6e9, 3e9, -1e10]


def with_offset(rng, shape, offset):
    """f32 logits a few f32 steps (at least a few units) around `offset`: a softmax like any other, whose
    reference point's product with the scale is rounded by up to 2^6."""
    step = max(1.0, float(np.spacing(np.float32(abs(offset)))))
    return (offset + np.round(rng.standard_normal(shape) * 3) * step).astype(np.float32)


@pytest.mark.parametrize("offset", OFFSETS)
def test_rows_far_from_zero(offset):
    rng = np.random.default_rng(3)
    for R, V, k in ((3, 40000, 30), (600, 20000, 8)):
        x = to_dev(with_offset(rng, (R, V), offset), "f32", 1)
        for t in (0.7, 1.0, 2.0):
            out = distill.top_logits(x, k, temperature=t)
            check_top(x[:4], k, t, first_rows(out, 4))
    for N, V in ((4, 701), (4, 40000), (900, 40000)):
        x = with_offset(rng, (4, V), offset)
        ids = np.stack([rng.choice(V, 12, replace=False) for _ in range(4)]).astype(np.int32)
        t = rng.standard_normal((4, 12)).astype(np.float32) * 2
        lse = (lse_ref(t.astype(np.float64)) + 0.3).astype(np.float32)
        xs = torch.zeros((1, N, V), device=DEV)
        xs[0, -4:] = to_dev(x, "f32")
        full = lambda a, fill: torch.cat([torch.full((N - 4,) + a.shape[1:], fill, dtype=torch.from_numpy(a).dtype),
                                          torch.from_numpy(a)])[None].to(DEV)
        weight = torch.zeros((1, N), device=DEV)
        weight[0, -4:] = 1.0
        for forward in (True, False):
            out = distill.distill_fwd_bwd(xs, full(ids, IGNORE), full(t, 0.0), full(lse, 0.0), weight,
                                          divergence="forward" if forward else "reverse")
            x64 = x.astype(np.float64)
            for r in range(4):
                l, grad, mag, lb = row_ref(x64[r] - x64[r].max(), ids[r], t[r].astype(np.float64), float(lse[r]), 1.0, forward)
                assert abs(float(out.token_loss[0, N - 4 + r]) - l) <= lb + 2.0 ** -24 * abs(l)
                bar = REL * mag / 4
                off = np.abs(host64(out.dlogits[0, N - 4 + r]) - grad / 4)
                assert (off <= bar + half_step("f32", grad / 4) + 2.0 ** -42 * np.abs(grad).max() + 2.0 ** -126).all()
    for S in (2, 30):
        n, V = 2, 9001
        x = with_offset(rng, (S, n + 1, V), offset)
        y = with_offset(rng, (S, n, V), -offset)
        d = np.argmax(y + rng.gumbel(size=y.shape), -1).astype(np.int64)
        u = rng.random((S, n + 1)).astype(np.float32)
        for draft in (None, to_dev(y, "f32")):
            out = step.verify_drafts(to_dev(x, "f32"), torch.from_numpy(d).to(DEV), draft, uniforms=torch.from_numpy(u).to(DEV))
            want = verify_ref(x.astype(np.float64), None if draft is None else y.astype(np.float64), d, np.full(S, n), u, 1.0, V)
            assert np.array_equal(out.accepted.cpu().numpy(), want[1]) and np.array_equal(out.tokens.cpu().numpy(), want[0])
            assert (np.abs(host64(out.logp) - want[2]) <= 2.0 ** -24 * np.abs(want[2]) + 1e-12).all()
