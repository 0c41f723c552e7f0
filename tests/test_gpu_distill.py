"""Top logits and the distillation loss on the GPU against their definitions in 64 bits
(tests/distill_ref.py, which also derives the bars)."""
import numpy as np
import pytest
import torch

from distill_ref import IGNORE, REL, distill_ref, half_step, lse_ref, row_ref, top_ref
from pcp_amd import distill, grpo
from pcp_amd._lib import PcpError

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


def host64(t):
    return t.detach().double().cpu().numpy()


def rows_like_a_model(rng, shape, scale=3.0):
    x = rng.standard_normal(shape).astype(np.float32) * scale
    flat = x.reshape(-1, shape[-1])
    for r in flat:
        n = min(6, shape[-1])
        r[rng.choice(shape[-1], n, replace=False)] += rng.random(n).astype(np.float32) * 12
    return x


# ---- top logits ------------------------------------------------------------------------

TOP = [("f32", 1, 1, 1), ("bf16", 3, 7, 7), ("f16", 5, 64, 64), ("f32", 4, 255, 20), ("bf16", 6, 1000, 256),
       ("bf16", 2, 1003, 65), ("f32", 3, 8191, 128), ("bf16", 5, 16385, 256), ("f16", 2, 50257, 33),
       ("f32", 2, 50257, 256), ("bf16", 1, 151936, 64), ("bf16", 300, 16000, 8), ("f32", 2100, 513, 5),
       ("bf16", 2, 262144, 256), ("f16", 2049, 4096, 64)]


def check_top(x, k, temperature, out):
    v, i, lse = top_ref(host64(x), k, temperature)
    assert np.array_equal(out.ids.cpu().numpy(), i)
    assert np.array_equal(host64(out.values), v)
    bar = 1e-5 * np.maximum(1.0, np.abs(lse)) * max(1.0, 1.0 / temperature)
    assert (np.abs(host64(out.lse) - lse) <= bar).all()


@pytest.mark.parametrize("dtype,R,V,k", TOP)
@pytest.mark.parametrize("offset", [0, 1])
def test_top_logits(dtype, R, V, k, offset):
    rng = np.random.default_rng(R * V + k)
    x = to_dev(rows_like_a_model(rng, (R, V)), dtype, offset)
    check_top(x, k, 1.0, distill.top_logits(x, k))
    check_top(x, k, 2.0, distill.top_logits(x, k, temperature=2.0, ids_dtype=torch.int64))


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two_values", "masked", "all_but_one_masked", "zeros"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("R,V,k", [(2, 40000, 256), (2, 40000, 1), (2200, 5000, 40)])
def test_top_logits_orders(kind, dtype, R, V, k):
    """Rows that defeat a threshold: many equal values, every later value larger, masks."""
    rng = np.random.default_rng(5)
    x = np.zeros((R, V), np.float32)
    if kind == "equal":
        x[:] = -1.5
    elif kind == "rising":
        x[:] = np.linspace(-20, 20, V)
    elif kind == "falling":
        x[:] = np.linspace(20, -20, V)
    elif kind == "two_values":
        x[:] = rng.integers(0, 2, (R, V))
    elif kind in ("masked", "all_but_one_masked"):
        x[:] = -np.inf
        n = 1 if kind == "all_but_one_masked" else 17
        for r in range(R):
            x[r, rng.choice(V, n, replace=False)] = rng.standard_normal(n)
    else:
        x[:] = np.where(rng.random((R, V)) < 0.5, 0.0, -0.0)   # both zeros are one value
    x = to_dev(x, dtype)
    check_top(x, k, 1.0, distill.top_logits(x, k))


@pytest.mark.parametrize("dtype", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("R,V,k", [(3, 40000, 200), (2100, 5000, 30), (2, 600, 256)])
def test_top_logits_masks_of_the_lowest_value(dtype, R, V, k):
    """Two thirds of the vocabulary at the type's lowest value or -inf, in runs and scattered,
    with one row of NaN between (which outranks nothing)."""
    rng = np.random.default_rng(R + k)
    x = rows_like_a_model(rng, (R, V))
    low = float(torch.finfo(DT[dtype]).min)
    x[:, V // 3:2 * V // 3] = low
    x[rng.random((R, V)) < 0.4] = low
    x[1::2][x[1::2] == low] = -np.inf
    check_top(to_dev(x, dtype), k, 1.0, distill.top_logits(to_dev(x, dtype), k))
    x[1] = np.nan
    x[1, 5:5 + k - 1] = 1.0
    t = to_dev(x, dtype)
    ctx = grpo.Context(0)
    out = distill.top_logits(t, k, sync=False, ctx=ctx)
    with pytest.raises(PcpError):
        ctx.sync()
    assert torch.equal(out.ids[1, :k - 1].cpu(), torch.arange(5, 5 + k - 1, dtype=torch.int32))
    assert torch.isnan(out.values[1, k - 1]) and int(out.ids[1, k - 1]) == 0
    check_top(t[2:], k, 1.0, distill.TopLogits(out.values[2:], out.ids[2:], out.lse[2:]))


def test_top_logits_rows_apart_and_long():
    """Rows further apart than the vocabulary, and offsets past 2^31 elements."""
    rng = np.random.default_rng(1)
    wide = to_dev(rows_like_a_model(rng, (9, 1203)), "f16")
    check_top(wide[:, 1:1002], 50, 1.0, distill.top_logits(wide[:, 1:1002], 50))
    R, V = 14500, 151936                      # 2.2e9 elements
    x = torch.empty((R, V), dtype=torch.bfloat16, device=DEV)
    x.fill_(-3.0)
    last = to_dev(rows_like_a_model(rng, (2, V)), "bf16")
    x[-2:] = last
    out = distill.top_logits(x, 16)
    check_top(last, 16, 1.0, distill.TopLogits(out.values[-2:], out.ids[-2:], out.lse[-2:]))
    assert torch.equal(out.ids[0].cpu(), torch.arange(16, dtype=torch.int32))
    assert not torch.any(out.values[:-2] != -3.0)


def test_top_logits_more_rows_than_a_grid_holds():
    x = torch.arange(70000, device=DEV, dtype=torch.float32)[:, None] * torch.tensor([1.0, -1.0, 0.5], device=DEV)
    out = distill.top_logits(x, 2)
    assert torch.equal(out.ids[1:].cpu(), torch.tensor([[0, 2]] * 69999, dtype=torch.int32))
    assert torch.equal(out.values[:, 1].cpu(), x[:, 2].cpu())


def test_top_logits_nonfinite_rows_are_reported():
    x = to_dev(rows_like_a_model(np.random.default_rng(2), (4, 3000)), "f32")
    clean = distill.top_logits(x, 10)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[2, 1234] = bad
        with pytest.raises(PcpError) as e:
            distill.top_logits(y, 10)
        assert e.value.code == -4
        ctx = grpo.Context(0)
        out = distill.top_logits(y, 10, sync=False, ctx=ctx)
        with pytest.raises(PcpError) as e:
            ctx.sync()
        assert e.value.code == -4
        for r in (0, 1, 3):
            assert torch.equal(out.ids[r], clean.ids[r]) and torch.equal(out.lse[r], clean.lse[r])
        if np.isnan(bad):
            assert torch.equal(out.ids[2, :9].cpu()[out.ids[2, :9].cpu() != 1234], out.ids[2, :9].cpu())
    y = x.clone()
    y[1] = -float("inf")
    with pytest.raises(PcpError):
        distill.top_logits(y, 10)


# ---- distillation ----------------------------------------------------------------------


def make_case(rng, S, LS, V, k, TS=None, cut=True, mask="lengths"):
    TS = TS or LS
    x = rows_like_a_model(rng, (S, LS, V))
    t = x + rng.standard_normal(x.shape).astype(np.float32)
    ids = np.full((S, LS, k), IGNORE, np.int64)
    val = np.zeros((S, LS, k), np.float32)
    lse = lse_ref(t.astype(np.float64)).astype(np.float32)
    for s in range(S):
        for r in range(LS):
            n = min(k, V)
            if cut:
                n = int(rng.integers(0, n + 1)) if rng.random() < 0.5 else n
            at = np.argsort(-t[s, r], kind="stable")[:n]
            where = rng.permutation(k)[:n]            # entries in any order, unused ones between
            ids[s, r, where], val[s, r, where] = at, t[s, r, at]
    if mask == "lengths":
        m = (np.arange(TS)[None] < rng.integers(0, TS + 1, (S, 1))).astype(np.float32)
    elif mask == "weights":
        m = rng.random((S, TS)).astype(np.float32) * (rng.random((S, TS)) < 0.7)
    else:
        m = np.ones((S, TS), np.float32)
    return x, ids, val, lse, m.astype(np.float32)


def check_distill(x_dev, out, case, out_dtype, *, tail, **kw):
    _, ids, val, lse, mask = case
    want, bars = distill_ref(host64(x_dev), ids, val, lse if tail else None, mask, **kw)
    tok = host64(out.token_loss)
    assert (np.abs(tok - want[1]) <= bars[1] + 2.0 ** -24 * np.abs(want[1])).all(), np.abs(tok - want[1]).max()
    assert abs(float(out.loss) - want[0]) <= bars[0] + 1e-6 * abs(want[0])
    if out.dlogits is not None:
        d = host64(out.dlogits)
        bar = bars[2] + half_step(out_dtype, want[2]) + (2.0 ** -8) * bars[2]
        worst = np.abs(d - want[2]) - bar
        assert (worst <= 0).all(), (np.unravel_index(worst.argmax(), worst.shape), worst.max())
        assert (d[bars[2].max(-1) == 0] == 0).all()     # rows without weight or entries


def run_distill(case, dtype, out_dtype, *, tail=True, ids_dtype=torch.int32, x_off=0, d_off=0, in_place=False,
                mask_dtype=torch.float32, forward=True, tau=1.0, rows=None, off=0, **kw):
    x, ids, val, lse, mask = case
    xd = to_dev(x, dtype, x_off)
    kept = xd.clone()
    dl = None
    if in_place:
        dl = xd
    elif d_off:
        dl = to_dev(np.full(x.shape, 7.0), out_dtype, d_off)
    out = distill.distill_fwd_bwd(
        xd, torch.from_numpy(ids).to(DEV, ids_dtype), torch.from_numpy(val).to(DEV),
        torch.from_numpy(lse).to(DEV) if tail else None, torch.from_numpy(mask).to(DEV, mask_dtype), rows=rows,
        tok_offset=off, divergence="forward" if forward else "reverse", temperature=tau, dlogits=dl,
        dlogits_dtype=DT[out_dtype], **kw)
    return kept, out


SHAPES = [(1, 1, 1, 1), (2, 3, 2, 4), (2, 4, 7, 3), (3, 5, 50, 64), (2, 6, 255, 65), (4, 9, 1000, 8), (2, 4, 1003, 256),
          (2, 3, 4099, 20), (1, 5, 16385, 64), (2, 3, 33000, 130), (1, 3, 50257, 32), (1, 4, 151936, 64),
          (1, 2, 170001, 256)]


@pytest.mark.parametrize("S,T,V,k", SHAPES)
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("mode", ["forward", "renormalised", "reverse"])
def test_distill(S, T, V, k, dtype, out, mode):
    case = make_case(np.random.default_rng(V + k), S, T, V, k)
    tail = mode != "renormalised"
    xd, o = run_distill(case, dtype, out, tail=tail, forward=mode != "reverse")
    check_distill(xd, o, case, out, tail=tail, rows=T, off=0, forward=mode != "reverse")


@pytest.mark.parametrize("x_off,d_off", [(1, 0), (0, 1), (3, 3), (2, 5)])
@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("V", [13, 1000, 20011])
def test_distill_rows_off_16_bytes(x_off, d_off, dtype, out, V):
    case = make_case(np.random.default_rng(V), 2, 5, V, 24)
    xd, o = run_distill(case, dtype, out, x_off=x_off, d_off=d_off)
    check_distill(xd, o, case, out, tail=True, rows=5, off=0)


@pytest.mark.parametrize("mode", ["forward", "reverse"])
@pytest.mark.parametrize("dtype,V", [("bf16", 3001), ("f32", 30000), ("bf16", 151936)])
def test_distill_in_place(mode, dtype, V):
    case = make_case(np.random.default_rng(3), 2, 4, V, 40)
    xd, o = run_distill(case, dtype, dtype, in_place=True, forward=mode == "forward")
    check_distill(xd, o, case, dtype, tail=True, rows=4, off=0, forward=mode == "forward")


@pytest.mark.parametrize("tau,weight,norm", [(2.0, 1.0, 0.0), (0.7, 3.5, 0.0), (1.0, 0.25, 11.0)])
@pytest.mark.parametrize("mode", ["forward", "renormalised", "reverse"])
def test_distill_scales_and_layout(tau, weight, norm, mode):
    """Temperature, weight and loss norm; logits[:, :-1] against the next tokens' weights."""
    rng = np.random.default_rng(9)
    S, T, V, k = 3, 7, 700, 33
    x, ids, val, _, m = make_case(rng, S, T, V, k, mask="weights")
    full = rows_like_a_model(rng, (S, T, V)) + x
    lse = lse_ref(full.astype(np.float64) / tau).astype(np.float32)
    for s in range(S):
        for r in range(T):
            used = ids[s, r] != IGNORE
            val[s, r, used] = full[s, r, ids[s, r, used]]
    case = (x, ids, val, lse, m)
    tail = mode != "renormalised"
    xd, o = run_distill(case, "f32", "f32", tail=tail, forward=mode != "reverse", tau=tau, weight=weight,
                        loss_norm=norm, rows=T - 1, off=1, ids_dtype=torch.int64)
    check_distill(xd, o, case, "f32", tail=tail, rows=T - 1, off=1, tau=tau, weight=weight, loss_norm=norm,
                  forward=mode != "reverse")


def test_distill_bool_mask_no_mask_and_loss_alone():
    rng = np.random.default_rng(4)
    case = make_case(rng, 3, 6, 900, 12)
    a = run_distill(case, "f32", "f32")[1]
    b = run_distill(case, "f32", "f32", mask_dtype=torch.bool)[1]
    assert torch.equal(a.dlogits, b.dlogits) and torch.equal(a.loss, b.loss)
    c = run_distill(case, "f32", "f32", want_dlogits=False)[1]
    assert c.dlogits is None
    want, bars = distill_ref(case[0].astype(np.float64), *case[1:], rows=6, off=0)
    assert (np.abs(host64(c.token_loss) - want[1]) <= bars[1] + 2.0 ** -24 * np.abs(want[1])).all()
    x, ids, val, lse, _ = case
    d = distill.distill_fwd_bwd(to_dev(x, "f32"), torch.from_numpy(ids).to(DEV, torch.int32),
                                torch.from_numpy(val).to(DEV), torch.from_numpy(lse).to(DEV))
    check_distill(to_dev(x, "f32"), d, (x, ids, val, lse, np.ones((3, 6), np.float32)), "f32", tail=True, rows=6, off=0)


@pytest.mark.parametrize("mode", ["forward", "reverse"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distill_masked_vocabulary(mode, dtype):
    """Logits of -inf (or the type's lowest) outside and inside the entries, teacher entries of
    -inf, a tail of nothing, entries that cover the vocabulary."""
    rng = np.random.default_rng(6)
    S, T, V, k = 1, 6, 600, 16
    x, ids, val, lse, m = make_case(rng, S, T, V, k, cut=False, mask="ones")
    low = float(torch.finfo(DT[dtype]).min)
    x[0, 0, 100:] = np.minimum(x[0, 0, 100:], -np.inf)
    x[0, 1, 100:] = low
    x[0, 2] = -np.inf
    for r in (0, 1, 2):
        keep = np.arange(k) if r != 2 else np.arange(50, 50 + k)
        ids[0, r], val[0, r] = keep, rng.standard_normal(k)
        x[0, r, keep] = rng.standard_normal(k)
        lse[0, r] = lse_ref(val[0, r].astype(np.float64)[None])[0] + 0.1
    val[0, 3, 4:] = -np.inf                    # unused entries by their logit
    case = (x, ids, val, lse, m)
    xd, o = run_distill(case, dtype, dtype, forward=mode == "forward")
    check_distill(xd, o, case, dtype, tail=True, rows=T, off=0, forward=mode == "forward")
    if mode == "forward":                      # a student that rules out what the teacher says: infinite, no NaN
        x2 = x.copy()
        x2[0, 4, ids[0, 4, 0]] = -np.inf
        _, o = run_distill((x2, ids, val, lse, m), dtype, dtype)
        assert float(o.token_loss[0, 4]) == float("inf") and bool(torch.isfinite(o.dlogits).all())
    small = make_case(rng, 2, 3, 9, 12, cut=False, mask="ones")
    xd, o = run_distill(small, dtype, dtype, forward=mode == "forward")
    check_distill(xd, o, small, dtype, tail=True, rows=3, off=0, forward=mode == "forward")


@pytest.mark.parametrize("mode", ["forward", "reverse"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,V", [(3, 700), (3, 40000), (900, 40000)])
def test_distill_entries_that_the_student_masks(mode, dtype, N, V):
    """Every entry's logit -inf, or the type's lowest value, with the rest ordinary: the student
    gives the entries nothing. (Forward, the loss is infinite or next to it; its gradient is not.)"""
    rng = np.random.default_rng(V + N)
    case = make_case(rng, 1, 3, V, 20, cut=False, mask="ones")
    x, ids, val, lse, m = case
    for r in range(3):
        x[0, r, ids[0, r]] = (-np.inf, float(torch.finfo(DT[dtype]).min), -np.inf)[r]
    x[0, 2] += 200 if dtype == "f32" else 0
    xs = torch.zeros((1, N, V), dtype=DT[dtype], device=DEV)
    xs[0, -3:] = to_dev(x[0], dtype)

    def all_rows(t, fill):
        out = torch.full((1, N) + t.shape[2:], fill, dtype=torch.from_numpy(t).dtype)
        out[0, -3:] = torch.from_numpy(t[0])
        return out.to(DEV)

    out = distill.distill_fwd_bwd(xs, all_rows(ids, IGNORE), all_rows(val, 0.0), all_rows(lse, 0.0), all_rows(m, 0.0),
                                  divergence=mode, sync=False, ctx=grpo.Context(0))
    want, bars = distill_ref(host64(xs[:, -3:]), ids, val, lse, m, rows=3, off=0, forward=mode == "forward")
    d = host64(out.dlogits[:, -3:])
    assert (np.abs(d - want[2]) <= bars[2] + half_step(dtype, want[2]) + 2.0 ** -8 * bars[2] + 2.0 ** -126).all()
    if mode == "reverse":
        tok = host64(out.token_loss)[:, -3:]
        assert (np.abs(tok - want[1]) <= bars[1] + 2.0 ** -24 * np.abs(want[1])).all()


@pytest.mark.parametrize("mode", ["forward", "renormalised", "reverse"])
def test_distill_gradient_against_differences(mode):
    """Central differences of the kernel's own token losses, one logit of one row each:
    h = 0.05 leaves h^2 / 6 of the third derivative (below 1) and 2 REL / h of the losses."""
    rng = np.random.default_rng(8)
    V, k, h = 40, 9, 0.05
    x, ids, val, lse, _ = make_case(rng, 1, 1, V, k, cut=False)
    many = np.repeat(x.reshape(1, 1, V), 2 * V + 1, axis=1).astype(np.float32)
    for v in range(V):
        many[0, 1 + v, v] += h
        many[0, 1 + V + v, v] -= h
    N = 2 * V + 1
    case = (many, np.repeat(ids, N, 1), np.repeat(val, N, 1), np.repeat(lse, N, 1), np.ones((1, N), np.float32))
    tail = mode != "renormalised"
    _, o = run_distill(case, "f32", "f32", tail=tail, forward=mode != "reverse", loss_norm=1.0 / N)
    tok = host64(o.token_loss)[0]
    diff = (tok[1:1 + V] - tok[1 + V:]) / (many[0, 1:1 + V, :].diagonal() - many[0, 1 + V:, :].diagonal())
    assert np.abs(diff - host64(o.dlogits)[0, 0]).max() <= h * h / 6 * 4 + 4e-5 * 3 / h


def test_distill_reports_bad_rows_and_leaves_the_others():
    rng = np.random.default_rng(11)
    x, ids, val, lse, m = make_case(rng, 2, 4, 2000, 8, cut=False, mask="ones")
    clean = run_distill((x, ids, val, lse, m), "bf16", "bf16")[1]

    def bad(change, code, row_zero=True, weights=None):
        x2, i2, v2, l2 = x.copy(), ids.copy(), val.copy(), lse.copy()
        change(x2, i2, v2, l2)
        m2 = m if weights is None else weights
        ctx = grpo.Context(0)
        args = (to_dev(x2, "bf16"), torch.from_numpy(i2).to(DEV), torch.from_numpy(v2).to(DEV),
                torch.from_numpy(l2).to(DEV), torch.from_numpy(m2).to(DEV))
        out = distill.distill_fwd_bwd(*args, sync=False, ctx=ctx)
        if code is None:
            ctx.sync()
        else:
            with pytest.raises(PcpError) as e:
                ctx.sync()
            assert e.value.code == code
        assert torch.equal(out.dlogits[0], clean.dlogits[0])
        if row_zero:
            assert not out.dlogits[1, 2].any() and float(out.token_loss[1, 2]) == 0.0
        with pytest.raises(PcpError) if code is not None else _nothing():
            distill.distill_fwd_bwd(*args, ctx=ctx)
        return out

    def put(i, v):
        return lambda x2, i2, v2, l2: i2.__setitem__((1, 2, i), v)

    bad(put(3, 2000), -3)
    bad(put(0, -1), -3)
    bad(put(7, 1 << 40), -3)
    bad(lambda x2, i2, v2, l2: i2.__setitem__((1, 2, 5), i2[1, 2, 1]), -1)
    bad(lambda x2, i2, v2, l2: x2.__setitem__((1, 2, 77), np.nan), -4, row_zero=False)
    bad(lambda x2, i2, v2, l2: v2.__setitem__((1, 2, 3), np.nan), -4, row_zero=False)
    bad(lambda x2, i2, v2, l2: l2.__setitem__((1, 2), np.inf), -4, row_zero=False)
    # The same faults in a row without weight are not looked at.
    w = m.copy()
    w[1, 2] = 0

    def all_of_them(x2, i2, v2, l2):
        x2[1, 2], i2[1, 2, 0], v2[1, 2, 1], l2[1, 2] = np.nan, 1 << 33, np.nan, np.nan

    clean = run_distill((x, ids, val, lse, w), "bf16", "bf16")[1]
    bad(all_of_them, None, weights=w)


class _nothing:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


@pytest.mark.parametrize("V", [17, 1500, 40000])
def test_distill_twice_used_ids_wherever_they_lie(V):
    rng = np.random.default_rng(12)
    x, ids, val, lse, m = make_case(rng, 1, 1, V, 12, cut=False, mask="ones")
    for at in (0, 1, V // 2, V - 2, V - 1):
        i2 = ids.copy()
        i2[0, 0, 2] = i2[0, 0, 11] = at
        others = [j for j in range(12) if j not in (2, 11)]
        free = [v for v in range(V) if v != at][:10]
        i2[0, 0, others] = free
        for off in (0, 1):
            with pytest.raises(PcpError) as e:
                run_distill((x, i2, val, lse, m), "bf16", "bf16", x_off=off)
            assert e.value.code == -1 and "twice" in str(e.value)


def test_distill_offsets_past_32_bits():
    """2.2e9 logits in place: the last rows live, all others without weight and zeroed."""
    rng = np.random.default_rng(13)
    V, T = 151936, 14500
    x = torch.full((1, T, V), 1.0, dtype=torch.bfloat16, device=DEV)
    case = make_case(rng, 1, 3, V, 16, cut=False, mask="ones")
    x[0, -3:] = to_dev(case[0][0], "bf16")
    kept = x[:, -3:].clone()
    ids = torch.full((1, T, 16), IGNORE, dtype=torch.int32, device=DEV)
    val = torch.zeros((1, T, 16), device=DEV)
    lse = torch.zeros((1, T), device=DEV)
    ids[0, -3:] = torch.from_numpy(case[1][0]).to(DEV, torch.int32)
    val[0, -3:], lse[0, -3:] = torch.from_numpy(case[2][0]).to(DEV), torch.from_numpy(case[3][0]).to(DEV)
    mask = torch.zeros((1, T), device=DEV)
    mask[0, -3:] = 1
    out = distill.distill_fwd_bwd(x, ids, val, lse, mask, dlogits=x)
    check_distill(kept, distill.DistillOutputs(out.loss, out.token_loss[:, -3:], out.dlogits[:, -3:]), case, "bf16",
                  tail=True, rows=3, off=0)
    assert not x[0, :-3].any()


def test_distill_and_top_captured_together():
    """Both calls in one graph, replayed on new inputs with eager work between, and the call
    that would have to grow the work buffer under capture."""
    rng = np.random.default_rng(14)
    S, T, V, k = 2, 8, 3000, 20
    ctx = grpo.Context(0)
    teacher, student = to_dev(rows_like_a_model(rng, (S, T, V)), "bf16"), to_dev(rows_like_a_model(rng, (S, T, V)), "bf16")
    mask = torch.ones((S, T), device=DEV)
    s = torch.cuda.Stream()

    def step(top=None, out=None, c=ctx):
        top = distill.top_logits(teacher, k, outputs=top, sync=False, ctx=c)
        return top, distill.distill_fwd_bwd(student, top.ids, top.values, top.lse, mask, outputs=out, sync=False, ctx=c)

    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        top, out = step()
    s.synchronize()
    cold = grpo.Context(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(top, out)
        with pytest.raises(PcpError) as e:
            distill.distill_fwd_bwd(student, top.ids, top.values, top.lse, mask, outputs=out, sync=False, ctx=cold)
    assert e.value.code == -1 and "captured" in str(e.value)
    for i in range(4):
        teacher.copy_(to_dev(rows_like_a_model(rng, (S, T, V)), "bf16"))
        student.copy_(to_dev(rows_like_a_model(rng, (S, T, V)), "bf16"))
        mask[:, 3 + i:] = 0
        g.replay()
        torch.cuda.synchronize()
        wtop, wout = step(c=grpo.Context(0))
        assert torch.equal(wtop.ids, top.ids) and torch.equal(wtop.lse, top.lse)
        assert torch.equal(wout.dlogits, out.dlogits) and torch.equal(wout.loss, out.loss)
        assert torch.equal(wout.token_loss, out.token_loss)
        mask.fill_(1)
    ctx.sync()


def test_distill_on_another_stream_and_repeated():
    """The same bits each time, on a stream of the caller's, by handle, and with buffers reused."""
    case = make_case(np.random.default_rng(15), 2, 40, 5003, 24)
    _, a = run_distill(case, "bf16", "bf16")
    s = torch.cuda.Stream()
    _, b = run_distill(case, "bf16", "bf16", stream=s, sync=False)
    s.synchronize()
    _, c = run_distill(case, "bf16", "bf16", stream=s.cuda_stream)
    for o in (b, c):
        assert torch.equal(a.dlogits, o.dlogits) and torch.equal(a.loss, o.loss) and torch.equal(a.token_loss, o.token_loss)
    _, d = run_distill(case, "bf16", "bf16", outputs=c)
    assert d is c and torch.equal(a.dlogits, c.dlogits)


def test_a_student_learns_its_teachers_distribution():
    """As the calls are used together: a teacher's rows handed on, the student moved along
    -dlogits once; the first-order change of the loss is -step * |dlogits|^2."""
    rng = np.random.default_rng(16)
    S, T, V, k = 2, 6, 2048, 64
    teacher = to_dev(rows_like_a_model(rng, (S, T, V)), "bf16")
    student = to_dev(rows_like_a_model(rng, (S, T, V)), "f32")
    top = distill.top_logits(teacher, k)
    assert top.ids.shape == (S, T, k) and top.lse.shape == (S, T)
    for divergence in ("forward", "reverse"):
        a = distill.distill_fwd_bwd(student, top.ids, top.values, top.lse, divergence=divergence)
        step = 1e-2 / float(a.dlogits.abs().max())
        b = distill.distill_fwd_bwd(student - step * a.dlogits, top.ids, top.values, top.lse, divergence=divergence)
        first = step * float((a.dlogits.double() ** 2).sum())
        assert abs((float(a.loss) - float(b.loss)) - first) <= 0.05 * first + 4e-5 * (1 + abs(float(a.loss)))
    # The student's own rows as the teacher: the loss is the divergence of equal distributions.
    own = distill.top_logits(student, k)
    zero = distill.distill_fwd_bwd(student, own.ids, own.values, own.lse)
    assert abs(float(zero.loss)) <= 4e-5


MANY = [("bf16", "bf16", 60, 6000, 7), ("f32", "f32", 1021, 2500, 64), ("f16", "f16", 5003, 2100, 20),
        ("bf16", "f32", 16001, 900, 256), ("f32", "f32", 20002, 820, 70), ("bf16", "bf16", 33003, 900, 256),
        ("f16", "f32", 60000, 800, 64), ("bf16", "bf16", 98003, 790, 130), ("f16", "f16", 130001, 780, 256),
        ("f32", "f32", 77001, 780, 33), ("bf16", "f32", 151936, 790, 64), ("bf16", "bf16", 155600, 1100, 256)]


@pytest.mark.parametrize("dtype,out,V,N,k", MANY)
@pytest.mark.parametrize("mode", ["forward", "renormalised", "reverse"])
def test_distill_more_rows_than_workgroups(dtype, out, V, N, k, mode):
    """Rows that follow each other in one workgroup, up to the widest that it keeps: trained ones
    between ones without weight, without entries and with bad entries; entries side by side; tails
    far above and below the entries; the gradient over the logits where types allow."""
    rng = np.random.default_rng(V)
    S, T = 2, N // 2
    g = torch.Generator(device=DEV).manual_seed(V)
    x = torch.randn((S, T, V), device=DEV, generator=g).mul_(3).to(DT[dtype])
    weight = rng.random((S, T)).astype(np.float32) + 0.25
    live = sorted(rng.choice(N, 40, replace=False))
    weight[rng.random((S, T)) < 0.5] = 0
    weight.reshape(-1)[live] = 1.5
    ids, val = np.full((S, T, k), IGNORE, np.int32), np.zeros((S, T, k), np.float32)
    lse = np.full((S, T), 40.0, np.float32)
    some = min(k, V)
    for n in range(N):
        first = int(rng.integers(0, V - some + 1))
        ids.reshape(N, k)[n, :some] = np.arange(first, first + some)
        val.reshape(N, k)[n, :some] = rng.standard_normal(some) + 30
    twice = [n for n in range(N) if n not in live][:2]
    bad = [n for n in range(N) if n not in live][2:4]
    weight.reshape(-1)[twice + bad] = 1
    if some > 1:
        ids.reshape(N, k)[twice, 1] = ids.reshape(N, k)[twice, 0]
    ids.reshape(N, k)[bad, 0] = V
    rows, oracle = x.view(N, V), {}
    for j, n in enumerate(live):
        r = rows[n].float().cpu().numpy()
        at = ids.reshape(N, k)[n]
        if j % 4 == 1:                                        # anywhere in the row
            at[:some] = rng.choice(V, some, replace=False)
        if j % 4 == 2:
            at[rng.random(k) < 0.7] = IGNORE                  # few entries, or none
        used = at[at != IGNORE]
        if len(used) and j % 8 in (2, 6):
            r[used] -= 180 if j % 8 == 2 else -180            # a tail beyond 2^100 on either side
        if j == 8:
            r[:] = -np.inf
            r[used] = 1.0
        rows[n] = torch.from_numpy(r).to(DT[dtype])
        t = rows[n].float().cpu().numpy() + rng.standard_normal(V).astype(np.float32)
        val.reshape(N, k)[n][at != IGNORE] = t[used]
        lse.reshape(-1)[n] = lse_ref(t[None].astype(np.float64))[0]
    forward, tail = mode != "reverse", mode != "renormalised"
    for n in live:
        oracle[n] = row_ref(host64(rows[n]), ids.reshape(N, k)[n], val.reshape(N, k)[n].astype(np.float64),
                            float(lse.reshape(-1)[n]) if tail else None, 1.0, forward)
    ctx = grpo.Context(0)
    args = (torch.from_numpy(ids).to(DEV), torch.from_numpy(val).to(DEV),
            torch.from_numpy(lse).to(DEV) if tail else None, torch.from_numpy(weight).to(DEV))
    o = distill.distill_fwd_bwd(x, *args, divergence="forward" if forward else "reverse", dlogits_dtype=DT[out],
                                sync=False, ctx=ctx)
    with pytest.raises(PcpError):
        ctx.sync()
    tok, dz = host64(o.token_loss).reshape(-1), o.dlogits.view(N, V)
    L = np.maximum(weight.astype(np.float64).sum(1), 1.0)
    for n in live:
        if oracle[n] is None:
            assert tok[n] == 0 and not dz[n].any()
            continue
        l, grad, mag, lb = oracle[n]
        w = float(weight.reshape(-1)[n])
        assert abs(tok[n] - w * l) <= w * lb + 2.0 ** -24 * abs(w * l), n
        c = w / (S * L[n // T])
        bar = c * REL * mag
        # The length is summed in f32: its relative error, 2^-24 log2(T) at most, moves c. A term
        # 2^(x k2 - m) below 2^-126 is 0, with m within 2^60 V of the tail's largest (V <= 2^24): at
        # most 2^-42 of the largest gradient; and so is a result below 2^-126.
        flushed = 2.0 ** -42 * np.abs(c * grad).max() + 2.0 ** -126
        worst = (np.abs(host64(dz[n]) - c * grad) - bar - half_step(out, c * grad) - 2.0 ** -8 * bar
                 - 1e-6 * c * np.abs(grad) - flushed)
        assert worst.max() <= 0, (n, worst.argmax(), worst.max())
    dead = torch.from_numpy((weight.reshape(-1) == 0)).to(DEV)
    dead[bad] = True
    if some > 1:
        dead[twice] = True
    for n in dead.nonzero()[:, 0].tolist():
        assert tok[n] == 0
    assert not dz[dead].any()
    if DT[dtype] == DT[out]:                                  # the same bits over the logits themselves
        distill.distill_fwd_bwd(x, *args, divergence="forward" if forward else "reverse", dlogits=x, sync=False, ctx=ctx)
        with pytest.raises(PcpError):
            ctx.sync()
        assert torch.equal(x, o.dlogits)


def test_distill_two_contexts_at_once():
    """Calls on two streams, each with its own context, give what each gives alone."""
    cases = [make_case(np.random.default_rng(s), 2, 30, 9001, 40) for s in (21, 22)]
    want = [run_distill(c, "bf16", "bf16")[1] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    ctxs = [grpo.Context(0) for _ in cases]
    outs = [[run_distill(c, "bf16", "bf16", stream=s, ctx=x, sync=False)[1] for c, s, x in zip(cases, streams, ctxs)]
            for _ in range(3)]
    for x in ctxs:
        x.sync()
    torch.cuda.synchronize()
    for again in outs:
        for o, w in zip(again, want):
            assert torch.equal(o.dlogits, w.dlogits) and torch.equal(o.token_loss, w.token_loss)
