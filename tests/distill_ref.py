"""64-bit references of the top logits, the distillation loss and the draft verification, from
their definitions in include/pcp_distill.h and include/pcp_sample.h, on the CPU with numpy.

Bars of the distillation tests, by forward error analysis. Outside the teacher's entries a
gradient is c (P q_v - p_T q_v / q_T), at an entry c (q_i P - p_i), reversed
c q_v (f_v - l): the kernels form each term in f32 from q_v = 2^(x k2 - m) / s. Relative to a
term: the sum s of a lane's up to 160 values and the trees over lanes, waves and parts, about
190 roundings of 2^-24 (1.1e-5); the exponent's fma and k2's own rounding, each 2^-24 ln 2 of
an exponent of at most 60 (2.5e-6 twice); v_exp_f32, the products and the quotient 2^-22 in
all. REL = 2e-5 covers the sum, 1.7e-5, and applies to the sum of the terms' magnitudes, since
they cancel. The log-probabilities have the sum's relative error as an absolute one, so a
token's loss is within REL (1 + sum of |probability * log ratio|). A result rounded to 16 bits
moves by half a step more: 2^-8 (bf16), 2^-11 (f16) of it, or 2^-25 below f16's normal range.
"""
import numpy as np

REL = 2e-5
FLOOR = 2.0 ** -24
IGNORE = -100


def top_ref(x, k, temperature=1.0):
    """x float64 [R, V]: values, ids, lse."""
    x = np.asarray(x, np.float64)
    order = np.argsort(np.where(np.isnan(x), -np.inf, x) * -1.0, axis=1, kind="stable")[:, :k]
    return np.take_along_axis(x, order, 1), order, lse_ref(x / temperature)


def lse_ref(z):
    m = z.max(-1)
    m = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore"):
        return m + np.log(np.exp(z - m[..., None]).sum(-1))


def row_ref(x, ids, t, lse, tau, forward):
    """One row: (l, dl/dz / c with c = 1/tau taken out, sum of term magnitudes per element, bar of l)."""
    V = len(x)
    z = x / tau
    used = (ids != IGNORE) & (t != -np.inf)
    K = ids[used].astype(np.int64)
    if len(K) == 0:
        return None
    tt = t[used] / tau
    lq = lse_ref(z[None])[0]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.exp(z - lq)
        log_q = z[K] - lq
        inside = np.zeros(V, bool)
        inside[K] = True
        rest = z[~inside]
        has_tail = lse is not None and len(rest) > 0 and lse_ref(rest[None])[0] - lq >= -126 * np.log(2)
        log_p = tt - (lse if lse is not None else lse_ref(tt[None])[0])
        p = np.exp(log_p)
        pt = max(1.0 - p.sum(), FLOOR) if has_tail else 0.0
        log_qt = lse_ref(rest[None])[0] - lq if has_tail else 0.0
        qt = np.exp(log_qt) if has_tail else 0.0
        share = np.zeros(V)
        if has_tail:
            share[~inside] = np.exp(rest - lse_ref(rest[None])[0])      # q_v / q_T
        g = np.zeros(V)
        mag = np.zeros(V)
        if forward:
            terms = np.where(p > 0, p * (log_p - log_q), 0.0)
            l = terms.sum()
            size = np.abs(terms).sum()
            if has_tail:
                l += pt * (np.log(pt) - log_qt)
                size += abs(pt * (np.log(pt) - log_qt))
            P = p.sum() + pt
            g = P * q - pt * share
            mag = P * q + pt * share
            g[K] = q[K] * P - p
            mag[K] = q[K] * P + p
        else:
            f = np.where(q[K] > 0, log_q - log_p, 0.0)
            ft = log_qt - np.log(pt) if has_tail else 0.0
            l = (q[K] * f).sum() + qt * ft
            size = np.abs(q[K] * f).sum() + abs(qt * ft)
            g = q * (ft - l) if has_tail else np.zeros(V)
            mag = q * (1.0 + abs(ft) + size)
            g[K] = q[K] * (f - l)
            mag[K] = q[K] * (1.0 + np.abs(f) + size)
    return l, g, mag, REL * (1.0 + size)


def distill_ref(x, ids, t, lse, mask, *, rows, off, tau=1.0, weight=1.0, loss_norm=0.0, forward=True):
    """x float64 [S, LS, V]; returns loss, token_loss [S, TS], dlogits, and bars for the three."""
    S, LS, V = x.shape
    TS = mask.shape[1]
    norm = loss_norm if loss_norm > 0 else S
    tau = float(np.float32(tau))              # the argument is an f32
    tok, tok_bar = np.zeros((S, TS)), np.zeros((S, TS))
    dz, bar = np.zeros(x.shape), np.zeros(x.shape)
    loss = loss_bar = 0.0
    for s in range(S):
        m = mask[s, off:off + rows].astype(np.float64)
        L = max(m.sum(), 1.0)
        for r in range(rows):
            if m[r] == 0:
                continue
            out = row_ref(x[s, r], ids[s, r], t[s, r].astype(np.float64),
                          None if lse is None else float(lse[s, r]), tau, forward)
            if out is None:
                continue
            l, g, mag, lb = out
            c = m[r] * weight / (norm * L * tau)
            tok[s, off + r], tok_bar[s, off + r] = m[r] * l, abs(m[r]) * lb
            dz[s, r], bar[s, r] = c * g, abs(c) * REL * mag
            loss += m[r] * l * weight / (norm * L)
            loss_bar += (abs(m[r]) * lb + 1e-6 * abs(m[r] * l)) * weight / (norm * L)
    return (loss, tok, dz), (loss_bar, tok_bar, bar)


def half_step(dtype, x):
    """Half a step of a 16-bit (or f32) result near x."""
    x = np.abs(x)
    if dtype == "bf16":
        return 2.0 ** -8 * x
    if dtype == "f16":
        return np.maximum(2.0 ** -11 * x, 2.0 ** -25)
    return 2.0 ** -24 * x


def verify_ref(x, y, d, lens, u, T, V):
    """x [S, n+1, V], y [S, n, V] or None (float64), d [S, n], u [S, n+1]."""
    S, n1, _ = x.shape
    n = n1 - 1
    tokens = np.full((S, n1), IGNORE, np.int64)
    accepted, logp = np.zeros(S, np.int32), np.zeros((S, n1))

    def softmax(row):
        e = np.exp((row - row.max()) / T)
        return e / e.sum()

    for s in range(S):
        i = 0
        while True:
            drafted = i < lens[s]
            if T < 1e-6:
                best = int(np.argmax(x[s, i]))
                tokens[s, i] = best
                if drafted and d[s, i] == best:
                    i += 1
                    continue
                break
            p = softmax(x[s, i])
            r = p
            if drafted:
                ok = 0 <= d[s, i] < V
                q = np.zeros(V)
                if ok and y is not None:
                    q = softmax(y[s, i])
                elif ok:
                    q[d[s, i]] = 1.0
                if ok and u[s, i] * q[d[s, i]] < p[d[s, i]]:
                    tokens[s, i], logp[s, i] = d[s, i], np.log(p[d[s, i]])
                    i += 1
                    continue
                r = np.maximum(p - q, 0.0)
                if not r.any():
                    r = p
            c = np.cumsum(r)
            v = int(np.searchsorted(c, float(u[s, n]) * c[-1], side="right"))
            tokens[s, i] = min(v, np.flatnonzero(r)[-1])
            logp[s, i] = np.log(p[tokens[s, i]])
            break
        accepted[s] = i
    return tokens, accepted, logp
