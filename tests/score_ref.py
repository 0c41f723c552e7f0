"""64-bit references of the token scores and their gradient, from the definitions in include/pcp_score.h, on the
CPU with numpy, and the bars of their tests by forward error analysis.

Forward. A term 2^d, d = (x - m) k2, has the relative error of its exponent's absolute one, ln 2 (2^-24 |d| for
the fma and as much for k2's own rounding), and of v_exp_f32, 2^-23. Weighted by the terms themselves the exponents'
part is 2^-23 of the entropy. A lane adds up to 64 of them in f32, 63 * 2^-24 = 3.8e-6, everything above that in f64.
The logarithm of the sum is therefore off by less than 5e-6 + 2^-23 H, the entropy's other part, sum p (m - x) /
temperature (at most H), by as much of itself and 2^-24 more: REL = 1e-5 of (1 + 2 H) covers them. Outputs are
rounded to f32 once.

Backward. dz = p (A + B d): p from the given row_max and log_sum has the relative error of d, (2^-24 |d| for the fma,
for k2, for log_sum's product with log2 e and for its rounding, natural units: 2^-22 |log p| and 2^-22 |log_sum|), and
2^-23 for the exponential; the products and sums 2^-22 of the terms' magnitudes; the forward's errors of log_sum (REL) and of
the entropy (REL (1 + 2 H) dentropy p) add. A result rounded to 16 bits moves by half a step.
"""
import numpy as np

REL = 1e-5
IGNORE = -100


def softmax_parts(x, tau):
    """x float64 [..., V]: m, log_sum, log p (-inf where p is 0). The temperature is the entry points' f32."""
    m = x.max(-1, keepdims=True)
    d = (x - m) / float(np.float32(tau))
    log_sum = np.log(np.exp(d).sum(-1, keepdims=True))
    return m[..., 0], log_sum[..., 0], d - log_sum


def entropy_of(log_p):
    p = np.exp(log_p)
    return -np.where(p > 0, p * np.where(p > 0, log_p, 0.0), 0.0).sum(-1)


def score_ref(x, ids, tau=1.0, k=0):
    """x float64 [R, V], ids [R] (None: none): logp, entropy, row_max, log_sum, top_logp, top_ids."""
    m, log_sum, log_p = softmax_parts(x, tau)
    logp = np.take_along_axis(log_p, np.asarray(ids)[:, None], 1)[:, 0] if ids is not None else None
    order = np.argsort(-x, axis=1, kind="stable")[:, :k]
    return logp, entropy_of(log_p), m, log_sum, np.take_along_axis(log_p, order, 1), order


def bars(entropy):
    return REL * (1 + 2 * entropy)


def close(got, want, bar):
    """|got - want| within bar and a rounding to f32; infinities where the reference has them."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    # The nearest f32 of a number from 2^128 - 2^103 on (f32's largest and half a step) is infinite: a lowest-value mask
    # over a temperature below 1 is one.
    want = np.where(np.abs(want) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, want), want)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine]), (got[~fine], want[~fine])
    err = np.abs(got[fine] - want[fine])
    lim = np.broadcast_to(bar, want.shape)[fine] + 2.0 ** -24 * np.abs(want[fine])
    assert (err <= lim).all(), (err.max(), lim[np.argmax(err - lim)])


def grad_ref(x, ids, gl, gh, tau=1.0):
    """x float64 [R, V], gl / gh [R]: dlogits float64 [R, V] and the bar of each before its rounding."""
    tau = float(np.float32(tau))
    m, log_sum, log_p = softmax_parts(x, tau)
    h = entropy_of(log_p)[:, None]
    p = np.exp(log_p)
    lp = np.where(p > 0, log_p, 0.0)
    gl, gh = np.asarray(gl, np.float64)[:, None], np.asarray(gh, np.float64)[:, None]
    hot = np.zeros_like(x)
    if ids is not None:
        hot[np.arange(len(x)), ids] = 1.0
    g = (gl * (hot - p) - gh * p * (lp + h)) / tau
    size = p * (np.abs(gl) + np.abs(gh) * (np.abs(lp) + h)) / tau
    rel = REL + 2.0 ** -21 + 2.0 ** -22 * (np.abs(lp) + np.abs(log_sum)[:, None])
    bar = rel * size + REL * (1 + 2 * h) * np.abs(gh) * p / tau + 2.0 ** -23 * np.abs(gl) * hot / tau
    return g, bar + 1e-36 * (np.abs(gl) + np.abs(gh)) / tau


def half_step(v, dtype):
    """How far a value's rounding to `dtype` moves it at most."""
    v = np.abs(v)
    if dtype == "bf16":
        return 2.0 ** -8 * v
    if dtype == "f16":
        return np.maximum(2.0 ** -11 * v, 2.0 ** -25)
    return np.maximum(2.0 ** -24 * v, 2.0 ** -150)
