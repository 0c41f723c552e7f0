"""Bars of the token scores' outputs one by one, by forward error analysis, and long rows whose mass lies where a scan over
them could lose or double an element.

Of a row with logits x, u = (m - x) / temperature >= 0, E = sum p u and M = sum p u^2 (the entropy is log_sum + E).
A term 2^d, d = -u log2 e, has the relative error of its exponent's absolute one, ln 2 |d| 2^-24 for the fma and as much
for the constant's rounding, and of v_exp_f32, 2^-23. A lane adds up to 64 terms of a batch in f32 (63 roundings of
2^-24), takes the largest one's residue out (2^-23 for an exponential, 2^-24 for a product), and everything above that is f64,
but for its rescaling to a new maximum, an exponential (2^-23, and 3 * 2^-24 of the drop, which is part of u) per batch
of the lane and three times more (lanes, waves, parts). With b batches a term is off by
    eps + 2^-22 u,    eps = 64 * 2^-24 + (b + 5) * 2^-23
of itself, and so log_sum by eps + 2^-22 E, which the log-probs take over. sum p u adds to that its own f32 sums (66 roundings
of 2^-24), the error of u as a factor (2^-22 of it), and the division by the sum of the terms:
    2 eps E + 66 * 2^-24 E + 2^-22 (M + E + E^2).
The logarithm has its mantissa's part in f32, 2^-23 of at most 0.35; results are rounded to f32 once.
"""
import numpy as np

BATCH = 8 * 256   # 16-byte vectors


def sharp_bars(x, tau, elem):
    """x float64 [R, V] of logits with elem bytes each: the bars of log_sum (and every log-prob) and of the entropy, [R]."""
    u = (x.max(-1, keepdims=True) - x) / float(np.float32(tau))
    p = np.exp(-u)
    p /= p.sum(-1, keepdims=True)
    u = np.where(p > 0, u, 0.0)
    E, M = (p * u).sum(-1), (p * u * u).sum(-1)
    b = -(-x.shape[-1] * elem // (16 * BATCH))
    eps = 64 * 2.0 ** -24 + (b + 5) * 2.0 ** -23
    log_sum = eps + 2.0 ** -22 * E + 2.0 ** -24
    return log_sum, log_sum + 2 * eps * E + 66 * 2.0 ** -24 * E + 2.0 ** -22 * (M + E + E * E)


def edge_positions(V, elem, offset):
    """Elements of a row that begins `offset` elements past 16 bytes at which a scan of it begins or ends something: the
    row's head and tail, its first and last whole vector, and every 256th vector's first and last element."""
    epv = 16 // elem
    head = min(V, -offset % epv)
    at = set(range(min(V, epv + 1))) | set(range(max(0, V - epv - 1), V))
    for e in range(head, V, 256 * epv):
        at |= {e, e - 1, e + epv - 1}
    return np.array(sorted(i for i in at if 0 <= i < V))


def edge_row(V, elem, offset):
    """A row whose mass, to e^-20 of it, lies at edge_positions, in nearly equal shares."""
    at = edge_positions(V, elem, offset)
    x = np.full(V, -32.0)
    x[at] = 1.0 + np.arange(len(at)) % 7 / 8.0
    return x, at
