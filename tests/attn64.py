"""Attention rows in 64 bits, with the error that a kernel's declared roundings
allow each value.

Weights w_k = softmax(s)_k, o = sum_k w_k v_k.  A score off by d_k changes o by
sum_k w_k d_k (v_k - o) to first order, a V value off by a relative e_v by at
most e_v sum_k w_k |v_k|, a weight off by a relative e_w by e_w sum_k w_k |v_k|
in the numerator and e_w |o| through the sum.  The result is rounded once to the
output type (half a step: eps / 2, relative).
"""
import numpy as np

HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the smallest subnormal


def attend(q, k, v, scale, qt, e_k=0.0, e_v=0.0, mixed=False):
    """q [d], k, v [n][d] in float64 -> (o [d], allowed error [d]).  e_k, e_v: relative
    roundings of K and V values on their way into the products; mixed: bf16 V whose
    chunks of 16 keys differ in size."""
    d = q.shape[-1]
    if len(k) == 0:
        return np.zeros(d), np.zeros(d)
    prod = k * q
    s = prod.sum(1) * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    o = w @ v
    # scores: fp32 sums of d products (any order: d roundings at most) and their
    # scaling; the exponential, by base 2 with a rounded product, 2^-22 of |s| + 2
    # roundings; relative roundings of K
    size = np.abs(prod).sum(1) * abs(scale)
    ds = size * ((d + 2) * 2.0 ** -24 + e_k) + np.abs(s - s.max()) * 2.0 ** -22 + 2.0 ** -22
    # fp32 sums over the keys, 64 at a time, and of their partial results: n_seq
    # roundings in sequence
    n_seq = 64 + 3 * (len(k) // 64 + 1) / 16
    es = n_seq * 2.0 ** -24
    # weights on their way into the products with V.  For a bf16 result one fp16 term,
    # cut: off by x_k in 0 .. 2^-10, in the sum of the weights too, so that
    # o moves by sum_k w_k x_k (v_k - o), where any constant may be taken off x
    # (sum_k w_k (v_k - o) = 0): 2^-11 sum_k w_k |v_k - o| at most.  For an
    # fp16 result two terms, and a sum of the weights as they were: two of 8 bits would
    # leave 2^-17 of the weight, two of fp16 leave 2^-23 (and the end of fp16: weights
    # of 2^-31 of the largest and less)
    ew = 2.0 ** -11 if qt == "bf16" else 2.0 ** -17
    av = w @ np.abs(v)
    err = (w * ds) @ (np.abs(v) + np.abs(o)) + es * (av + np.abs(o)) + (ew + e_v) * av
    # bf16 V as fp16, 16 keys by a power of two: cut, off by 2^-24 over the scale, which is 2^8,
    # or 1 beside values of 256 and more.  Weights of 2^-31 of the largest and less meet
    # the end of fp16, 2^20 earlier where a chunk is scaled that much more than another
    if qt == "bf16":
        err = err + ew * np.abs(o) + 2.0 ** -31 * w.max() * (np.abs(v).sum(0) + len(v) * np.abs(o))
        err = err + 2.0 ** (-24 if mixed else -32)
        if mixed:
            err = err + 2.0 ** -11 * w.max() * np.abs(v * (np.abs(v).max(1, keepdims=True) < 2.0 ** -12)).sum(0)
            err = err + 2.0 ** -23 * w.max() * np.abs(v).sum(0)
    err = err * 1.02  # second order
    return o, err + (np.abs(o) + err) * HALF_STEP[qt] + TINY[qt]


def check(got, want, err, what=""):
    bad = ~(np.abs(got - want) <= err)
    bad &= ~((got == want) | (np.isnan(got) & np.isnan(want)))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} values off, first at {i}: "
                             f"{got[i]} for {want[i]}, allowed {err[i]:.3g}")
