"""What attention's rounding may come to, term by term, for the tests that compare with the definition in 64 bits.

With s_j = scale q . k_j, a_j = scale sum_i |q_i k_ji| and w_j the weights:

* scores. fp32: an operand is a tf32 number and a rest (2^-10 of it, truncated to 11 bits); dropped are rest x rest and the rests'
  truncation, each at most 2^-20 of a product, so 3 x 2^-20 a_j at most (queries split to the nearest: half of it); d / 8 additions, of
  which a sum sees half and truncates each by 2^-23 a_j. bf16: products are exact, d / 16 truncated additions.
  eps_j = (3 x 2^-21 + (d / 16 + 4) 2^-23) a_j (fp32), (d / 16 + 4) 2^-23 a_j (bf16); the 4: scaling, maximum, exponential.
* a weight is off by eps_j, their sum by the mean of it: sum_j w_j eps_j |v_j| + (sum_j w_j eps_j) sum_j w_j |v_j|.
* products with values. fp32: 3 x 2^-21 again, four truncated additions per block, a rounded one per block and warp:
  (n / 256 + 16) 2^-23. bf16: weights rounded to 2^-8 of themselves, 2^-16 for exponentials and additions of 16 and of blocks:
  (2^-8 + 2^-16 + n 2^-26) sum_j w_j |v_j|.
* the output's rounding, 2^-24 or 2^-8 of it.
"""

import numpy as np


def attn_bounds(q, k, v, seen, scale, dtype):
    """One head: q [n, d], k / v [m, d] float64, seen [n, m]. Returns (out, lse, bound of out, bound of lse); rows that see nothing: 0, -inf."""
    d, m = q.shape[1], k.shape[0]
    n_seen = seen.sum(1, keepdims=True)
    s = np.where(seen, scale * (q @ k.T), -np.inf)
    a = abs(scale) * (abs(q) @ abs(k).T)
    top = np.where(n_seen > 0, s.max(1, keepdims=True, initial=-np.inf), 0.0)
    w = np.exp(s - top)
    total = w.sum(1, keepdims=True)
    w = w / np.where(total == 0, 1, total)
    out = w @ v
    with np.errstate(divide="ignore"):
        lse = (top + np.log(total))[:, 0]
    eps = ((3 * 2.0 ** -21 if dtype == "f32" else 0) + (d / 16 + 4) * 2.0 ** -23) * a
    mean = (w * eps).sum(1, keepdims=True)
    mag = w @ abs(v)
    err = (w * eps) @ abs(v) + mean * mag
    if dtype == "f32":
        err = err + (3 * 2.0 ** -21 + (n_seen / 256 + 16) * 2.0 ** -23) * mag + 2.0 ** -24 * abs(out)
    else:
        err = err + (2.0 ** -8 + 2.0 ** -16 + n_seen * 2.0 ** -26) * mag + 2.0 ** -8 * abs(out)
    return out, lse, 1.01 * err + 1e-37, 1.01 * (mean[:, 0] + (n_seen[:, 0] / 256 + 16) * 2.0 ** -23) + 2.0 ** -22 * abs(np.where(np.isfinite(lse), lse, 0))


def visible(n, kv_len, window=0, sinks=0):
    j, p = np.arange(kv_len)[None], (kv_len - n + np.arange(n))[:, None]
    return (j <= p) & ((window == 0) | (j > p - window) | (j < sinks))
