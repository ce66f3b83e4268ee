"""What attention over the 8-bit cache guarantees, element by element, from its arithmetic (numpy, float64).

A weight is w = 2^(s + ev - m) with m at least the row's running maximum of s + ev less 8 (s the score in log2 units, ev
the exponent of the token's V block), held as one or two f16 terms times a bias: two terms are good to 2^-21 of the
weight, one to 2^-11, and either ends at half of f16's smallest subnormal, which under the kernels' biases is FLOOR of the
row's largest weight. So an element's error has a part relative to sum p |v| and a part relative to the row's loudest
visible term: FLOOR * max_j(p_j 2^ev_j) * sum_j |code_j|. The denominator is summed from unrounded weights.
"""
from __future__ import annotations

import math

import numpy as np

from oracle import q8 as ref

FLOOR = 2.0 ** -31           # prompts: bias 2^6; single tokens have a bias of 2^10 and stay below it


def attend(q, k, v_codes, v_exps, length, window, sinks, scale, *, terms, out_half_ulp, weight=None):
    """One (batch, group): q [h,T,d], k [C,d] values, v_codes uint8 [C,d], v_exps int8 [NB]. Returns (out, bound), both
    [h,T,d]. `weight` (a function of the weights, scaled so that the row's largest is 2^10) plants a mistake in them."""
    h, T, d = q.shape
    codes = ref._VALUES[v_codes]
    ev = np.repeat(v_exps.astype(np.float64), ref.BLOCK)[:codes.shape[0]]
    out, tol = np.zeros((h, T, d)), np.zeros((h, T, d))
    for t in range(T):
        p = length - T + t
        j = np.nonzero(ref.sees(p, np.arange(length), window, sinks))[0] if p >= 0 else np.zeros(0, int)
        if j.size == 0:
            continue
        for i in range(h):
            s = k[j] @ q[i, t] * scale
            mag = float((np.abs(k[j]) @ np.abs(q[i, t])).max()) * abs(scale)
            w = np.exp(s - s.max())
            prob = w / w.sum()
            if weight is not None:
                scaled = np.exp2(s / math.log(2) + ev[j] - (s / math.log(2) + ev[j]).max() + 10)
                prob = prob * (weight(scaled) / scaled)
            values = codes[j] * np.exp2(ev[j])[:, None]
            out[i, t] = prob @ values
            # a score: 128 products summed in 32 bits (each sum within 2^-23, cut off or rounded), q good to 2^-22 of its
            # largest element; the exponential's argument is rounded at up to A
            A = 16 + float(np.ptp(s / math.log(2) + ev[j]))
            rel = 2 * ((128 * 2 ** -23 + 2 ** -22) * mag + A * 2 ** -23 + 2 ** -22
                       + (2 ** -21 if terms == 2 else 2 ** -11) + j.size * 2 ** -23)
            floor = FLOOR * float((prob * np.exp2(ev[j])).max()) * np.abs(codes[j]).sum(axis=0)
            tol[i, t] = rel * (prob @ np.abs(values)) + floor + out_half_ulp * np.abs(out[i, t])
    return out, tol
