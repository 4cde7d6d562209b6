"""CPU restatement, in numpy float64, of the decoder operators that have no counterpart in the reference: prompt attention with a
sliding window and sinks, the 8-bit key / value cache, and answer probabilities.

TEST INFRASTRUCTURE ONLY — imported by tests/ and by nothing in the product. Written from the formulas; together with every result
comes the largest error that the kernels' roundings can cause (half steps: FP16 2^-11, e4m3 2^-4 relative), so that a test's
tolerance is a bound that follows from its inputs, not a number that was tried.
"""
from __future__ import annotations

import numpy as np

from . import valu

HALF16 = 2.0 ** -11          # half a step of FP16, relative
TINY16 = 2.0 ** -25          # half a step of the smallest FP16 numbers
BLOCK = 64


def rotated(x: np.ndarray, positions, theta: float, llama3: bool = False) -> np.ndarray:
    """x [tokens, dim] in 64 bits, rotated at its positions (pairs p, p + dim / 2)."""
    d = x.shape[1]
    ang = np.asarray(positions, dtype=np.float64)[:, None] * valu.rope_inv_freq(d, theta, llama3)[None, :]
    a, b = x[:, : d // 2], x[:, d // 2:]
    return np.concatenate([a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)], axis=1)


def visible(n_q: int, first: int, n_k: int, window: int, sinks: int) -> np.ndarray:
    """[n_q, n_k]: what the tokens first, first + 1, ... see of the tokens 0 .. n_k - 1 of their sequence."""
    t, c = first + np.arange(n_q)[:, None], np.arange(n_k)[None, :]
    see = c <= t
    return see if window == 0 else see & ((c > t - window) | (c < sinks))


def attend(q, k, v, see, score_err: float, weight_err: float = HALF16, least_weight: float = 2.0 ** -32):
    """softmax(q k^T / sqrt(d)) v over visible keys, and a bound on a kernel's error.

    A score that is off by at most delta_i (here score_err * sum_d |q_d k_d| / sqrt(d)) changes a weight by a factor within
    e^(+-2 delta), the second delta coming in through the sum; weights are rounded by weight_err on their way into the product (the sum
    is taken before); the result is rounded to FP16. 2^-18 stands for 32-bit exponentials and sums.

    `least_weight` bounds the rounding of weights too small for a relative one. A kernel holds 2^s w as FP16, w the weight relative to the
    largest of its column so far, and FP16 numbers below 2^-14 are off by up to 2^-25: w by 2^(-25 - s). Later, larger weights only
    shrink that, and the sum by which all is divided is at least 1 in the same units, so every value adds at most 2^(-25 - s) |v|. s is 7
    for prompts (2^-32). For tokens against the cache it is 15, and the weight carries a factor between 1 and 2 of the values' scale:
    the sum is at least 1/2 in those units, which makes 2^-39."""
    dim = q.shape[1]
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.where(see, q @ k.T / np.sqrt(dim), -np.inf)
        mag = np.where(see, np.abs(q) @ np.abs(k).T / np.sqrt(dim), 0.0)
        delta = score_err * mag.max(axis=1, keepdims=True)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        o = np.zeros((q.shape[0], v.shape[1]))
        spread, floor = np.zeros_like(o), np.zeros_like(o)
        for i in range(q.shape[0]):                     # hidden rows do not enter, whatever they hold
            rows = see[i]
            o[i] = p[i, rows] @ v[rows]
            spread[i] = p[i, rows] @ np.abs(v[rows])
            floor[i] = least_weight * np.abs(v[rows]).sum(axis=0)
    bound = (np.expm1(2.0 * delta) + weight_err + 2.0 ** -18) * spread + floor
    return o, bound + HALF16 * (np.abs(o) + bound) + TINY16


def window_attention(q, k, v, h_q, h_kv, seq_len, columns, window, sinks, theta, llama3=False):
    """q [h_q * dim, columns ...] and so on, channel-major FP16 values in 64 bits -> (out, bound), [h_q * dim, columns].
    q and k reach the tensor cores as FP16 (half a step each) and meet in 32-bit sums."""
    dim = q.shape[0] // h_q
    out, bound = np.zeros((h_q * dim, columns)), np.zeros((h_q * dim, columns))
    for s0 in range(0, columns, seq_len):
        n = min(seq_len, columns - s0)
        pos = np.arange(n)
        see = visible(n, 0, n, window, sinks)
        for h in range(h_q):
            g = h // (h_q // h_kv)
            qq = rotated(q[h * dim: (h + 1) * dim, s0: s0 + n].T, pos, theta, llama3)
            kk = rotated(k[g * dim: (g + 1) * dim, s0: s0 + n].T, pos, theta, llama3)
            o, b = attend(qq, kk, v[g * dim: (g + 1) * dim, s0: s0 + n].T, see, 2.0 * HALF16 * 1.001 + dim * 2.0 ** -24)
            out[h * dim: (h + 1) * dim, s0: s0 + n], bound[h * dim: (h + 1) * dim, s0: s0 + n] = o.T, b.T
    return out, bound


# ---- 8 bits ---------------------------------------------------------------------------------------------------------------------
def e4m3_values() -> np.ndarray:
    """The 256 numbers of e4m3 by code: sign, 4 exponent bits (bias 7), 3 mantissa bits; codes 0x7f and 0xff are NaN."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    mag = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.astype(np.float64) - 10))
    mag = np.where((c & 127) == 127, np.nan, mag)
    return np.where(c & 128, -mag, mag)


def e4m3_half_step(x: np.ndarray) -> np.ndarray:
    """Half a step of e4m3 at |x| (in units of the scale): 2^-4 relative to the power of two below, 2^-10 at least."""
    return np.maximum(2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -30))) - 4), 2.0 ** -10)


# A kernel forms x / scale as x * (1 / scale) in 32 bits: two roundings of 2^-24, 2^-23 of a number that is at most 32 half steps (a half
# step is 1/16 of the power of two below it), so that a value next to the middle between two codes may be up to 32 * 2^-23 = 2^-18 half
# steps beyond it. 2^-17 leaves room for the double rounding of the scale itself.
CODE_SLACK = 1.0 + 2.0 ** -17


def block_scale(x: np.ndarray) -> float:
    """x: the FP16 numbers of a block; NaN does not count, infinities count as the largest number."""
    a = np.minimum(np.abs(x[~np.isnan(x)]), 65504.0)
    return max(float(a.max()) if a.size else 0.0, 2.0 ** -24) / 448.0


# ---- answers ----------------------------------------------------------------------------------------------------------------------
def logprobs(x: np.ndarray):
    """x [rows, columns] FP16 values in 64 bits -> (log probabilities [rows, columns], entropy [columns])."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(axis=0)                      # NaN goes through
        z = x - m
        p = np.exp(z)
        total = p.sum(axis=0)
        lp = z - np.log(total)
        ent = np.log(total) - np.where(p > 0, p * np.where(p > 0, z, 0.0), 0.0).sum(axis=0) / total
        ent = np.where(np.isnan(lp).all(axis=0) | np.isnan(total), np.nan, ent)
    return lp, ent


def top_rows(x: np.ndarray, top: int) -> np.ndarray:
    """[top, columns]: the rows of the largest values, the lowest first among equals; NaN comes last."""
    y = np.where(np.isnan(x), -np.inf, x) + 0.0
    order = np.lexsort((np.broadcast_to(np.arange(x.shape[0])[:, None], x.shape), np.isnan(x), -y), axis=0)
    return order[:top]
