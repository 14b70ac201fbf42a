"""Plain 64-bit forms of the packed and int8-cache ops, with the error bounds their tests use."""
from __future__ import annotations

import numpy as np


def attention(q, k, v, position, heads, kv_heads):
    """q [n, heads * hd], k / v [m, kv_heads * hd] as f64 values, position [n]: query t sees keys [0, position[t]].

    Returns out [n, heads, hd], spread = sqrt(sum_j (p_j v_j)^2) of each output, dot [n, heads] = the largest
    sum_i |q_i k_i| / sqrt(hd) over the keys of a row (what a score's rounding errors are relative to), and mass
    [n, heads, hd] = sum_j |v_j|."""
    n, m = q.shape[0], k.shape[0]
    hd = q.shape[1] // heads
    q = q.reshape(n, heads, hd).astype(np.float64)
    k = k.reshape(m, kv_heads, hd).astype(np.float64)
    v = v.reshape(m, kv_heads, hd).astype(np.float64)
    out, spread, mass, dot = (np.zeros((n, heads, hd)[:k]) for k in (3, 3, 3, 2))
    group = heads // kv_heads
    for t in range(n):
        reach = min(int(position[t]) + 1, m)
        if reach <= 0:
            continue
        for h in range(heads):
            kk, vv = k[:reach, h // group], v[:reach, h // group]
            s = kk @ q[t, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h] = p @ vv
            spread[t, h] = np.sqrt((p * p) @ (vv * vv))
            mass[t, h] = np.abs(vv).sum(0)
            dot[t, h] = np.abs(kk * q[t, h]).sum(1).max() / np.sqrt(hd)
    return out, spread, dot, mass


def attention_bound(out, spread, dot, mass, hd, unit_p, unit_out, floor_p=2.0 ** -38):
    """How far a kernel's out may be off, from the arithmetic:

    - a probability rounded by at most unit_p moves an output by a sum of independent terms, each at most unit_p p_j
      |v_j|: by Hoeffding it passes 8 unit_p spread with probability 2 exp(-32);
    - a score summed in f32 (truncating adds of 16 products, so 2^-23 a step, hd / 16 steps and as many for the
      operand split) is off by at most (hd / 8 + 4) 2^-23 dot, and an exp2 of it by 2^-22 more; the same factor on
      every weight cancels, so half the range counts, on terms of random sign: again 8 spread;
    - sums of weights and of values in f32, rescaled from tile to tile: 64 steps of 2^-23 of the output, and of spread;
    - a weight in f16 has steps of 2^-24 at least, where weights are held under a factor 2^14 that is half a step of
      2^-39 of the largest for each of two terms: floor_p of it on every value, however small its weight;
    - the result's own rounding, unit_out relative."""
    f32 = 2.0 ** -23
    score = (hd / 8 + 4) * f32 * dot[..., None] + 2 * f32
    return 8 * spread * (unit_p + score) + 64 * f32 * (np.abs(out) + spread) + unit_out * np.abs(out) + floor_p * mass + 1e-30


def codes_of(x, scale):
    """rint(x / scale), ties to even, of the real quotient; 0 where the scale is 0 or not finite. x f64, scale f32."""
    scale = np.asarray(scale, np.float32)
    with np.errstate(all="ignore"):
        fine = (scale > 0) & np.isfinite(scale)
        q = np.rint(np.asarray(x, np.float64) / np.where(fine, scale, 1).astype(np.float64))
        return np.where(fine, np.clip(np.nan_to_num(q), -127, 127), 0).astype(np.int8)


def store(x, codes, scales, start, block):
    """Stores x [n, kv_heads, hd] (f64 values) at slots start.. of codes [slots, kv_heads, hd] and scales [blocks,
    kv_heads], in place."""
    n = x.shape[0]
    for b in range(start // block, -(-(start + n) // block)):
        lo, hi = max(b * block, start), min((b + 1) * block, start + n)
        rows = x[lo - start:hi - start]
        with np.errstate(all="ignore"):
            scale = (np.abs(rows).max((0, 2)) / 127.0).astype(np.float32)
        if lo > b * block:
            old = scales[b].copy()
            scale = np.maximum(scale, old)  # a NaN of either wins
            grown = ~(scale == old)
            with np.errstate(all="ignore"):
                kept = codes_of(codes[b * block:lo].astype(np.float64) * old[:, None].astype(np.float64), scale[:, None])
            both_nan = np.isnan(scale) & np.isnan(old)
            pick = (grown & ~both_nan)[None, :, None]
            codes[b * block:lo] = np.where(pick, kept, codes[b * block:lo])
        codes[lo:hi] = codes_of(rows, scale[:, None])
        scales[b] = scale


def values(codes, scales, block):
    """codes [slots, kv_heads, hd], scales [blocks, kv_heads] -> f64 values."""
    with np.errstate(all="ignore"):
        return codes.astype(np.float64) * np.repeat(scales, block, 0)[:codes.shape[0], :, None].astype(np.float64)
