"""The 8-bit paged KV cache in plain numpy, 64 bits: codes, values, attention,
and how far a kernel's output may be from it.

Quantisation: with M = 448 (E4M3) or 127 (INT8), x' = 0 for NaN else x clamped to
+-M 2^119, e the smallest integer >= -100 with max|x'| <= M 2^e, code = x' 2^-e
rounded to the nearest code, ties to even.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import numpy as np

E_MIN = -100
MAX = {"e4m3": 448.0, "int8": 127.0}


def e4m3_table() -> np.ndarray:
    """Values of the 256 E4M3 bytes (the two NaN codes as NaN)."""
    out = np.empty(256)
    for b in range(256):
        x, m = (b >> 3) & 15, b & 7
        a = math.nan if (x, m) == (15, 7) else m * 2.0 ** -9 if x == 0 else (8 + m) * 2.0 ** (x - 10)
        out[b] = -a if b & 128 else a
    return out


def code_values(codes: np.ndarray, fmt: str) -> np.ndarray:
    """codes as bytes -> their values."""
    return e4m3_table()[codes] if fmt == "e4m3" else codes.view(np.int8).astype(np.float64)


def quantise(x: np.ndarray, fmt: str):
    """Rows x [..., hd] (float64) -> (codes as bytes, exponents int8)."""
    top = MAX[fmt]
    x = np.where(np.isnan(x), 0.0, x)
    x = np.clip(x, -top * 2.0 ** 119, top * 2.0 ** 119)
    a = np.abs(x).max(-1)
    e = np.full(a.shape, E_MIN)
    for i, v in np.ndenumerate(a):
        k = E_MIN
        while v > top * 2.0 ** k:
            k += 1
        e[i] = k
    y = x * 2.0 ** -e[..., None].astype(np.float64)
    if fmt == "int8":
        return np.rint(y).astype(np.int8).view(np.uint8), e.astype(np.int8)
    grid = e4m3_table()[:127]
    m = np.abs(y)
    hi = np.clip(np.searchsorted(grid, m), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - m, m - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code + 128 * np.signbit(y)).astype(np.uint8), e.astype(np.int8)


def dequantise(codes: np.ndarray, exps: np.ndarray, fmt: str) -> np.ndarray:
    return code_values(codes, fmt) * 2.0 ** exps[..., None].astype(np.float64)


class Sizes(NamedTuple):
    """What a row's error is measured by, per (row, head) but the first."""
    vabs: np.ndarray  # sum_j w_j |V_j|, per dim
    mag: np.ndarray   # max_j scale sum_d |q_d K_jd|
    wide: np.ndarray  # max_j scale max_d|q_d| sum_d |K_jd|
    top: np.ndarray   # max_j w_j max_d|V_jd|
    n: np.ndarray     # visible positions
    far: np.ndarray   # scale sum_d|q_d| max|K| over all positions, seen or not


def attention(q, k, v, first_pos: int, group: int, scale: float, window: int = 0, sinks: int = 0):
    """q [rows, H, hd], k, v [ctx, Hkv, hd] (float64) -> (out, Sizes)."""
    rows, H, hd = q.shape
    ctx = k.shape[0]
    kk, vv = np.repeat(k, group, 1), np.repeat(v, group, 1)
    z = np.einsum("rhd,jhd->rhj", q, kk) * scale
    p = first_pos + np.arange(rows)[:, None]
    j = np.arange(ctx)[None]
    seen = j <= p
    if window:
        seen &= (j > p - window) | (j < sinks)
    z = np.where(seen[:, None], z, -np.inf)
    z -= z.max(-1, keepdims=True)
    w = np.exp(z)
    w /= w.sum(-1, keepdims=True)
    mag = np.einsum("rhd,jhd->rhj", np.abs(q), np.abs(kk)) * scale
    mag = np.where(seen[:, None], mag, 0.0).max(-1)
    wide = np.where(seen[:, None], np.abs(kk).sum(-1).T[None], 0.0).max(-1) * np.abs(q).max(-1) * scale
    top = (w * np.abs(vv).max(-1).T[None]).max(-1)
    n = np.broadcast_to(seen.sum(-1)[:, None], (rows, H))
    return np.einsum("rhj,jhd->rhd", w, vv), Sizes(np.einsum("rhj,jhd->rhd", w, np.abs(vv)), mag, wide, top, n,
                                                   np.abs(q).sum(-1) * np.abs(kk).max((0, 2)) * scale)


# Roundings, relative to the value: half a step of each type.
HALF = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
# What the kernels may round a softmax weight to before the product with V: two
# fp16 terms for fp32 rows, one bf16 for bf16 rows, one fp16 for fp16 rows.
WEIGHT = {"fp32": 2.0 ** -22, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
# An fp16 result below 2^-14 is a multiple of 2^-24, so rounding to it is off by up
# to 2^-25 whatever its size (an output is that small where the only value with a
# weight that counts is 0); fp32 and bf16 steps go down to 2^-149 and 2^-133.
SMALLEST = {"fp32": 2.0 ** -150, "bf16": 2.0 ** -134, "fp16": 2.0 ** -25}


def tolerance(out, b: Sizes, hd: int, dtype: str) -> np.ndarray:
    """How far an output may be from the exact one.

    A score is a sum of hd products in 32 bits: its error is at most
    (hd + 8) 2^-23 mag (a truncating adder loses a whole step per addition; the 8
    for the scale, the logarithm's base and the exponent's argument). q enters as
    fp16 terms of the row scaled to [1, 2): two leave at most 2^-23 of the row's
    largest element, one (bf16 and fp16 rows) 2^-25 where an element is below
    2^-14 of it: 2^-23 wide. In the kernel for many rows a key's values are fp16
    relative to the largest exponent A of 64 keys, in steps of 2^(A - 30) at the
    coarsest (INT8; 2^(A - 32) for E4M3), where the largest key reaches 2^(A + 6)
    (2^(A + 7)): 2^-36 far. The exponential adds 2^-22. A weight then is off by
    exp(ds) - 1, the sum of the weights by as much plus its n additions, and the
    sum with V by n additions more. A weight is rounded relative to itself, but to
    no less than 2^-25 of the largest contribution w_j 2^(e_j) (an fp16 step
    below 2^-14); times a code that is at most M 2^(e_j) < 2 max_d|V_jd|: n
    2^-24 top in all. The output's own rounding comes on top."""
    ds = (hd + 8) * 2.0 ** -23 * b.mag + 2.0 ** -23 * b.wide + 2.0 ** -36 * b.far + 2.0 ** -22
    rel = 2 * np.expm1(ds) + (2 * b.n + 16) * 2.0 ** -23 + WEIGHT[dtype]
    return (rel[..., None] * b.vabs + (b.n * b.top)[..., None] * 2.0 ** -24 + HALF[dtype] * np.abs(out)
            + SMALLEST[dtype])
