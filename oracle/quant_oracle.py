"""The 8-bit serving operators of include/denoiser_b200_quant.h in 64 bits
(numpy), from their definition."""
from __future__ import annotations

import numpy as np

TINY = np.float32(2.0 ** -126)


def quantise(x, bits: int = 8, group: int = 0):
    """Codes (int8, one a value) and scales (FP32) of the rows of x (FP16 or
    FP32): s = max(fl32(max |x| fl32(1 / qmax)), 2^-126), the code the whole number
    nearest to x / s, halves to even. The quotient in 64 bits decides every
    border of 24-bit numbers rightly: it is a half exactly, or further from one
    than its rounding. A group with a NaN or an infinity: s = NaN, codes 0."""
    x = np.asarray(x)
    rows, cols = x.shape
    group = group or cols
    qmax = 127 if bits == 8 else 7
    v = x.astype(np.float64).reshape(rows, cols // group, group)
    fine = np.isfinite(v).all(axis=2, keepdims=True)
    a = np.where(fine, np.abs(np.where(fine, v, 0.0)).max(axis=2, keepdims=True), 0.0).astype(np.float32)
    s = np.maximum(a * (np.float32(1) / np.float32(qmax)), TINY)
    q = np.rint(np.where(fine, v, 0.0) / s.astype(np.float64)).astype(np.int8)
    s = np.where(fine, s, np.float32(np.nan))
    return q.reshape(rows, cols), s.reshape(rows, cols // group)


def pack(q, bits: int):
    """Code bytes of the rows as the cache holds them (without row padding)."""
    if bits == 8:
        return q.view(np.uint8)
    rows, cols = q.shape
    n = np.zeros((rows, (cols + 1) // 2 * 2), np.uint8)
    n[:, :cols] = q.view(np.uint8) & 15
    return n[:, 0::2] | (n[:, 1::2] << 4)


def values(q, s):
    """What codes and scales stand for, in 64 bits."""
    rows, cols = q.shape
    return (q.astype(np.float64).reshape(rows, s.shape[1], cols // s.shape[1]) * s.astype(np.float64)[:, :, None]).reshape(rows, cols)


def product(q, s, qw, sw, bias=None, gate: bool = False, segments: int = 1):
    """The layer's output in 64 bits from codes (rows, K), scales (rows,
    segments), weight codes (cout, K) and scales (cout, 1); and for each output
    the bound on what `roundings(segments)` FP32 roundings of its terms add up
    to."""
    rows, k = q.shape
    c = k // segments
    eps = 2.0 ** -24
    terms = np.zeros((rows, qw.shape[0]))
    y = np.zeros_like(terms)
    for t in range(segments):
        acc = (q[:, t * c:(t + 1) * c].astype(np.float64) @ qw[:, t * c:(t + 1) * c].astype(np.float64).T)
        p = acc * s[:, t:t + 1].astype(np.float64) * sw.astype(np.float64).T
        y += p
        terms += np.abs(p)
    if bias is not None:
        y = y + np.asarray(bias, np.float64)
        terms = terms + np.abs(np.asarray(bias, np.float64))
    e = (segments + 4) * eps * terms
    if gate:
        h = y.shape[1] // 2
        a, b, ea, eb = y[:, :h], y[:, h:], e[:, :h], e[:, h:]
        e = np.abs(a) * eb + np.abs(b) * ea + ea * eb + eps * np.abs(a * b)
        y = a * b
    return y, e


def output_bound(y, e, dtype):
    """`e` and the rounding to the output type: half a step relative to the
    value, or half the smallest step."""
    half = 2.0 ** -11 if np.dtype(dtype) == np.float16 else 2.0 ** -24
    least = 2.0 ** -25 if np.dtype(dtype) == np.float16 else 2.0 ** -150
    return e + (np.abs(y) + e) * half + least
