"""Plain implementations of the 8-bit serving operators in numpy, for their tests: the group
quantisation and its uses in the operators' own f32 order of operations (codes, scales and
products are compared bit for bit), the attention in float64."""
from __future__ import annotations

import numpy as np

F32 = np.float32
TINY = F32(2.0 ** -100)


def scale_of(amax):
    amax = np.asarray(amax, F32)
    with np.errstate(all="ignore"):
        s = np.where(amax < TINY, F32(0), amax / F32(127))
    return np.where(np.isfinite(amax), s, F32(np.nan)).astype(F32)


def codes_of(x, scale):
    x, scale = np.asarray(x, F32), np.asarray(scale, F32)
    with np.errstate(all="ignore"):
        inv = np.where(scale > 0, F32(1) / scale, F32(0)).astype(F32)
        c = np.rint(x * inv)
    return np.where(np.broadcast_to(scale > 0, c.shape), np.nan_to_num(c), 0).clip(-127, 127).astype(np.int8)


def quantize_rows(x):
    s = scale_of(np.abs(np.asarray(x, F32)).max(1))
    return codes_of(x, s[:, None]), s


def matmul(x, xs, w, ws, add=None):
    """f32 result before its rounding to the output type."""
    acc = (x.astype(np.int64) @ w.astype(np.int64).T).astype(F32)
    y = acc * xs[:, None].astype(F32) * ws.astype(F32)
    return y if add is None else y + add.astype(F32)


def rope_table(n, dim, base=1e4):
    a = np.outer(np.arange(n), base ** (-np.arange(0, dim, 2) / dim))
    return np.stack([np.cos(a), np.sin(a)], -1).astype(F32)


def make_ready(x, pos, norm=None, eps=0.0, rope=None, interleaved=False):
    """x [tokens][heads][dim] f32: norm and rotation in the operator's order of f32 operations."""
    x = np.asarray(x, F32)
    if norm is not None:
        ms = (x.astype(np.float64) ** 2).sum(-1, keepdims=True) / x.shape[-1] + np.float64(F32(eps))
        x = x * (1.0 / np.sqrt(ms)).astype(F32) * norm.astype(F32)
    if rope is None:
        return x
    half = rope.shape[1]
    c, s = rope[pos, :, 0][:, None], rope[pos, :, 1][:, None]
    x = x.copy()
    a = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    p, q = x[..., a[0]].copy(), x[..., a[1]].copy()
    x[..., a[0]] = p * c - q * s
    x[..., a[1]] = p * s + q * c
    return x


def append(codes, scales, table, lens, new, x):
    """New rows x [tokens][kv heads][dim] f32 into codes [pages][heads][page][dim] and scales, in place."""
    page, at = codes.shape[2], 0
    for s, (n, m) in enumerate(zip(lens, new)):
        p = n - m
        while p < n:
            end = min(n, p // 16 * 16 + 16)
            rows, r0 = x[at:at + end - p], p % 16
            pg, blk = table[s][p // page], p % page // 16
            for h in range(codes.shape[1]):
                fresh = scale_of(np.abs(rows[:, h]).max())
                old = F32(0) if r0 == 0 else scales[pg, h, blk]
                now = F32(np.nan) if np.isnan(fresh) or np.isnan(old) else max(old, fresh)
                cell = codes[pg, h, blk * 16:blk * 16 + 16]
                if r0 and not now == old:
                    ratio = old / now if now > 0 else F32(0)
                    cell[:r0] = np.rint(cell[:r0].astype(F32) * ratio).astype(np.int8)
                scales[pg, h, blk] = now
                cell[r0:r0 + end - p] = codes_of(rows[:, h], now)
            at, p = at + end - p, end


def values(codes, scales, table_row, n):
    """float64 [positions][kv heads][dim] of a sequence's first n positions."""
    page = codes.shape[2]
    need = -(-n // page)
    c = codes[table_row[:need]].astype(np.float64) * np.repeat(scales[table_row[:need]].astype(np.float64), 16, 2)[..., None]
    return c.transpose(0, 2, 1, 3).reshape(-1, codes.shape[1], codes.shape[3])[:n]


def attention(q, k, v, first, scale, weight_eps=0.0):
    """q [tokens][heads][dim] at positions first + i over k, v [positions][kv heads][dim], float64.
    Returns the output and a bound on an f32 implementation's error (see the GPU tests)."""
    q = q.astype(np.float64)
    g = q.shape[1] // k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape[:2])
    for i in range(q.shape[0]):
        n = max(0, first + i + 1)
        for h in range(q.shape[1]):
            if n == 0:
                continue
            kk, vv = k[:n, h // g], v[:n, h // g]
            x = kk @ q[i, h] * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            out[i, h] = w @ vv
            # scores: q in fixed point, 22 bits under its row's maximum (half a step of 2^-22),
            # the sum of the three limbs, the factor, the added exponent and the difference to the
            # maximum rounded once each in f32 (6 x 2^-24 of the largest score in base 2)
            dx = np.abs(q[i, h]).max() * 2.0 ** -22 * np.abs(kk).sum(1).max() * abs(scale)
            dx += 6 * 2.0 ** -24 * (np.abs(x).max() + 40)
            # weights: exp2 2^-22, two f16 parts 2^-22; the sums over blocks of 16, warps and chunks
            dw = 2.0 ** -21 + (n / 16 + 16) * 2.0 ** -23
            # weight_eps: weights rounded once to fewer bits, each off by at most that share of
            # itself: |sum (w + dw) v - sum w v| <= weight_eps sum w |v| (the sum that divides them is
            # of the weights before that rounding)
            tol[i, h] = (2 * dx + 2 * dw + weight_eps) * (w @ np.abs(vv)).max() + 1e-30
    return out, tol
