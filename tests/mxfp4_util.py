"""MXFP4 rows, tables and the operators over them in 64 bits (numpy), for the tests."""
import math

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
D, BLOCK = 128, 32


def bf16_round(x):
    """FP64 -> the nearest BF16 value (ties to even), as FP64; finite values past the
    largest BF16 become infinities."""
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        m, e = np.frexp(x)
        e = np.maximum(e, -125)  # BF16 subnormals: multiples of 2^-133
        y = np.ldexp(np.rint(np.ldexp(x, 8 - e)), e - 8)
        y = np.where(np.abs(y) > float(2 ** 128 - 2 ** 120), np.copysign(np.inf, x), y)
    return np.where(np.isfinite(x), y, x)


def bf16_bits(x):
    """FP64 values that BF16 holds -> their 16 bits."""
    return (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def bf16_values(bits):
    return (np.asarray(bits, np.uint32) << 16).view(np.float32).astype(np.float64)


def values(codes, scales):
    """codes [..., 64], scales [..., 4] (uint8) -> FP64 [..., 128]."""
    n = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], D)
    v = GRID[n & 7] * np.where(n & 8, -1.0, 1.0)
    s = np.ldexp(1.0, scales.astype(np.int64) - 127)
    s = np.where(scales == 255, np.nan, s)
    return v * np.repeat(s, BLOCK, -1)


def quantise(v):
    """FP64 [..., 128] -> (codes, scales), one value after another by distance."""
    b = np.asarray(v, np.float64).reshape(-1, BLOCK)
    bad = ~np.isfinite(b).all(1)
    a = np.abs(np.where(bad[:, None], 0.0, b))
    big = a.max(1)
    e = np.clip(np.where(big > 0, np.frexp(big)[1] - 1, -1000) - 2, -126, 125)
    u = np.ldexp(a, -e[:, None])
    hi = np.clip(np.searchsorted(GRID, u), 1, 7)
    down, up = u - GRID[hi - 1], GRID[hi] - u
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    code = code | np.where(np.signbit(b), 8, 0)
    code[bad] = 0
    code = code.reshape(*v.shape).astype(np.uint8)
    scale = np.where(bad, 255, e + 127).astype(np.uint8).reshape(*v.shape[:-1], D // BLOCK)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def table(rng, lens, page, spare=3):
    """(pool, indptr, indices, last): pages drawn by a permutation of the pool."""
    pages = [max(1, -(-n // page)) for n in lens]
    indptr = np.concatenate([[0], np.cumsum(pages)]).astype(np.int32)
    pool = int(indptr[-1]) + spare
    indices = rng.permutation(pool)[: indptr[-1]].astype(np.int32)
    last = np.array([n - (p - 1) * page for n, p in zip(lens, pages)], np.int32)
    return pool, indptr, indices, last


def random_cache(rng, pool, page, hkv):
    """Head-major codes [pool, hkv, page, 64] and scales [pool, hkv, page, 4] of rows of
    unlike size."""
    codes = rng.integers(0, 256, (pool, hkv, page, 64), dtype=np.uint8)
    scales = rng.integers(123, 128, (pool, hkv, page, 4), dtype=np.uint8)
    return codes, scales


def in_layout(codes, layout):
    return codes if layout == "HND" else np.ascontiguousarray(codes.swapaxes(1, 2))


def rows_of(cache, indptr, indices, r, n):
    """Request r's first n rows [n, hkv, 128] of a head-major cache (codes, scales)."""
    pages = indices[indptr[r]:indptr[r + 1]]
    v = values(cache[0][pages], cache[1][pages]).swapaxes(1, 2)
    return v.reshape(-1, v.shape[2], D)[:n]


def attend(q, k, v, scale=D ** -0.5):
    """q [hq, 128] over k, v [n, hkv, 128]: (out [hq, 128], lse [hq] in log2)."""
    hkv = k.shape[1]
    group = q.shape[0] // hkv
    out, lse = np.empty(q.shape), np.empty(q.shape[0])
    with np.errstate(invalid="ignore", over="ignore"):
        for h in range(hkv):
            heads = slice(h * group, (h + 1) * group)
            s = np.ascontiguousarray(k[:, h]) @ q[heads].T * scale
            m = s.max(0)
            p = np.exp(s - m)
            total = p.sum(0)
            out[heads] = (p / total).T @ np.ascontiguousarray(v[:, h])
            lse[heads] = (m + np.log(total)) / math.log(2)
    return out, lse


def norm_rotate(x, w, pos, eps, theta):
    """x [T, H, 128] (FP64) normed per head by weights w (None: not) and rotated."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    a = np.asarray(pos, np.float64)[:, None] * theta ** (-2.0 * np.arange(64) / 128)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    x1, x2 = x[..., :64], x[..., 64:]
    return np.concatenate([x1 * c - x2 * s, x2 * c + x1 * s], -1)
