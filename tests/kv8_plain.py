"""The 8-bit key/value cache, rotary positions and the norm in 64 bits, on the CPU, written from their definitions
(include/w4a16.h) with numpy. (Attention over what a cache holds is kv4_plain.attention.)"""
from __future__ import annotations

import math

import numpy as np
import torch

# e4m3 by code 0..126: exponent field 0 counts 2^-9, field f adds (8 + mantissa) 2^(f - 10)
TABLE = np.array([m * 2.0 ** -9 if f == 0 else (8 + m) * 2.0 ** (f - 10) for f in range(16) for m in range(8)][:127])
VALUES = np.concatenate((TABLE, [np.nan], -TABLE, [np.nan]))


def e4m3(x: np.ndarray):
    """(codes, values) of x, |x| <= 464: the nearest, of two the one with an even code."""
    a = np.abs(np.asarray(x, np.float64))
    up = np.clip(np.searchsorted(TABLE, a), 1, 126)
    lo, hi = TABLE[up - 1], TABLE[up]
    code = np.where(a - lo < hi - a, up - 1, np.where(a - lo > hi - a, up, np.where(up % 2 == 0, up, up - 1)))
    code = np.where(np.signbit(x), code + 128, code).astype(np.uint8)
    return code, VALUES[code]


def scale_of(most: float) -> float:
    """The smallest 2^e, e >= -60, of which 448 are `most` or more."""
    e = -60
    while 448.0 * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


def places(D: int):
    """Byte of a block at which token t's key [16, D] and value [16, D] of dimension d lies."""
    t, d = np.arange(16)[:, None], np.arange(D)[None, :]
    r, x = d // (D // 16), d % (D // 16)
    return 256 * (d // 16) + 16 * t + d % 16, 16 * D + 1024 * (x // 4) + 256 * (t // 4) + 16 * r + 4 * (x % 4) + t % 4


def block_rows(block: np.ndarray, D: int):
    """(keys, values) [16, D] that a block's bytes stand for, in 64 bits; NaN for rows that are not finite."""
    tail = block[32 * D:].tobytes()
    scales, bad = np.frombuffer(tail[:8], np.float32).astype(np.float64), int(np.frombuffer(tail[8:12], np.uint32)[0])
    out = []
    for which, place in enumerate(places(D)):
        x = VALUES[block[place]] * scales[which]
        rows = (bad >> (16 * which + np.arange(16))) & 1
        out.append(np.where(rows[:, None] == 1, np.nan, x))
    return out


def append(cache: np.ndarray, table, b: int, first: int, k: np.ndarray, v: np.ndarray):
    """Tokens first.. of sequence b into the bytes of a cache [pages, Hkv, page / 16, 32 D + 16]: k, v [n, Hkv, D]."""
    pages, Hkv, blocks, width = cache.shape
    D, page = (width - 16) // 32, 16 * blocks
    cap = table.shape[1] * page
    todo = [i for i in range(len(k)) if 0 <= first + i < cap]
    for blk in sorted({(first + i) // 16 for i in todo}):
        number = int(table[b][16 * blk // page])
        if not 0 <= number < pages:
            continue
        mine = [i for i in todo if (first + i) // 16 == blk]
        older = (first + mine[0]) % 16 if first + mine[0] > 0 else 0
        for h in range(Hkv):
            block = cache[number, h, blk % blocks]
            tail = bytearray(block[32 * D:].tobytes())
            bad = int(np.frombuffer(bytes(tail[8:12]), np.uint32)[0])
            for which, (x, place) in enumerate(zip((k, v), places(D))):
                rows = np.asarray(x[mine, h], np.float64)
                fine = np.isfinite(rows).all(-1)
                s = scale_of(np.abs(rows[fine]).max() if fine.any() else 0.0)
                old = float(np.frombuffer(bytes(tail[4 * which:4 * which + 4]), np.float32)[0])
                if older and old > s:
                    s = old
                if older and old < s:
                    block[place[:older]] = e4m3(VALUES[block[place[:older]]] * (old / s))[0]
                for i, row, ok in zip(mine, rows, fine):
                    t = (first + i) % 16
                    block[place[t]] = e4m3(row / s)[0] if ok else 0
                keep = ((1 << older) - 1) << (16 * which)
                mask = 0xFFFF << (16 * which)
                new = sum(1 << (16 * which + (first + i) % 16) for i, ok in zip(mine, fine) if not ok)
                bad = (bad & ~mask & 0xFFFFFFFF) | (bad & keep) | new
                tail[4 * which:4 * which + 4] = np.float32(s).tobytes()
            tail[8:12], tail[12:16] = np.uint32(bad).tobytes(), bytes(4)
            block[32 * D:] = np.frombuffer(bytes(tail), np.uint8)


def held(cache: np.ndarray, table, b: int, n: int):
    """(keys, values) [n, Hkv, D] in 64 bits of sequence b's first n tokens; pages that do not exist: zeros."""
    pages, Hkv, blocks, width = cache.shape
    D, page = (width - 16) // 32, 16 * blocks
    out = np.zeros((2, max(n, 0), Hkv, D))
    for blk in range((n + 15) // 16):
        number = int(table[b][16 * blk // page])
        if 0 <= number < pages:
            m = min(16, n - 16 * blk)
            for h in range(Hkv):
                for which, x in enumerate(block_rows(cache[number, h, blk % blocks], D)):
                    out[which, 16 * blk:16 * blk + m, h] = x[:m]
    return out


def frequencies(rot: int, base: float, scaling: str = "none", factor: float = 1.0, length: float = 0.0, slow: float = 1.0, fast: float = 32.0):
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "ramp":
        share = [min(1.0, max(0.0, (length * x / (2 * math.pi) - slow) / (fast - slow))) for x in f]
        f = [x * s + x / factor * (1 - s) for x, s in zip(f, share)]
    return np.array(f)


def rotate(x: np.ndarray, positions, freq, interleaved: bool, magnitude: float = 1.0):
    """(rows [T, H, D] rotated, bound on what each result was computed from: |a| + |b|)."""
    half = len(freq)
    w = np.asarray(positions, np.float64)[:, None] * freq
    w = np.mod(w, 2 * math.pi)[:, None]
    i = np.arange(half)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, reach = np.array(x, np.float64), np.zeros(x.shape)
    a, b = y[..., lo].copy(), y[..., hi].copy()
    y[..., lo] = magnitude * (a * np.cos(w) - b * np.sin(w))
    y[..., hi] = magnitude * (a * np.sin(w) + b * np.cos(w))
    reach[..., lo] = reach[..., hi] = np.abs(a) + np.abs(b)
    return y, reach * abs(magnitude)


def norm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual=None):
    """(h, y) in 64 bits of rows [..., K]."""
    h = x.double().cpu() if residual is None else x.double().cpu() + residual.double().cpu()
    return h, h / torch.sqrt((h * h).mean(-1, keepdim=True) + float(np.float32(eps))) * weight.double().cpu()
