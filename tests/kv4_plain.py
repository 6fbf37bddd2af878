"""The 4-bit key/value cache in 64 bits, on the CPU: quantisation, block layout and attention,
written from their definitions (include/w4a16.h) with numpy and loops over tokens."""
from __future__ import annotations

import numpy as np
import torch


def quantise(x: torch.Tensor):
    """Rows [..., D] of fp16 or bfloat16 as (nibbles, scale (x's type), zero, value held in 64 bits)."""
    d = x.double().numpy()
    with np.errstate(all="ignore"):
        lo, hi = np.minimum(d.min(-1), 0), np.maximum(d.max(-1), 0)
        s16 = torch.from_numpy(((hi - lo) / 15).astype(np.float32)).to(x.dtype)
        bad = ~np.isfinite(d).all(-1)
        s = s16.double().numpy()
        some = (s > 0) & ~bad
        div = np.where(some, s, 1.0)
        z = np.where(some, np.clip(np.rint(-lo / div), 0, 15), 0.0)
        n = np.clip(np.rint(d / div[..., None]) + z[..., None], 0, 15)
        n = np.where(some[..., None], n, 0.0)
        held = np.where(bad[..., None], np.nan, (n - z[..., None]) * s[..., None])
    s16 = torch.where(torch.from_numpy(bad), torch.full_like(s16, float("nan")), s16)
    return n.astype(np.uint8), s16, z.astype(np.uint32), held


def rounded(held: np.ndarray, dtype) -> torch.Tensor:
    most = torch.finfo(dtype).max
    return torch.from_numpy(np.clip(held, -most, most)).to(torch.float32).to(dtype)


def pack(cache: np.ndarray, slot: int, h: int, which: int, n, s16: torch.Tensor, z):
    """One quantised row into the cache's bytes, nibble by nibble."""
    D = (cache.shape[3] - 128) // 16
    page = cache.shape[2] * 16
    block = cache[slot // page, h, slot % page // 16]
    t = slot % 16
    for d in range(D):
        if which == 0:
            nib = t * D + d
        else:
            c, r = divmod(d, D // 16)
            u, p, i = t // 4, t // 2 % 2, t % 2
            nib = 2 * (8 * D + u * 2 * D + c * (D // 8) + p * (D // 16) + (r // 4) * 4 + 2 * i) + r % 4
        b, sh = nib // 2, 4 * (nib % 2)
        block[b] = (int(block[b]) & ~(15 << sh) & 255) | int(n[d]) << sh
    at = 16 * D + 64 * which + 4 * t
    word = int(s16.view(torch.int16).item()) & 0xFFFF | int(z) << 16
    block[at:at + 4] = np.frombuffer(np.uint32(word).tobytes(), np.uint8)


def attention(q, k, v, nq, lens, causal=True, window=0, scale=None, seen=None):
    """(out, lse, spread, reach, vtop) in 64 bits: q [T, Hq, D] rows of sequence after sequence, k and v
    lists of [len, Hkv, D] arrays. spread: sum p |v| / sum p; reach: the largest sum of |q k| scale of
    a row, vtop: the largest |v| of its sequence and head, all for error bounds. seen: per sequence a mask [len] of keys that exist at all."""
    T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out, spread = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    lse, reach = np.full((T, Hq), -np.inf), np.zeros((T, Hq))
    vtop = np.zeros((T, Hq))
    at = 0
    for b, (n, L) in enumerate(zip(nq, lens)):
        G = Hq // k[b].shape[1]
        for i in range(n):
            pos = L - n + i
            j = np.arange(L)
            see = (j <= pos) if causal else np.ones(L, bool)
            if window:
                see &= j > pos - window
            if seen is not None:
                see &= seen[b]
            if not see.any():
                continue
            for a in range(Hq):
                vtop[at + i, a] = np.abs(v[b][:, a // G]).max()
                kk, vv = k[b][see, a // G], v[b][see, a // G]
                with np.errstate(all="ignore"):
                    w = kk @ q[at + i, a] * scale
                    m = w.max()
                    p = np.exp(w - m)
                    out[at + i, a] = p @ vv / p.sum()
                    spread[at + i, a] = p @ np.abs(vv) / p.sum()
                    lse[at + i, a] = m + np.log(p.sum())
                    reach[at + i, a] = (np.abs(kk) @ np.abs(q[at + i, a])).max() * abs(scale)
        at += n
    return out, lse, spread, reach, vtop
