"""The operators between a decoder layer's linear layers: root-mean-square norm with the residual's
addition (its result in 16 bits, or in 8 with scales), rotary positions, and a key/value cache held
in 8 bits with a scale for each block of 16 tokens and head: writing it (keys rotated on the way),
reading it back, and attention over it, from one token of one sequence to prompts and long contexts.

`run` computes them in plain torch operations where `own` is false, and through the library where
it is true, on the same inputs and cache bytes. "8 bits" is e4m3 (no infinities, largest value 448).

  norm       h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight; the sum h is returned too.
             In 8 bits: scale = max(largest |y| of a group / 448, 2^-100), y / scale rounded to e4m3.
  rope       pairs (a, b) of a row, dimensions (i, i + rot / 2) or (2 i, 2 i + 1), become
             m (a cos w - b sin w, a sin w + b cos w) with w = position * frequency i and a magnitude
             m; what lies beyond rot dimensions stays.
  cache      uint8 [pages, kv heads, page_size / 16, 32 D + 16]: blocks of 16 tokens of one head:
               keys     [D / 16][16 tokens][16 dimensions]
               values   [D / 64 g][4 quads][16 r][4 e][4 i]: token 4 quad + i, dimension r D / 16 + 4 g + e
               scales   fp32 of keys, of values; then 8 bytes for rows that are not finite (none here)
             A block's scale is the smallest power of two, 2^-60 at least, such that nothing in it
             passes 448 scales. Tokens are appended: a block that has some already keeps its scale or
             raises it, and then holds the older rows rounded at the new one.
  attention  softmax(scale q k^T) v over what the cache holds, and ln of the sum of exponentials.

A case is a dict of plain values: `op` is "norm", "rope", "roundtrip" (rows are rotated, written and
read back) or "attention" (`q` new tokens of each of `B` sequences, whose lengths with them are at
most `kv`).
"""
from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
MOST = 448.0
EPS = 1e-5
BASE = 500000.0


def _package():
    """The package of the tree this process runs in (its folder is no Python identifier)."""
    name = "triton_rs_amd"
    if name not in sys.modules:
        path = os.path.join(ROOT, "triton-rs_amd")
        spec = importlib.util.spec_from_file_location(
            name, os.path.join(path, "__init__.py"), submodule_search_locations=[path])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ------------------------------------------------------------------ the cases

def _norm(name, T, H, K, dtype, residual=True, group=-1):
    """`group`: -1 a result in 16 bits, else in 8 with a scale for so many values (0: for a row)."""
    c = {"op": "norm", "T": T, "H": H, "K": K, "dtype": dtype, "residual": residual, "group": group}
    return {"name": name, **c} if name else c


def _rope(name, T, Hq, Hkv, D, dtype, rot=0, interleaved=False, scaling="none", at=0):
    c = {"op": "rope", "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "rot": rot or D,
         "interleaved": interleaved, "scaling": scaling, "at": at}
    return {"name": name, **c} if name else c


def _roundtrip(name, B, q, kv, Hq, Hkv, D, page, dtype, ragged=False, rot=-1, interleaved=False):
    c = {"op": "roundtrip", "B": B, "q": q, "kv": kv, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
         "dtype": dtype, "ragged": ragged, "rot": D if rot < 0 else rot, "interleaved": interleaved}
    return {"name": name, **c} if name else c


def _attention(name, B, q, kv, Hq, Hkv, D, page, dtype, ragged=False, causal=True, window=0):
    c = {"op": "attention", "B": B, "q": q, "kv": kv, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
         "dtype": dtype, "ragged": ragged, "causal": causal, "window": window}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the norm ahead of a linear layer for one token: latency
        _norm("norm_t1_k4096", 1, 1, 4096, "f16"),
        # rows of an odd width for a program's own 8-bit product, a scale a row, no residual
        _norm("norm_8bit_t777_k5003", 777, 1, 5003, "bf16", residual=False, group=0),
        # a prompt's rows in 8 bits with a scale for every 128 values
        _norm("norm_8bit_t8192_k4096_g128", 8192, 1, 4096, "bf16", group=128),
        # the queries and keys of a decode step, sixteen tokens, each at its own position
        _rope("rope_t16", 16, 32, 8, 128, "f16"),
        # those of a long prompt far into a document: part of the head, neighbours paired, stretched
        _rope("rope_partial_t8192", 8192, 32, 8, 128, "bf16", rot=96, interleaved=True, scaling="ramp", at=900000),
        # the new token of each of 48 sequences, appended to blocks that are partly filled
        _roundtrip("append_b48", 48, 1, 4096, 32, 8, 128, 16, "bf16", ragged=True),
        # the rows of prompts of all lengths
        _roundtrip("prompts_b5_t2048", 5, 2048, 2048, 32, 8, 128, 64, "f16", ragged=True),
        # one decode step of one sequence that has just begun: latency
        _attention("decode_b1_kv500", 1, 1, 500, 32, 8, 128, 16, "f16"),
        # one decode step of a serving batch, sequences of all lengths
        _attention("decode_b48_kv4096", 48, 1, 4096, 32, 8, 128, 16, "bf16", ragged=True),
        # five drafted tokens of each of eight sequences verified at once, sliding window, one
        # wide head of keys and values to eight of queries
        _attention("verify_b8_q5_kv6000", 8, 5, 6000, 16, 2, 256, 32, "f16", ragged=True, window=4096),
        # a batch of prompts of all lengths, as many heads of keys as of queries
        _attention("prompts_b7_q1500", 7, 1500, 1500, 16, 16, 64, 16, "f16", ragged=True),
        # a prefill chunk behind a long context
        _attention("chunk_q1024_kv32768", 1, 1024, 32768, 32, 8, 128, 64, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


HEADS = [(32, 8, 128), (32, 8, 128), (64, 8, 128), (28, 4, 128), (16, 16, 64), (12, 12, 64), (16, 2, 256),
         (24, 1, 128), (12, 4, 192)]


def draw(rng):
    kind = rng.choice(["norm", "norm", "rope", "rope", "roundtrip", "roundtrip", "decode", "verify", "prompt", "chunk"])
    dtype, page = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
    if kind == "norm":
        if rng.random() < 0.25:   # the heads of queries or keys
            H, K = rng.choice([(8, 128), (32, 128), (16, 64), (16, 256), (5, 80)])
            return _norm(None, _log_int(rng, 1, 8192), H, K, dtype, residual=False)
        K = rng.choice([rng.randint(32, 16384), 64 * rng.randint(1, 256), 128 * rng.randint(1, 128)])
        groups = [-1, -1, 0] + [g for g in (32, 64, 128) if K % g == 0]
        return _norm(None, _log_int(rng, 1, min(8192, 8192 * 4096 // K)), 1, K, dtype, rng.random() < 0.7, rng.choice(groups))
    Hq, Hkv, D = rng.choice(HEADS)
    rot = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
    if kind == "rope":
        T = _log_int(rng, 1, 8192 * 5120 // ((Hq + Hkv) * D))
        return _rope(None, T, Hq, Hkv, D, dtype, rot, rng.random() < 0.5, rng.choice(["none", "linear", "base", "ramp"]),
                     rng.choice([0, _log_int(rng, 1, 1000000)]))
    if kind == "roundtrip":
        rot = rng.choice([0, rot, rot])
        B = _log_int(rng, 1, 64)
        if rng.random() < 0.5:
            q = rng.randint(1, 8)
            return _roundtrip(None, B, q, rng.randint(q, 4096), Hq, Hkv, D, page, dtype, True, rot, rng.random() < 0.5)
        q = _log_int(rng, 1, max(1, int(10240 * 1024 / (B * max(1024, Hkv * D)))))
        return _roundtrip(None, B, q, q, Hq, Hkv, D, page, dtype, B > 1, rot, rng.random() < 0.5)
    cost = Hkv * D / 1024.0
    window = rng.choice([0, 0, 0, _log_int(rng, 64, 4096)])
    if kind in ("decode", "verify"):
        B = _log_int(rng, 1, 64)
        kv = _log_int(rng, 1, int(min(65536, 262144 / B / max(1.0, cost))))
        q = 1 if kind == "decode" else min(kv, rng.randint(2, 16))
        return _attention(None, B, q, kv, Hq, Hkv, D, page, dtype, rng.random() < 0.6, True, window)
    # the products of one pass, and the logits that the plain form holds, within the largest listed
    most = 1024 * 32768 * 32
    if kind == "prompt":
        B = _log_int(rng, 1, 8)
        q = _log_int(rng, 17, int(min(2048, math.sqrt(most * 128 / (B * Hq * max(D, 128))))))
        return _attention(None, B, q, q, Hq, Hkv, D, page, dtype, B > 1, rng.random() < 0.8, window)
    q = _log_int(rng, 17, 1024)
    kv = _log_int(rng, q, int(min(32768, max(q, most * 128 / (q * Hq * max(D, 128))))))
    return _attention(None, 1, q, kv, Hq, Hkv, D, page, dtype, False, True, window)


def _lengths(case):
    """(new tokens, length with them) of each sequence, from the case alone."""
    B, q, kv = case["B"], case["q"], case["kv"]
    if not case["ragged"]:
        return [q] * B, [kv] * B
    rng = random.Random(B * 7919 + q * 31 + kv)
    if q == kv:   # whole prompts
        n = [q] + [rng.randint(1, q) for _ in range(B - 1)]
        return n, n
    return [q] * B, [kv] + [rng.randint(q, kv) for _ in range(B - 1)]


def _scaling(case):
    """How frequencies are stretched: (kind, factor, original length, slow, fast turns), magnitude."""
    kind = case.get("scaling", "none")
    return (kind, 1.0 if kind == "none" else 8.0, 8192.0, 1.0, 4.0), 1.2 if kind == "ramp" else 1.0


# ------------------------------------------------------------------ the plain forms

def _round(x, dtype):
    """x in the element type, saturated to its largest finite value."""
    most = torch.finfo(dtype).max
    return x.clamp(-most, most).to(dtype)


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    total = [] if s["residual"] is None else [h.to(s["x"].dtype)]
    if s["group"] < 0:
        return [y.to(s["x"].dtype)] + total
    g = y.unflatten(-1, (-1, s["group"] or y.shape[-1]))
    scale = (g.abs().amax(-1) / MOST).clamp(min=2.0 ** -100)
    return [(g / scale[..., None]).to(E4M3).flatten(-2), scale] + total


def _frequencies(rot, scaling):
    """Radians a position of pair i, float64 [rot / 2]."""
    kind, factor, length, slow, fast = scaling
    base = BASE * factor ** (rot / (rot - 2)) if kind == "base" and rot > 2 else BASE
    f = base ** (torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / -rot)
    if kind == "linear":
        return f / factor
    if kind == "ramp":
        share = ((length * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        return f * (share + (1 - share) / factor)
    return f


def _rotate(x, positions, freq, magnitude, interleaved):
    """Rows x [T, H, D] rotated at positions [T], in fp32 (angles in 64 bits)."""
    rot = 2 * freq.numel()
    w = positions.double()[:, None, None] * freq
    cos, sin = (magnitude * w.cos()).float(), (magnitude * w.sin()).float()
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, d = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _scale_of(most):
    """The smallest power of two, 2^-60 at least, of which 448 are `most` or more (fp32)."""
    _, e = torch.frexp(most / 448.0)   # most / 448 <= 2^e, and 2^(e - 1) where that is what it is
    e = e - (torch.ldexp(torch.ones_like(most), e - 1) * 448.0 >= most).int()
    return torch.ldexp(torch.ones_like(most), torch.where(most > 0, e, -60).clamp(min=-60))


def _values_order(D):
    """Dimension and token of each byte of a block's values [16 D]."""
    at = torch.arange(16 * D, device="cuda")
    g, quad, r, e, i = at // 1024, at // 256 % 4, at // 16 % 16, at // 4 % 4, at % 4
    return r * (D // 16) + 4 * g + e, 4 * quad + i


def _pack(k, v):
    """Blocks' keys and values [..., 16, D] (fp32), and their scales, as bytes [..., 32 D + 16]."""
    lead, D = k.shape[:-2], k.shape[-1]
    sk, sv = (_scale_of(x.abs().amax((-2, -1))) for x in (k, v))
    return _pack_at(k, v, sk, sv, lead, D)


def _pack_at(k, v, sk, sv, lead, D):
    nk = (k / sk[..., None, None]).to(E4M3).view(torch.uint8)
    nv = (v / sv[..., None, None]).to(E4M3).view(torch.uint8)
    dim, tok = _values_order(D)
    nk = nk.view(*lead, 16, D // 16, 16).transpose(-2, -3).reshape(*lead, 16 * D)
    words = torch.stack((sk, sv, torch.zeros_like(sk), torch.zeros_like(sk)), -1)
    return torch.cat((nk, nv[..., tok, dim], words.contiguous().view(torch.uint8)), -1)


def _blocks(blocks):
    """Keys and values [..., 16, D] in fp32 of whole blocks [..., 32 D + 16], and their scales."""
    D = (blocks.shape[-1] - 16) // 32
    lead = blocks.shape[:-1]
    words = blocks[..., 32 * D:32 * D + 8].contiguous().view(torch.float32)
    k = blocks[..., :16 * D].contiguous().view(E4M3).float().view(*lead, D // 16, 16, 16).transpose(-2, -3)
    dim, tok = _values_order(D)
    order = torch.empty(16 * D, dtype=torch.long, device="cuda")
    order[tok * D + dim] = torch.arange(16 * D, device="cuda")
    v = blocks[..., 16 * D:32 * D][..., order].view(E4M3).float().view(*lead, 16, D)
    return k.reshape(*lead, 16, D) * words[..., 0, None, None], v * words[..., 1, None, None], words


def _plain_roundtrip(s):
    k, v, cache = s["k"].float(), s["v"].float(), s["cache"]
    Hkv, D = k.shape[1:]
    positions, slots = s["positions"], s["slots"].long()
    q = []
    if s["freq"] is not None:
        k = _rotate(s["k"], positions, s["freq"], 1.0, s["interleaved"])
        q = [_round(_rotate(s["q"], positions, s["freq"], 1.0, s["interleaved"]), s["q"].dtype)]
    # the blocks that are written, as they are
    number, block = torch.unique(slots // 16, return_inverse=True)
    per = cache.shape[2]
    place = (number // per, slice(None), number % per)
    old_k, old_v, words = _blocks(cache[place])                       # [U, Hkv, 16, D]
    first = torch.full((len(number),), 16, device="cuda").scatter_reduce_(0, block, slots % 16, "amin")
    older = (torch.arange(16, device="cuda") < first[:, None])[:, None, :, None]
    some = (first > 0)[:, None]
    new, held = [], []
    for x, old, word in ((k, old_k, words[..., 0]), (v, old_v, words[..., 1])):
        rows = torch.where(older, old, 0)
        rows[block, :, slots % 16] = x
        scale = torch.maximum(_scale_of(rows.abs().amax((-2, -1))), torch.where(some, word, 0))
        new.append((rows, scale))
        held.append((rows / scale[..., None, None]).to(E4M3).float() * scale[..., None, None])
    cache[place] = _pack_at(new[0][0], new[1][0], new[0][1], new[1][1], new[0][0].shape[:2], D)
    return [_round(x[block, :, slots % 16], s["k"].dtype) for x in held] + q


def _plain_attention(s):
    q, cache, lens, cu = s["q"], s["cache"], s["kv_lens"].long(), s["cu_q"].long()
    Hq, D = q.shape[1:]
    Hkv = cache.shape[1]
    B, maxq, maxkv, G = len(lens), s["max_q"], s["max_kv"], Hq // Hkv
    # [B, pages, Hkv, blocks, 16, D] -> [B, Hkv, kv, D]
    k, v = (x.movedim(2, 1).reshape(B, Hkv, -1, D) for x in _blocks(cache[s["page_table"].long()])[:2])
    nq = cu[1:] - cu[:-1]
    i = torch.arange(maxq, device=q.device)
    rows = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)   # [B, maxq]
    x = q[rows].float().reshape(B, maxq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * maxq, D)
    w = torch.matmul(x, k[:, :, :maxkv].transpose(-1, -2)).mul_(s["scale"]).view(B, Hkv, G, maxq, maxkv)
    j = torch.arange(maxkv, device=q.device)
    at = (lens - nq)[:, None] + i                          # each query's position
    hide = (j >= lens[:, None])[:, None, :]
    if s["causal"]:
        hide = hide | (j > at[..., None])
    if s["window"]:
        hide = hide | (j <= at[..., None] - s["window"])
    w.masked_fill_(hide[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top > -math.inf, top, 0)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(B, Hkv, G * maxq, maxkv), v[:, :, :maxkv]).view(B, Hkv, G, maxq, D)
    o = o / torch.where(total > 0, total, 1)
    lse = (top + total.log())[..., 0]
    seq = torch.repeat_interleave(torch.arange(B, device=q.device), nq, output_size=q.shape[0])
    tok = torch.arange(q.shape[0], device=q.device) - cu[seq]
    return [_round(o.permute(0, 3, 1, 2, 4).reshape(B, maxq, Hq, D)[seq, tok], q.dtype),
            lse.permute(0, 3, 1, 2).reshape(B, maxq, Hq)[seq, tok]]


# ------------------------------------------------------------------ inputs

def _kv(gen, T, Hkv, D, dtype):
    """Keys, some of whose channels are large and off zero as rotated keys' are, and values; tokens
    of several sizes."""
    wide = torch.randn((Hkv, D), generator=gen, device="cuda").mul_(0.5).exp_()
    mean = torch.randn((Hkv, D), generator=gen, device="cuda").mul_(0.5)
    size = torch.randn((2, T, 1, 1), generator=gen, device="cuda").mul_(0.3).exp_()
    k = torch.randn((T, Hkv, D), generator=gen, device="cuda").mul_(wide).add_(mean).mul_(size[0])
    v = torch.randn((T, Hkv, D), generator=gen, device="cuda").mul_(size[1])
    return k.to(dtype), v.to(dtype)


def _rows_of(case, gen, per):
    """Keys and values of every token of every page of a case's sequences."""
    return _kv(gen, case["B"] * per * case["page"], case["Hkv"], case["D"], DTYPES[case["dtype"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    dtype, op = DTYPES[case["dtype"]], case["op"]
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")   # noqa: E731
    if op == "norm":
        T, H, K = case["T"], case["H"], case["K"]
        # (heads: the middle of wider rows, as a projection of queries, keys and values leaves them)
        x = randn(T, H + 2, K)[:, 1:H + 1].to(dtype) if H > 1 else randn(T, K).to(dtype)
        weight = (1 + 0.2 * randn(K)).to(dtype)
        s = {"op": op, "group": case["group"], "x": x, "weight": weight, "residual": None, "total": None,
             "out": torch.empty_like(x, dtype=dtype if case["group"] < 0 else E4M3, memory_format=torch.contiguous_format)}
        if case["residual"]:   # large in a few channels, as a residual stream is
            wide = torch.where(randn(K) > 2.5, 30.0, 1.0)
            s["residual"] = (randn(T, K) * wide * 3).to(dtype)
            s["total"] = torch.empty_like(s["residual"])
        if case["group"] >= 0:
            s["scales"] = torch.empty((T, K // (case["group"] or K)), device="cuda")
        return s
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if op == "rope":
        T = case["T"]
        scaling, magnitude = _scaling(case)
        qkv = randn(T, Hq + 2 * Hkv, D).to(dtype)   # a projection's rows
        if T <= 64:   # a sequence each
            positions = torch.randint(0, 100000, (T,), generator=gen, device="cuda") + case["at"]
        else:
            positions = case["at"] + torch.arange(T, device="cuda")
        q, k = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv]
        return {"op": op, "q": q, "k": k, "positions": positions.int(), "rot": case["rot"], "interleaved": case["interleaved"],
                "scaling": scaling, "magnitude": magnitude, "freq": _frequencies(case["rot"], scaling),
                "q_out": torch.empty((T, Hq, D), dtype=dtype, device="cuda"),
                "k_out": torch.empty((T, Hkv, D), dtype=dtype, device="cuda")}
    nq, lens = _lengths(case)
    B, page, maxkv = case["B"], case["page"], max(lens)
    per = -(-maxkv // page)
    table = torch.randperm(B * per, generator=gen, device="cuda").view(B, per)
    k, v = _rows_of(case, gen, per)
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0)
    n, length = torch.tensor(nq, device="cuda"), torch.tensor(lens, device="cuda")
    j = torch.arange(per * page, device="cuda")
    there = j < (length - n if op == "roundtrip" else length)[:, None]   # tokens the cache has
    blocks = [torch.where(there.view(-1, 1, 1), x, 0).float().view(B, per, page // 16, 16, Hkv, D).movedim(-2, 2) for x in (k, v)]
    cache = torch.zeros((B * per, Hkv, page // 16, 32 * D + 16), dtype=torch.uint8, device="cuda")
    cache[table] = _pack(*blocks)
    s = {"op": op, "cache": cache, "page_table": table.int(), "cu_q": cu.int(), "kv_lens": length.int(), "max_q": max(nq)}
    q = randn(sum(nq), Hq, D).to(dtype)
    if op == "attention":
        return {**s, "q": q, "max_kv": maxkv, "scale": D ** -0.5, "causal": case["causal"], "window": case["window"],
                "out": torch.empty_like(q), "lse": torch.empty(q.shape[:2], device="cuda")}
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), n)
    positions = torch.arange(sum(nq), device="cuda") - cu[seq] + (length - n)[seq]
    slots = table[seq, positions // page] * page + positions % page
    at = seq * per * page + positions
    rot = case["rot"]
    return {**s, "k": k[at], "v": v[at], "q": q if rot else None, "q_out": torch.empty_like(q) if rot else None,
            "positions": positions, "slots": slots.int(), "rot": rot, "interleaved": case["interleaved"],
            "scaling": _scaling(case)[0], "magnitude": 1.0, "freq": _frequencies(rot, _scaling(case)[0]) if rot else None,
            "k_out": torch.empty_like(k[at]), "v_out": torch.empty_like(v[at])}


def _handle(s):
    """The library's handle of the case's rotation, kept between calls as a program does."""
    if "rope" not in s:
        kind, factor, length, slow, fast = s["scaling"]
        s["rope"] = _package().Rope(s["rot"], base=BASE, interleaved=s["interleaved"], scaling=kind, factor=factor,
                                    original_length=length, slow=slow, fast=fast, magnitude=s["magnitude"])
    return s["rope"]


def run(state):
    s = state
    if not own:
        if s["op"] == "norm":
            return _plain_norm(s)
        if s["op"] == "rope":
            return [_round(_rotate(s[n], s["positions"], s["freq"], s["magnitude"], s["interleaved"]), s[n].dtype) for n in ("q", "k")]
        return _plain_roundtrip(s) if s["op"] == "roundtrip" else _plain_attention(s)
    pkg = _package()
    if s["op"] == "norm":
        sums = {"residual": s["residual"], "residual_out": s["total"]}
        total = [] if s["total"] is None else [s["total"]]
        if s["group"] < 0:
            return [pkg.rms_norm(s["x"], s["weight"], EPS, out=s["out"], **sums)] + total
        return [*pkg.rms_norm_8bit(s["x"], s["weight"], EPS, group=s["group"], out=s["out"], scales=s["scales"], **sums)] + total
    if s["op"] == "rope":
        pkg.rope(s["q"], s["positions"], _handle(s), k=s["k"], q_out=s["q_out"], k_out=s["k_out"])
        return [s["q_out"], s["k_out"]]
    if s["op"] == "roundtrip":
        rotation = {} if s["freq"] is None else {"rope": _handle(s), "q": s["q"], "q_out": s["q_out"]}
        pkg.kv8_write(s["k"], s["v"], s["cache"], s["page_table"], s["kv_lens"], cu_q=s["cu_q"], max_q_len=s["max_q"], **rotation)
        pkg.kv8_read(s["cache"], s["slots"], k_out=s["k_out"], v_out=s["v_out"])
        return [s["k_out"], s["v_out"]] + ([s["q_out"]] if rotation else [])
    if "workspace" not in s:   # kept between calls, as a serving program does
        s["workspace"] = pkg.kv8_attention_workspace(s["q"], s["cache"], len(s["kv_lens"]), s["max_q"], s["max_kv"])
    pkg.kv8_attention(s["q"], s["cache"], s["page_table"], s["kv_lens"], cu_q=s["cu_q"], max_q_len=s["max_q"],
                      max_kv_len=s["max_kv"], scale=s["scale"], causal=s["causal"], window=s["window"], out=s["out"],
                      lse=s["lse"], workspace=s["workspace"])
    return [s["out"], s["lse"]]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    if op == "norm":
        n = case["T"] * case["H"] * case["K"]
        out = 2.0 if case["group"] < 0 else 1.0 + 4.0 / (case["group"] or case["K"])
        return {"bytes": n * (2 + (4 if case["residual"] else 0) + out) + 2.0 * case["K"], "flops": 0.0}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if op == "rope":
        return {"bytes": case["T"] * ((Hq + Hkv) * D * 4.0 + 4) + case["rot"] * 4, "flops": 0.0}
    nq, lens = _lengths(case)
    row = Hkv * (2 * D + 1)   # a token's keys and values in 8 bits, with its part of the scales
    if op == "roundtrip":   # in 16 bits to 8 and back: what is read back was just written
        return {"bytes": float(sum(nq)) * (row + 2 * 2 * Hkv * D * 2 + (4 * Hq * D if case["rot"] else 0) + 4), "flops": 0.0}
    seen = reads = 0
    for n, length in zip(nq, lens):
        first = length - n
        lo = max(0, first - case["window"] + 1) if case["window"] else 0
        reads += length - lo
        for p in range(first, length):
            top = p + 1 if case["causal"] else length
            seen += top - (max(0, p - case["window"] + 1) if case["window"] else 0)
    b = reads * row + sum(nq) * Hq * (2 * 2 * D + 4)
    return {"bytes": float(b), "flops": 4.0 * seen * Hq * D}


# ------------------------------------------------------------------ the same in 64 bits

def _e4m3(x):
    """x (float64) at the nearest e4m3 value, ties to even; 448 at most."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _held(x, least=None):
    """What a cache holds of blocks x [..., 16, D]: e4m3 under a power of two, of `least` at least."""
    e = torch.ceil(torch.log2(x.abs().amax((-2, -1), keepdim=True) / 448)).clamp(min=-60)
    s = torch.exp2(e) if least is None else torch.maximum(torch.exp2(e), least)
    return _e4m3(x / s) * s


def _turned(x, positions, case):
    """Rows x [T, H, D] in 64 bits with each pair, as a complex number, times magnitude e^(i w)."""
    rot, D = case["rot"], case["D"]
    (kind, factor, length, slow, fast), magnitude = _scaling(case)
    angle = []
    for i in range(rot // 2):
        base = BASE * factor ** (rot / (rot - 2)) if kind == "base" and rot > 2 else BASE
        f = math.exp(-2 * i / rot * math.log(base))
        if kind == "linear":
            f /= factor
        elif kind == "ramp":
            turns = length * f / (2 * math.pi)
            part = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
            f = part * f + (1 - part) * f / factor
        angle.append(f)
    w = torch.outer(positions.double(), torch.tensor(angle, dtype=torch.float64, device="cuda"))
    turn = torch.polar(torch.full_like(w, magnitude), w)[:, None]
    x, y = x.double(), x.double().clone()
    half = [list(range(0, rot, 2)), list(range(1, rot, 2))] if case["interleaved"] else [list(range(rot // 2)), list(range(rot // 2, rot))]
    z = torch.complex(x[..., half[0]], x[..., half[1]]) * turn
    y[..., half[0]], y[..., half[1]] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        norm = torch.linalg.vector_norm(h, dim=-1, keepdim=True) / math.sqrt(case["K"])
        y = s["weight"].double() * h / torch.sqrt(norm ** 2 + EPS)
        total = [] if s["residual"] is None else [h]
        if case["group"] < 0:
            return [y] + total
        y = y.view(case["T"], -1, case["group"] or case["K"])
        scale = torch.linalg.vector_norm(y, ord=math.inf, dim=-1) / 448
        return [_e4m3(y / scale[..., None]).reshape(case["T"], case["K"]), scale] + total
    if op == "rope":
        return [_turned(s["q"], s["positions"], case), _turned(s["k"], s["positions"], case)]
    # the rows that the cache was filled from, in the order of the generator
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    per = s["page_table"].shape[1]
    torch.randperm(case["B"] * per, generator=gen, device="cuda")
    B, page, Hkv, D = case["B"], case["page"], case["Hkv"], case["D"]
    k, v = (x.view(B, per * page, Hkv, D) for x in _rows_of(case, gen, per))
    nq, lens = _lengths(case)
    rows = lambda x, b, n: x[b, :n].double().transpose(0, 1)   # noqa: E731  [Hkv, n, D]

    def blocks(x):   # [Hkv, n, D] -> [Hkv, blocks, 16, D], zeros behind
        return torch.nn.functional.pad(x, (0, 0, 0, -x.shape[1] % 16)).unflatten(1, (-1, 16))

    if op == "roundtrip":
        out_k, out_v = [], []
        for b, (n, length) in enumerate(zip(nq, lens)):
            first = length - n
            lo = first // 16 * 16
            for x, out in ((k, out_k), (v, out_v)):
                x = rows(x, b, length)
                old = x[:, lo:first]
                least = torch.exp2(torch.ceil(torch.log2(old.abs().amax((1, 2)) / 448)).clamp(min=-60)) if first > lo else None
                new = x[:, first:]
                if out is out_k and case["rot"]:
                    new = _turned(new.transpose(0, 1), torch.arange(first, length, device="cuda"), case).transpose(0, 1)
                if first > lo:
                    old = _held(old[:, None], least[:, None, None, None])[:, 0]
                y = blocks(torch.cat((old, new), 1))
                floor = torch.full((Hkv, y.shape[1], 1, 1), 2.0 ** -60, dtype=torch.float64, device="cuda")
                if first > lo:
                    floor[:, 0, 0, 0] = least
                out.append(_held(y, floor).flatten(1, 2)[:, first - lo:first - lo + n].transpose(0, 1))
        q = [_turned(s["q"], s["positions"], case)] if case["rot"] else []
        return [torch.cat(out_k), torch.cat(out_v)] + q
    G = case["Hq"] // Hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, length) in enumerate(zip(nq, lens)):
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        see = torch.ones((n, length), dtype=torch.bool, device="cuda")
        if case["causal"]:
            see &= key <= pos
        if case["window"]:
            see &= key > pos - case["window"]
        kb, vb = (_held(blocks(rows(x, b, length))).flatten(1, 2)[:, :length] for x in (k, v))
        for h in range(Hkv):
            for g in range(h * G, (h + 1) * G):
                score = (s["q"][at:at + n, g].double() @ kb[h].t()) / math.sqrt(D)
                score[~see] = -math.inf
                lse[at:at + n, g] = torch.logsumexp(score, dim=1)
                out[at:at + n, g] = torch.softmax(score, dim=1) @ vb[h]
        at += n
    return [out, lse]
