"""The operators on a key/value cache held in 4 bits: writing it, reading it back, and attention
over it, from one token of one sequence to prompts and long contexts.

`run` computes them in plain torch operations where `own` is false, and through the library where
it is true, on the same cache bytes. A cache is a uint8 tensor [pages, kv heads, page_size / 16,
16 D + 128]: blocks of 16 tokens of one head, each with its keys, its values and one parameter
word a token for either:

  keys     [16 tokens][D / 2] bytes, dimension 2 b in the low nibble of byte b
  values   [4 quads][16 columns][2 pairs][D / 64][2 tokens][2] bytes: token 4 quad + 2 pair + i,
           dimensions column D / 16 + 4 h + (0..3), lowest nibble first
  params   [2: keys, values][16 tokens] 32-bit words: scale (bits 0..15, the element type),
           zero point (bits 16..31); a nibble n stands for (n - zero) scale

A row of D values is quantised over the range that it and 0 span: scale = (max - min) / 15, rounded
to fp32 and then to the element type; zero = rint(-min / scale); n = rint(x / scale) + zero,
clamped to 0..15; a scale of 0 gives zeros throughout.

A case is a dict of plain values: `op` is "roundtrip" (rows are written and read back), "read" or
"attention" (`q` new tokens of each of `B` sequences, whose lengths with them are at most `kv`).
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

def _rows(name, op, T, Hkv, D, page, dtype, padded=False):
    c = {"op": op, "T": T, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "padded": padded}
    return {"name": name, **c} if name else c


def _attention(name, B, q, kv, Hq, Hkv, D, page, dtype, ragged=False, causal=True, window=0):
    c = {"op": "attention", "B": B, "q": q, "kv": kv, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
         "dtype": dtype, "ragged": ragged, "causal": causal, "window": window}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the keys and values of one decode step of sixteen sequences, each into a page of its own
        _rows("roundtrip_decode_t16", "roundtrip", 16, 8, 128, 16, "f16"),
        # those of a short chunk with padding behind it (slots of -1), small heads
        _rows("roundtrip_padded_t333", "roundtrip", 333, 12, 64, 32, "bf16", padded=True),
        # those of a prompt
        _rows("roundtrip_prompt_t8192", "roundtrip", 8192, 8, 128, 64, "bf16"),
        # a cached prefix of some length back to 16 bits, for a program's own attention
        _rows("read_prefix_t1000", "read", 1000, 8, 128, 16, "f16"),
        # a long one
        _rows("read_prefix_t65536", "read", 65536, 8, 128, 64, "bf16"),
        # one decode step of one sequence that has just begun: latency
        _attention("decode_b1_kv500", 1, 1, 500, 32, 8, 128, 16, "f16"),
        # one decode step of a serving batch, sequences of all lengths
        _attention("decode_b48_kv4096", 48, 1, 4096, 32, 8, 128, 16, "bf16", ragged=True),
        # one decode step over long documents
        _attention("decode_b4_kv65536", 4, 1, 65536, 32, 8, 128, 64, "f16"),
        # five drafted tokens of each of eight sequences verified at once, sliding window, one
        # wide head of keys and values to eight of queries
        _attention("verify_b8_q5_kv6000", 8, 5, 6000, 16, 2, 256, 32, "f16", ragged=True, window=4096),
        # a batch of prompts of all lengths, as many heads of keys as of queries
        _attention("prompts_b7_q1500", 7, 1500, 1500, 16, 16, 64, 16, "f16", ragged=True),
        # one prompt of 2048 tokens
        _attention("prompt_q2048", 1, 2048, 2048, 32, 8, 128, 64, "f16"),
        # a prefill chunk behind a long context
        _attention("chunk_q1024_kv32768", 1, 1024, 32768, 32, 8, 128, 64, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["roundtrip", "read", "decode", "decode", "verify", "prompt", "chunk"])
    dtype, page = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
    if kind in ("roundtrip", "read"):
        Hkv, D = rng.choice([(1, 256), (2, 128), (8, 128), (8, 128), (12, 64), (4, 192)])
        most = 8192 if kind == "roundtrip" else 65536
        return _rows(None, kind, _log_int(rng, 1, most * 1024 // max(1024, Hkv * D)), Hkv, D, page, dtype,
                     padded=rng.random() < 0.3)
    Hq, Hkv, D = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (28, 4, 128), (16, 16, 64),
                             (12, 12, 64), (16, 2, 256), (24, 1, 128), (12, 4, 192)])
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


# ------------------------------------------------------------------ the plain forms

def _quantise(x):
    """Rows x [..., D] as (nibbles uint8, scale in x's type, zero point int32)."""
    d = x.double()
    lo, hi = d.amin(-1).clamp(max=0), d.amax(-1).clamp(min=0)
    scale = ((hi - lo) / 15).float().to(x.dtype)
    s = scale.double()
    inv = torch.where(s > 0, s, torch.ones_like(s))
    zero = (torch.round(-lo / inv).clamp(0, 15) * (s > 0)).int()
    n = (torch.round(d / inv[..., None]) + zero[..., None]).clamp(0, 15)
    return (n * (s > 0)[..., None]).to(torch.uint8), scale, zero


def _bytes(n):
    """Nibbles [..., m] as bytes [..., m / 2], lower dimension in the lower nibble."""
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _nibbles(b):
    """Bytes [..., m] as nibbles [..., 2 m]."""
    return torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)


def _words(scale, zero):
    return ((zero << 16) | (scale.view(torch.int16).int() & 0xFFFF)).contiguous()


def _empty_cache(pages, Hkv, D, page):
    return torch.zeros((pages, Hkv, page // 16, 16 * D + 128), dtype=torch.uint8, device="cuda")


def _places(cache, slots):
    """(page, head, block, token), then the bytes of a row's keys and of its values in their block,
    then the words of their parameters, of rows [T, Hkv, ...] in these slots."""
    page, Hkv, D = cache.shape[2] * 16, cache.shape[1], (cache.shape[3] - 128) // 16
    slots = slots.long()[:, None, None]
    head = torch.arange(Hkv, device=cache.device)[None, :, None]
    tok, at = slots % 16, torch.arange(D // 2, device=cache.device)
    col, h = at // (D // 32), at % (D // 32) // 2
    value = 8 * D + tok // 4 * (2 * D) + col * (D // 8) + tok // 2 % 2 * (D // 16) + h * 4 + tok % 2 * 2 + at % 2
    return (slots // page, head, slots % page // 16), (tok * (D // 2) + at, value), (4 * D + tok, 4 * D + 16 + tok)


def _store(cache, k, v, slots):
    """Rows k, v [T, Hkv, D] quantised into the slots of the cache; negative slots are passed over."""
    keep = slots >= 0
    block, places, words = _places(cache, slots[keep])
    for x, place, word in zip((k, v), places, words):
        n, scale, zero = _quantise(x[keep])
        cache[(*block, place)] = _bytes(n)
        cache.view(torch.int32)[(*block, word)] = _words(scale, zero)[..., None]


def _params(words, dtype):
    """(scale, zero) in fp32 from parameter words."""
    return ((words & 0xFFFF).to(torch.int16).view(dtype).float(), (words >> 16).float())


def _blocks(blocks, dtype):
    """Keys and values [..., 16, D] in fp32 of whole blocks [..., 16 D + 128]."""
    D = (blocks.shape[-1] - 128) // 16
    lead = blocks.shape[:-1]
    words = blocks[..., 16 * D:].contiguous().view(torch.int32)
    nk = _nibbles(blocks[..., :8 * D].reshape(*lead, 16, D // 2))
    nv = blocks[..., 8 * D:16 * D].reshape(*lead, 4, 16, 2, D // 64, 2, 2)
    nv = _nibbles(nv.movedim((-4, -2), (-5, -4)).reshape(*lead, 16, D // 2))
    out = []
    for n, w in ((nk, words[..., :16]), (nv, words[..., 16:])):
        s, z = _params(w, dtype)
        out.append((n.float() - z[..., None]) * s[..., None])
    return out


def _round(x, dtype):
    """x in the element type, saturated to its largest finite value."""
    most = torch.finfo(dtype).max
    return x.clamp(-most, most).to(dtype)


def _plain_read(cache, slots, dtype):
    block, places, words = _places(cache, slots.clamp(min=0))
    out = []
    for place, word in zip(places, words):
        scale, zero = _params(cache.view(torch.int32)[(*block, word)], dtype)
        x = (_nibbles(cache[(*block, place)]).float() - zero) * scale
        out.append(torch.where((slots >= 0)[:, None, None], _round(x, dtype), 0))
    return out


def _plain_attention(s):
    q, cache, lens, cu = s["q"], s["cache"], s["kv_lens"].long(), s["cu_q"].long()
    Hq, D = q.shape[1:]
    Hkv, page = cache.shape[1], cache.shape[2] * 16
    B, maxq, maxkv, G = len(lens), s["max_q"], s["max_kv"], Hq // cache.shape[1]
    # [B, pages, Hkv, blocks, 16, D] -> [B, Hkv, kv, D]
    k, v = (x.movedim(2, 1).reshape(B, Hkv, -1, D) for x in _blocks(cache[s["page_table"].long()], q.dtype))
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
    """Keys, some of whose channels are large and off zero as rotated keys' are, and values."""
    wide = torch.randn((Hkv, D), generator=gen, device="cuda").mul_(0.5).exp_()
    mean = torch.randn((Hkv, D), generator=gen, device="cuda").mul_(0.5)
    k = torch.randn((T, Hkv, D), generator=gen, device="cuda").mul_(wide).add_(mean)
    v = torch.randn((T, Hkv, D), generator=gen, device="cuda")
    return k.to(dtype), v.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    Hkv, D, page, dtype = case["Hkv"], case["D"], case["page"], DTYPES[case["dtype"]]
    if case["op"] != "attention":
        # each row at the next token of a sequence's pages, or (few rows) each in a page of its own
        T = case["T"]
        pages = T if T <= 64 else -(-T // page)
        cache = _empty_cache(pages + 1, Hkv, D, page)
        perm = torch.randperm(pages + 1, generator=gen, device="cuda")
        t = torch.arange(T, device="cuda")
        slots = perm[t] * page + t * 7 % page if T <= 64 else perm[t // page] * page + t % page
        k, v = _kv(gen, T, Hkv, D, dtype)
        if case["op"] == "read":
            _store(cache, k, v, slots)
        if case["padded"]:
            slots[T - T // 8:] = -1
        s = {"op": case["op"], "cache": cache, "slots": slots.int(), "dtype": dtype,
             "k_out": torch.zeros_like(k), "v_out": torch.zeros_like(v)}
        return {**s, "k": k, "v": v} if case["op"] == "roundtrip" else s
    nq, lens = _lengths(case)
    B, maxkv = case["B"], max(lens)
    per = -(-maxkv // page)
    cache = _empty_cache(B * per, Hkv, D, page)
    table = torch.randperm(B * per, generator=gen, device="cuda").view(B, per)
    t = torch.arange(per * page, device="cuda")
    slots = (table[:, t // page] * page + t % page).flatten()
    k, v = _kv(gen, B * per * page, Hkv, D, dtype)
    _store(cache, k, v, slots)
    q = torch.randn((sum(nq), case["Hq"], D), generator=gen, device="cuda").to(dtype)
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0)
    return {"op": "attention", "q": q, "cache": cache, "page_table": table.int(), "cu_q": cu.int(),
            "kv_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "max_q": max(nq),
            "max_kv": maxkv, "scale": D ** -0.5, "causal": case["causal"], "window": case["window"],
            "out": torch.empty_like(q), "lse": torch.empty(q.shape[:2], device="cuda")}


def run(state):
    s = state
    if s["op"] == "attention":
        if own:
            pkg = _package()
            if "workspace" not in s:   # kept between calls, as a serving program does
                s["workspace"] = pkg.kv4_attention_workspace(s["q"], s["cache"], len(s["kv_lens"]),
                                                             s["max_q"], s["max_kv"])
            pkg.kv4_attention(s["q"], s["cache"], s["page_table"], s["kv_lens"], cu_q=s["cu_q"],
                              max_q_len=s["max_q"], max_kv_len=s["max_kv"], scale=s["scale"],
                              causal=s["causal"], window=s["window"], out=s["out"], lse=s["lse"],
                              workspace=s["workspace"])
            return [s["out"], s["lse"]]
        return _plain_attention(s)
    if own:
        pkg = _package()
        if s["op"] == "roundtrip":
            pkg.kv4_write(s["k"], s["v"], s["cache"], s["slots"])
        pkg.kv4_read(s["cache"], s["slots"], k_out=s["k_out"], v_out=s["v_out"])
        return [s["k_out"], s["v_out"]]
    if s["op"] == "roundtrip":
        _store(s["cache"], s["k"], s["v"], s["slots"])
    return _plain_read(s["cache"], s["slots"], s["dtype"])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    Hkv, D = case["Hkv"], case["D"]
    row = 2 * Hkv * (D // 2 + 4)   # a token's keys and values in 4 bits, with their parameters
    if case["op"] != "attention":
        T = case["T"] - (case["T"] // 8 if case["padded"] else 0)
        wide = T * 2 * Hkv * D * 2
        b = T * row + wide + 4 * case["T"]
        if case["op"] == "roundtrip":   # in 16 bits to 4 and back: what is read back was just written
            b += wide
        return {"bytes": float(b), "flops": 0.0}
    nq, lens = _lengths(case)
    seen = reads = 0
    for n, length in zip(nq, lens):
        first = length - n
        lo = max(0, first - case["window"] + 1) if case["window"] else 0
        reads += length - lo
        for p in range(first, length):
            top = p + 1 if case["causal"] else length
            seen += top - (max(0, p - case["window"] + 1) if case["window"] else 0)
    b = reads * row + sum(nq) * case["Hq"] * (2 * 2 * D + 4)
    return {"bytes": float(b), "flops": 4.0 * seen * case["Hq"] * D}


# ------------------------------------------------------------------ the same in 64 bits

def _exact_values(x):
    """What the cache holds of rows x: (n - zero) scale in 64 bits, from the definition."""
    most = torch.maximum(x.double().max(dim=-1, keepdim=True).values, torch.zeros((), device=x.device))
    least = torch.minimum(x.double().min(dim=-1, keepdim=True).values, torch.zeros((), device=x.device))
    step = ((most - least) / 15.0).to(torch.float32).to(x.dtype).to(torch.float64)
    units = x.double() / step
    zero = torch.round(0.0 - least / step)
    level = torch.round(units).add_(zero).clamp_(0, 15)
    return torch.nan_to_num(level.sub_(zero).mul_(step), nan=0.0)


def exact(case, seed):
    s = prepare(case, seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "roundtrip":
        live = (s["slots"] >= 0).double()[:, None, None]
        return [_exact_values(s[n]) * live for n in ("k", "v")]
    # the rows that the cache was filled from, in the order of the generator
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if case["op"] == "read":
        torch.randperm(s["cache"].shape[0], generator=gen, device="cuda")
        live = (s["slots"] >= 0).double()[:, None, None]
        return [_exact_values(x) * live for x in _kv(gen, case["T"], Hkv, D, dtype)]
    nq, lens = _lengths(case)
    per = s["page_table"].shape[1]
    torch.randperm(case["B"] * per, generator=gen, device="cuda")
    k, v = (x.view(case["B"], per * page, Hkv, D) for x in _kv(gen, case["B"] * per * page, Hkv, D, dtype))
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
        for h in range(Hkv):
            kh, vh = _exact_values(k[b, :length, h]), _exact_values(v[b, :length, h])
            for g in range(h * G, (h + 1) * G):
                score = (s["q"][at:at + n, g].double() @ kh.t()) / math.sqrt(D)
                score[~see] = -math.inf
                lse[at:at + n, g] = torch.logsumexp(score, dim=1)
                out[at:at + n, g] = torch.softmax(score, dim=1) @ vh
        at += n
    return [out, lse]
