"""The 4-bit key/value cache on the GPU: rows in and out bit for bit, attention against 64 bits."""
import numpy as np
import pytest
import torch

import kv4_plain as plain
from helpers import pkg

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return pkg()


def rows(gen, T, H, D, dtype, kind="normal"):
    x = torch.randn((T, H, D), generator=gen)
    if kind == "wide":          # a few channels far from zero
        x = x * torch.randn((1, H, D), generator=gen).mul(1.5).exp() + torch.randn((1, H, D), generator=gen)
    elif kind == "ties":        # multiples of half a step of a row spanning 15 steps: every other one a tie
        x = torch.randint(0, 31, (T, H, D), generator=gen).float() / 2
        x[..., 0], x[..., 1] = 0, 15
        x = x * 2.0 ** torch.randint(-6, 7, (T, H, 1), generator=gen)
    elif kind == "far":         # the type's ends, and values next to zero
        e = torch.randint(-24 if dtype == F16 else -133, 16 if dtype == F16 else 127, (T, H, 1), generator=gen)
        x = x.double().mul(2.0 ** e.double())
    elif kind == "constant":    # one value in the row: all positive, all negative or zero
        x = x[..., :1].expand(T, H, D).clone()
        x[::3] = 0
    most = torch.finfo(dtype).max
    return x.double().clamp(-most, most).float().to(dtype)


def same(a, b):
    """Bit for bit, any NaN equal to any."""
    a, b = a.cpu(), b.cpu()
    nan = torch.isnan(a) & torch.isnan(b)
    return bool(((a.view(torch.int16) == b.view(torch.int16)) | nan | ((a == 0) & (b == 0))).all())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("kind,T,H,page", [("normal", 1, 1, 16), ("wide", 37, 3, 32), ("ties", 33, 2, 64),
                                           ("far", 50, 2, 16), ("constant", 18, 1, 128)])
def test_rows_in_and_out(dtype, D, kind, T, H, page):
    P = need_gpu()
    gen = torch.Generator().manual_seed(T * 1000 + D)
    k, v = rows(gen, T, H, D, dtype, kind), rows(gen, T, H, D, dtype, kind)
    pages = T // page + 3
    slots = torch.randperm(pages * page, generator=gen)[:T].int()
    if T > 4:
        slots[2], slots[4] = -1, pages * page    # passed over
    cache = P.kv4_cache(pages, H, D, page)
    cache.random_(0, 256, generator=torch.Generator("cuda").manual_seed(1))
    want = cache.cpu().numpy().copy()
    got = P.kv4_write(k.cuda(), v.cuda(), cache, slots.cuda())
    assert got is cache
    held = []
    for which, x in enumerate((k, v)):
        n, s, z, val = plain.quantise(x)
        held.append(val)
        for t in range(T):
            for h in range(H):
                if 0 <= slots[t] < pages * page:
                    plain.pack(want, int(slots[t]), h, which, n[t, h], s[t, h], z[t, h])
    diff = np.argwhere(cache.cpu().numpy() != want)
    assert len(diff) == 0, diff[:8]
    fill = torch.full((2, T, H, D), 7.0, dtype=dtype, device="cuda")
    ko, vo = P.kv4_read(cache, slots.cuda(), k_out=fill[0], v_out=fill[1])
    for val, o in zip(held, (ko, vo)):
        exp = plain.rounded(val, dtype)
        if T > 4:
            exp[2] = exp[4] = 7.0
        assert same(o, exp)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_rows_not_finite(dtype):
    """A row with an infinity or NaN is NaN throughout, its neighbours are not."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(5)
    k, v = rows(gen, 6, 2, 128, dtype), rows(gen, 6, 2, 128, dtype)
    k[1, 0, 5], k[2, 1, 127], v[3, 0, 0], v[3, 1, 64] = float("nan"), float("inf"), -float("inf"), float("nan")
    cache = P.kv4_cache(1, 2, 128, 16)
    slots = torch.arange(6, dtype=torch.int32, device="cuda")
    P.kv4_write(k.cuda(), v.cuda(), cache, slots)
    for x, o in zip((k, v), P.kv4_read(cache, slots, dtype)):
        assert same(o, plain.rounded(plain.quantise(x)[3], dtype))


def test_rows_strided_repeated_and_rewritten():
    """Slices of a fused projection, head-major rows, one row read into two places, a slot written twice."""
    P = need_gpu()
    T, H, D = 21, 4, 128
    gen = torch.Generator().manual_seed(8)
    qkv = torch.randn((T, 3 * H, D), generator=gen).half().cuda()
    k, v = qkv[:, H:2 * H], qkv[:, 2 * H:].transpose(0, 1).contiguous().transpose(0, 1)
    cache = P.kv4_cache(2, H, D, 32)
    slots = torch.arange(T, dtype=torch.int32, device="cuda") * 3
    P.kv4_write(-k, -v, cache, slots)
    P.kv4_write(k, v, cache, slots)
    twice = torch.cat((slots, slots[:5]))
    big = torch.zeros((H, T + 5, 2 * D), dtype=F16, device="cuda")
    ko, vo = big[..., :D].transpose(0, 1), big[..., D:].transpose(0, 1)
    P.kv4_read(cache, twice, k_out=ko, v_out=vo)
    for x, o in ((k, ko), (v, vo)):
        exp = plain.rounded(plain.quantise(x.cpu())[3], F16)
        assert same(o[:T].contiguous(), exp) and same(o[T:].contiguous(), exp[:5])


# ------------------------------------------------------------------ attention

class Batch:
    """Sequences in a cache of shuffled pages, with queries, on the GPU and in 64 bits."""

    def __init__(self, P, nq, lens, Hq, Hkv, D, page, dtype, seed=0, kscale=1.0, vscale=1.0, spare=1):
        gen = torch.Generator().manual_seed(seed + 7 * D + Hq)
        self.nq, self.lens, self.dtype, self.D, self.Hq = nq, lens, dtype, D, Hq
        B, per = len(lens), max(1, -(-max(lens) // page)) + spare
        pages = B * per
        self.table = torch.randperm(pages, generator=gen).view(B, per).int()
        self.cache = P.kv4_cache(pages, Hkv, D, page)
        self.cache.random_(0, 256, generator=torch.Generator("cuda").manual_seed(3))   # what is not written: anything
        self.k, self.v = [], []
        for b, L in enumerate(lens):
            k = (rows(gen, L, Hkv, D, dtype, "wide").float() * kscale).to(dtype)
            v = (rows(gen, L, Hkv, D, dtype).float() * vscale).to(dtype)
            t = torch.arange(L)
            slots = (self.table[b, t // page] * page + t % page).int()
            if L:
                P.kv4_write(k.cuda(), v.cuda(), self.cache, slots.cuda())
            self.k.append(plain.quantise(k)[3] if L else np.zeros((0, Hkv, D)))
            self.v.append(plain.quantise(v)[3] if L else np.zeros((0, Hkv, D)))
        self.q = torch.randn((sum(nq), Hq, D), generator=gen).to(dtype)
        self.cu = torch.tensor([0] + nq).cumsum(0).int()

    def gpu(self, P, **over):
        T = len(self.q)
        a = dict(cu_q=self.cu.cuda(), max_q_len=max(1, max(self.nq)), max_kv_len=max(self.lens),
                 lse=torch.full((T, self.Hq), 5.0, device="cuda"))
        a.update(over)
        q = a.pop("q", None)
        out = P.kv4_attention(self.q.cuda() if q is None else q, self.cache, self.table.cuda(),
                              torch.tensor(self.lens, dtype=torch.int32, device="cuda"), **a)
        return out, a["lse"]

    def check(self, out, lse, causal=True, window=0, scale=None, seen=None, what=""):
        """Bounds: the weights p_j, rounded to fp16 (2^-11), times values; the logits, whose products
        (sum of |q k| at most `reach`) are summed in fp32 over D terms, an error in the exponent of p;
        sums over the keys in fp32; one rounding of the result. Weights below fp16's normal range move
        by half of 2^-24: they are p_j s_j 2^7 / r with r at most 4 times the largest scale s, so a key's
        share of the sum by 2^-25 2^-7 4 s |n - z| <= 2^-30 15 s <= 2^-29 max|v|, the sum of all p_j
        being 1 or more."""
        q = self.q.double().numpy()
        o, l, spread, reach, vtop = plain.attention(q, self.k, self.v, self.nq, self.lens, causal, window, scale, seen)
        keys = max(self.lens) + 8
        logit = (self.D + 8) * 2.0 ** -23 * (4 * reach + 1)
        eps = torch.finfo(self.dtype).eps / 2
        tiny = 2.0 ** -25 if self.dtype == F16 else 2.0 ** -134
        part = (2.0 ** -11 + 2 * logit + keys * 2.0 ** -23 + 2.0 ** -16)[..., None]
        tol = eps * np.abs(o) + part * (1 + eps) * 2 * spread + tiny + keys * 2.0 ** -29 * vtop[..., None]
        got = out.double().cpu().numpy()
        bad = ~(np.abs(got - o) <= tol)
        assert not bad.any(), (what, np.argwhere(bad)[:5], got[bad][:5], o[bad][:5], tol[bad][:5])
        gl = lse.double().cpu().numpy()
        empty = ~np.isfinite(l)
        assert (gl[empty] == -np.inf).all(), what
        lt = logit + keys * 2.0 ** -23 + 2.0 ** -22 * np.abs(np.where(empty, 0, l)) + 2.0 ** -20
        bad = ~empty & ~(np.abs(gl - np.where(empty, 0, l)) <= lt)
        assert not bad.any(), (what, np.argwhere(bad)[:5], gl[bad][:5], l[bad][:5], lt[bad][:5])


HEADS = [(4, 4, 64), (8, 2, 128), (6, 1, 192), (4, 1, 256), (24, 1, 64), (7, 1, 128), (40, 2, 128)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("lens,page", [([1], 16), ([0, 1, 15, 16, 17, 33], 16), ([257, 5, 64], 32), ([700, 1300], 128)])
def test_decode(dtype, Hq, Hkv, D, lens, page):
    P = need_gpu()
    b = Batch(P, [1] * len(lens), lens, Hq, Hkv, D, page, dtype)
    b.check(*b.gpu(P, cu_q=None))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,D", HEADS[:5])
@pytest.mark.parametrize("nq,lens,causal,window", [
    ([1, 3, 2], [1, 3, 70], True, 0),            # whole prompts and drafts
    ([17, 0, 40], [17, 9, 90], True, 0),         # a sequence without queries
    ([5, 9], [3, 4], True, 0),                   # more queries than keys: the first see nothing
    ([33, 70], [200, 70], True, 19),
    ([20, 3], [50, 0], False, 0),                # no keys at all
    ([66], [66], False, 7),
    ([130], [180], True, 300),
])
def test_several_queries(dtype, Hq, Hkv, D, nq, lens, causal, window):
    P = need_gpu()
    b = Batch(P, nq, lens, Hq, Hkv, D, 16, dtype)
    b.check(*b.gpu(P, causal=causal, window=window), causal=causal, window=window)
