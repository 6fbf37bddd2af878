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


def attention_path(P, T, B, Hq, Hkv, D, max_q, max_kv):
    """What kv4_attention runs: ("few", column tiles a wave, chunks a head at most, joined apart) or
    ("many", wave groups, chunks)."""
    import ctypes
    out = (ctypes.c_int32 * 4)()
    P.lib().w4a16_internal_kv4_path(T, B, Hq, Hkv, D, max_q, max_kv, out)
    return ("few", *out[1:]) if out[0] == 1 else ("many", *out[1:3])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,lens,Hq,Hkv,D,page,window,path", [
    # few columns: one and two column tiles a wave, one chunk a sequence and several, joined by the last
    # workgroup and by a kernel of their own, more sequences than a wave has lanes
    ([1] * 3, [100, 128, 7], 8, 2, 128, 16, 0, ("few", 1, 3, 0)),
    ([1] * 2, [1500, 900], 8, 8, 64, 32, 0, ("few", 1, 24, 0)),
    ([1], [3000], 4, 1, 128, 64, 0, ("few", 1, 24, 1)),
    ([1] * 5, [2100, 1, 850, 0, 1300], 24, 1, 128, 16, 0, ("few", 2, 85, 1)),
    ([5, 5, 3], [1100, 9, 1400], 16, 2, 64, 16, 300, ("few", 2, 36, 1)),
    ([5], [1000], 4, 1, 64, 16, 0, ("few", 2, 9, 0)),
    ([8, 2, 8], [1700, 800, 33], 8, 1, 256, 64, 0, ("few", 1, 42, 1)),
    ([4, 9], [900, 1000], 10, 2, 192, 32, 0, ("few", 1, 18, 1)),
    ([1] * 130, [(37 * i) % 331 + 600 * (i == 7) for i in range(130)], 2, 1, 64, 16, 0, ("few", 1, 910, 0)),
    ([1] * 300, [(53 * i) % 200 + 1100 * (i % 97 == 5) for i in range(300)], 2, 1, 64, 16, 0, ("few", 1, 1024, 0)),
    ([1] * 1100, [(29 * i) % 60 + 1000 * (i % 250 == 90) for i in range(1100)], 2, 2, 64, 16, 0, ("few", 1, 2560, 0)),
    # many: two groups of waves on a tile, one of them, keys in one chunk and in several
    ([300, 70], [300, 500], 2, 1, 128, 32, 0, ("many", 2, 1)),
    ([90], [2500], 4, 2, 64, 16, 0, ("many", 2, 5)),
    ([70, 66], [1500, 1030], 1, 1, 256, 64, 700, ("many", 1, 3)),
    ([65, 2], [600, 1200], 3, 3, 192, 16, 0, ("many", 1, 3)),
    ([129] * 172, [129 + i for i in range(172)], 3, 3, 64, 16, 33, ("many", 1, 1)),
])
def test_every_path(dtype, nq, lens, Hq, Hkv, D, page, window, path):
    P = need_gpu()
    assert attention_path(P, sum(nq), len(nq), Hq, Hkv, D, max(nq), max(lens)) == path
    b = Batch(P, nq, lens, Hq, Hkv, D, page, dtype)
    out, lse = b.gpu(P, window=window)
    b.check(out, lse, window=window)
    again, _ = b.gpu(P, window=window)
    assert torch.equal(out, again), "the same call twice"


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,lens,Hq,Hkv,D,window", [
    ([1, 1, 400, 1, 1], [300, 1, 420, 450, 64], 8, 2, 64, 0),                   # whole sequences beside one prompt
    ([1, 500, 16, 1, 0, 17, 2], [2300, 900, 700, 1, 40, 1100, 0], 8, 2, 128, 0),    # 16 queries of 4 heads: the most
    ([300, 1, 3, 32, 33], [2600, 1900, 1200, 800, 33], 4, 2, 256, 500),
    ([200] + [1] * 80, [900] + [(37 * i) % 800 + 1 for i in range(80)], 2, 2, 64, 0),
    ([1] * 150 + [300, 129, 1], [(31 * i) % 600 + 1 for i in range(150)] + [2100, 140, 9], 4, 1, 128, 0),
])
def test_single_tokens_beside_prompts(dtype, nq, lens, Hq, Hkv, D, window):
    """A batch most of whose sequences are far shorter than the longest runs on both kernels."""
    import ctypes
    P = need_gpu()
    path = (ctypes.c_int32 * 4)()
    P.lib().w4a16_internal_kv4_path(sum(nq), len(nq), Hq, Hkv, D, max(nq), max(lens), path)
    assert path[0] == 2 and path[3] == 64 // (Hq // Hkv)
    b = Batch(P, nq, lens, Hq, Hkv, D, 16, dtype)
    ws = P.kv4_attention_workspace(b.q.cuda(), b.cache, len(nq), max(nq), max(lens))
    first = None
    for _ in range(3):
        out, lse = b.gpu(P, window=window, workspace=ws)
        b.check(out, lse, window=window)
        first = out if first is None else first
        assert torch.equal(out, first) and int(ws[:P.KV4_COUNTER_BYTES].sum()) == 0


def test_long_sequence_and_workspace_of_many_calls():
    """70,000 keys; one workspace through calls of other shapes, back and forth."""
    P = need_gpu()
    a = Batch(P, [1, 1], [70000, 300], 8, 2, 64, 128, F16, seed=4)
    b = Batch(P, [40, 7], [600, 50], 8, 2, 64, 16, F16, seed=5)
    ws = P.kv4_attention_workspace(a.q.cuda(), a.cache, 2, 1, 70000)
    need = P.kv4_attention_workspace(b.q.cuda(), b.cache, 2, 40, 600).numel()
    if ws.numel() < need:
        ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        a.check(*a.gpu(P, cu_q=None, workspace=ws))
        b.check(*b.gpu(P, workspace=ws))
    assert int(ws[:P.KV4_COUNTER_BYTES].sum()) == 0


def test_beyond_32_bit_offsets():
    """Rows, and attention, in the pages past 4 GiB of a cache."""
    P = need_gpu()
    Hkv, D, page = 2, 128, 64
    per = P.lib().w4a16_kv4_cache_bytes(1, Hkv, D, page)
    pages = 5 * 2 ** 30 // per
    cache = torch.empty((pages, Hkv, page // 16, 16 * D + 128), dtype=torch.uint8, device="cuda")
    gen = torch.Generator().manual_seed(9)
    L = 150
    k, v = rows(gen, L, Hkv, D, F16), rows(gen, L, Hkv, D, F16)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    t = torch.arange(L)
    slots = (table[0, t // page].long() * page + t % page).int()
    assert pages * page < 2 ** 31 and (pages - 2) * per > 2 ** 32
    P.kv4_write(k.cuda(), v.cuda(), cache, slots.cuda())
    ko, vo = P.kv4_read(cache, slots.cuda())
    held = [plain.quantise(x)[3] for x in (k, v)]
    assert same(ko, plain.rounded(held[0], F16)) and same(vo, plain.rounded(held[1], F16))
    q = torch.randn((1, 4, D), generator=gen).half()
    out = P.kv4_attention(q.cuda(), cache, table.cuda(), torch.tensor([L], dtype=torch.int32, device="cuda"))
    o = plain.attention(q.double().numpy(), [held[0]], [held[1]], [1], [L])[0]
    assert np.abs(out.double().cpu().numpy() - o).max() <= 2.0 ** -9 * np.abs(o).max()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,lens", [([1, 1], [70, 200]), ([80, 90], [100, 95])])
def test_rows_that_are_not_finite(dtype, nq, lens):
    """A key or value row of NaN reaches the queries that see it, whole rows of them, and no other; a query
    with an infinity or NaN itself alone."""
    P = need_gpu()
    b = Batch(P, nq, lens, 4, 2, 64, 16, dtype)
    gen = torch.Generator().manual_seed(3)
    k, v = rows(gen, 2, 2, 64, dtype), rows(gen, 2, 2, 64, dtype)
    k[0, 1, 5], v[1, 0, 7] = float("nan"), float("inf")
    # the key at token len - 1 of sequence 0 (head 1), the value at token len - 1 of sequence 1 (head 0)
    last = torch.tensor([int(b.table[s, (lens[s] - 1) // 16]) * 16 + (lens[s] - 1) % 16 for s in (0, 1)], dtype=torch.int32)
    P.kv4_write(k.cuda(), v.cuda(), b.cache, last.cuda())
    for s in (0, 1):
        b.k[s][lens[s] - 1], b.v[s][lens[s] - 1] = plain.quantise(k)[3][s], plain.quantise(v)[3][s]
    b.q[0, 0, 3] = float("inf")
    if nq[0] > 1:
        b.q[0, 3, 3], b.q[1, 1, 0] = float("nan"), -float("inf")
    out, lse = (x.cpu().double().numpy() for x in b.gpu(P))
    want, wl, *_ = plain.attention(b.q.double().numpy(), b.k, b.v, nq, lens)
    assert (np.isnan(out) == np.isnan(want)).all()
    assert np.isnan(want).any() and not np.isnan(want).all()
    fine = ~np.isnan(want)
    assert np.abs(out[fine] - want[fine]).max() < 0.05


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("vscale", [2e4, 4e3])
@pytest.mark.parametrize("nq,L,at", [(1, 90, 3), (1, 90, 88), (90, 600, 3), (90, 600, 555)])
def test_value_rows_of_nan_at_no_weight(dtype, nq, L, at, vscale):
    """A value row of NaN makes the queries NaN that see it, though its weight is e^-200 and less of the sum's
    and the other values are large; where all queries see a step of keys, and where some do not. (At 2e4 some
    of fp16's rows hold an infinity themselves.)"""
    P = need_gpu()
    b = Batch(P, [nq], [L], 4, 2, 64, 16, dtype, vscale=vscale)
    k = rows(torch.Generator().manual_seed(1), 1, 2, 64, dtype)
    k[:] = -40.0
    b.q = (b.q.float().abs() + 1).to(dtype)
    v = torch.full_like(k, float("nan"))
    P.kv4_write(k.cuda(), v.cuda(), b.cache, (b.table[0, at // 16:at // 16 + 1] * 16 + at % 16).cuda())
    out, lse = b.gpu(P)
    b.v[0][at] = np.nan
    bad = np.isnan(b.v[0]).any(-1)                                      # [key, head]
    want = np.stack([bad[:L - nq + 1 + i].any(0) for i in range(nq)]).repeat(2, 1)
    assert (torch.isnan(out).cpu().numpy() == want[..., None]).all() and not torch.isnan(lse).any()
    if vscale < 1e4:
        assert (want == (np.arange(nq) + L - nq >= at)[:, None]).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,L,window", [(1, 90, 50), (5, 300, 0), (5, 300, 77), (150, 200, 0), (150, 400, 70)])
def test_rows_that_a_query_does_not_see(dtype, nq, L, window):
    """What masked tokens hold moves no bit of a query's result: any bytes before the window and behind the
    keys, and, for queries that do not see them, keys and values at the type's end, NaN and infinities."""
    P = need_gpu()
    b = Batch(P, [nq], [L], 4, 2, 64, 16, dtype, seed=6)
    out, lse = b.gpu(P, window=window)
    b.check(out, lse, window=window)
    blocks = b.cache[b.table[0].long()].cpu().numpy()          # pages of 16 tokens
    before = max(0, L - nq + 1 - window) if window else 0     # tokens that no query sees
    for t in [*range(before), *range(L, 16 * b.table.shape[1])]:
        for at in (16 * 64 + 4 * (t % 16), 16 * 64 + 64 + 4 * (t % 16)):   # scales of NaN and near the type's end
            blocks[t // 16, :, 0, at:at + 4] = np.frombuffer(np.uint32(0x7FFF if t % 3 else 0x7BFF).tobytes(), np.uint8)
    b.cache[b.table[0].long()] = torch.from_numpy(blocks).cuda()
    out2, lse2 = b.gpu(P, window=window)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    for x in (torch.finfo(dtype).max, float("nan"), float("inf")):   # the last token: the last query's alone
        far = torch.full((1, 2, 64), x, dtype=dtype, device="cuda")
        P.kv4_write(far, far, b.cache, (b.table[0, (L - 1) // 16:(L - 1) // 16 + 1] * 16 + (L - 1) % 16).cuda())
        out2, lse2 = b.gpu(P, window=window)
        assert torch.equal(out[:-1], out2[:-1]) and torch.equal(lse[:-1], lse2[:-1]), x


@pytest.mark.parametrize("dtype,q,k,v", [(F16, 4.0, 40.0, 1.0), (F16, 1e-3, 1e-2, 1e-4), (F16, 1.0, 1.0, 6e4 / 5), (F16, 0.0, 1.0, 1.0),
                                         (BF16, 1e4, 1e-4, 1e20), (BF16, 1e-20, 1e18, 1e-12), (BF16, 1e15, 1e-15, 1.0)])
def test_magnitudes(dtype, q, k, v):
    """Keys, values and queries far from 1; all weight on one key; none of it anywhere."""
    P = need_gpu()
    for nq, lens in (([1, 1], [400, 33]), ([70], [130])):
        b = Batch(P, nq, lens, 4, 1, 128, 16, dtype, kscale=k, vscale=v)
        b.q = (b.q.float() * q).to(dtype)
        b.check(*b.gpu(P), what=(q, k, v))


def test_scales_and_no_lse():
    P = need_gpu()
    for scale in (0.0, -0.3, 1.7):
        b = Batch(P, [1, 4], [50, 300], 4, 4, 64, 32, F16)
        b.check(*b.gpu(P, scale=scale), scale=scale)
    out = b.gpu(P, scale=1.7)[0]
    assert torch.equal(out, b.gpu(P, scale=1.7, lse=None)[0])


@pytest.mark.parametrize("nq,lens", [([1, 1, 1], [100, 260, 64]), ([40, 100, 3], [100, 260, 64])])
def test_pages_that_do_not_exist(nq, lens):
    """Keys in a page whose number is outside the cache are not seen."""
    P = need_gpu()
    b = Batch(P, nq, lens, 8, 2, 64, 16, F16)
    seen = [np.ones(L, bool) for L in lens]
    for s, at, number in ((0, 2, -1), (1, 0, len(b.cache)), (1, 9, -2 ** 31), (1, 16, 2 ** 31 - 1), (2, 3, -5)):
        b.table[s, at] = number
        seen[s][16 * at:16 * at + 16] = False
    b.check(*b.gpu(P), seen=seen)


@pytest.mark.parametrize("nq,lens,small", [([2, 3], [40, 20], True), ([70, 80], [90, 100], False)])
def test_rows_and_lengths_out_of_bounds(nq, lens, small):
    """Rows outside every sequence stay as they were; lengths are cut to the table and to max_kv_len, negative
    ones to 0; queries beyond max_q_len stay; what the arrays say beyond T is cut."""
    P = need_gpu()
    b = Batch(P, nq, lens, 4, 2, 64, 16, F16)
    T = sum(nq)
    q = torch.randn((T + 5, 4, 64)).half()
    q[2:2 + T] = b.q
    for cu, kv, want_lens in (([2, 2 + nq[0], 2 + T], lens, lens),
                              ([2, 2 + nq[0], 2 + T], [10 ** 9, -7], [lens[0], 0])):
        out = torch.full((T + 5, 4, 64), 3.0, dtype=F16, device="cuda")
        lse = torch.full((T + 5, 4), 3.0, device="cuda")
        # (10^9 is cut to max_kv_len)
        P.kv4_attention(q.cuda(), b.cache, b.table.cuda(), torch.tensor(kv, dtype=torch.int32, device="cuda"),
                        cu_q=torch.tensor(cu, dtype=torch.int32, device="cuda"), max_q_len=max(nq),
                        max_kv_len=lens[0] if want_lens[1] == 0 else max(lens), out=out, lse=lse)
        assert (out[:2] == 3).all() and (out[2 + T:] == 3).all() and (lse[:2] == 3).all() and (lse[2 + T:] == 3).all()
        keep = b.lens
        b.lens = want_lens
        b.k, b.v = ([x[:L] for x, L in zip(y, want_lens)] for y in (b.k, b.v))
        b.check(out[2:2 + T], lse[2:2 + T])
        b.lens = keep
    # two queries of each sequence only
    b = Batch(P, nq, lens, 4, 2, 64, 16, F16)
    out = torch.full((T, 4, 64), 3.0, dtype=F16, device="cuda")
    full, _ = b.gpu(P)
    b.gpu(P, out=out, max_q_len=2)
    for s in (0, 1):
        a = int(b.cu[s])
        assert (out[a + 2:int(b.cu[s + 1])] == 3).all()
        torch.testing.assert_close(out[a:a + 2], full[a:a + 2], rtol=2e-3, atol=2e-3)
    # sequences that overlap, run backwards or leave the rows: memory stays intact, the others' rows right
    out = b.gpu(P, cu_q=torch.tensor([0, nq[0], 10 ** 6], dtype=torch.int32, device="cuda"), max_q_len=T)[0]
    assert out.shape == (T, 4, 64)
    torch.testing.assert_close(out[:nq[0]], full[:nq[0]], rtol=2e-3, atol=2e-3)
    b.gpu(P, cu_q=torch.tensor([T, 3, -9], dtype=torch.int32, device="cuda"), max_q_len=T)
    torch.cuda.synchronize()


@pytest.mark.parametrize("nq", [1, 90])
def test_strided_queries_and_outputs(nq):
    """Queries out of a fused projection, results into head-major rows."""
    P = need_gpu()
    Hq, Hkv, D = 8, 2, 128
    b = Batch(P, [nq, nq], [100, 130], Hq, Hkv, D, 16, F16)
    qkv = torch.zeros((2 * nq, Hq + 2 * Hkv, D), dtype=F16, device="cuda")
    qkv[:, :Hq] = b.q.cuda()
    out = torch.zeros((Hq, 2 * nq, D), dtype=F16, device="cuda").transpose(0, 1)
    _, lse = b.gpu(P, q=qkv[:, :Hq], out=out)
    b.check(out, lse)


@pytest.mark.parametrize("nq,lens,D", [([1, 1], [1500, 40], 128), ([9, 2], [900, 1100], 256), ([200, 130], [300, 1500], 64)])
def test_out_in_the_place_of_q(nq, lens, D):
    """A program that keeps no second buffer: out is q, through one chunk and several, and either join."""
    P = need_gpu()
    b = Batch(P, nq, lens, 8, 2, D, 16, F16)
    want, _ = b.gpu(P)
    q = b.q.cuda()
    got, _ = b.gpu(P, q=q, out=q)
    assert got is q and torch.equal(got, want)


def test_no_work():
    P = need_gpu()
    cache = P.kv4_cache(2, 2, 64, 16)
    empty = torch.zeros((0, 2, 64), dtype=F16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    P.kv4_write(empty, empty, cache, none)
    assert P.kv4_read(cache, none)[0].shape == (0, 2, 64)
    assert P.kv4_attention(torch.zeros((0, 4, 64), dtype=F16, device="cuda"), cache,
                           torch.zeros((0, 1), dtype=torch.int32, device="cuda"), none).shape == (0, 4, 64)


def test_sizes_beyond_32_bits_are_refused():
    """(The C entry takes 32-bit sizes, and the upper bits of a Python integer would be dropped on the way.)"""
    P = need_gpu()
    b = Batch(P, [1], [20], 4, 2, 64, 16, F16)
    for over in (dict(max_kv_len=2 ** 32 + 20), dict(window=2 ** 32 + 1), dict(cu_q=b.cu.cuda(), max_q_len=2 ** 32 + 1)):
        with pytest.raises(P.InvalidArgument, match="32-bit"):
            b.gpu(P, **over)
    with pytest.raises(P.InvalidArgument, match="32-bit"):
        P.kv4_attention_workspace(b.q.cuda(), b.cache, 1, 1, 2 ** 32 + 20)
    k = torch.zeros((1, 2, 64), dtype=F16, device="cuda").as_strided((1, 2, 64), (2 ** 32, 64, 1))
    with pytest.raises(P.InvalidArgument, match="32-bit"):
        P.kv4_write(k, k, b.cache, torch.zeros(1, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------ as a program uses them

def test_steps_of_a_program():
    """A prompt, then token by token: written, attended over, on a captured graph that is replayed with new
    slots, lengths and rows; every step against 64 bits, and the eager call between them."""
    P = need_gpu()
    B, Hq, Hkv, D, page, dtype = 3, 8, 2, 128, 16, F16
    gen = torch.Generator().manual_seed(2)
    first, steps = [40, 15, 700], 5
    per = 46
    table = torch.randperm(B * per, generator=gen).view(B, per).int()
    cache = P.kv4_cache(B * per, Hkv, D, page)
    k = [rows(gen, n + steps, Hkv, D, dtype) for n in first]
    v = [rows(gen, n + steps, Hkv, D, dtype) for n in first]
    held_k, held_v = [plain.quantise(x)[3] for x in k], [plain.quantise(x)[3] for x in v]

    def slot(b, t):
        return int(table[b, t // page]) * page + t % page

    # the prompts
    slots = torch.tensor([slot(b, t) for b in range(B) for t in range(first[b])], dtype=torch.int32)
    P.kv4_write(torch.cat([x[:n] for x, n in zip(k, first)]).cuda(), torch.cat([x[:n] for x, n in zip(v, first)]).cuda(), cache, slots.cuda())
    # one step, captured
    d = {"k": torch.zeros((B, Hkv, D), dtype=dtype, device="cuda"), "v": torch.zeros((B, Hkv, D), dtype=dtype, device="cuda"),
         "q": torch.zeros((B, Hq, D), dtype=dtype, device="cuda"), "slots": torch.full((B,), -1, dtype=torch.int32, device="cuda"),
         "lens": torch.zeros(B, dtype=torch.int32, device="cuda"), "out": torch.zeros((B, Hq, D), dtype=dtype, device="cuda"),
         "lse": torch.zeros((B, Hq), device="cuda"), "table": table.cuda()}
    ws = P.kv4_attention_workspace(d["q"], cache, B, 1, per * page)

    def step(out, lse, ws):
        P.kv4_write(d["k"], d["v"], cache, d["slots"])
        P.kv4_attention(d["q"], cache, d["table"], d["lens"], out=out, lse=lse, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(d["out"], d["lse"], ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(d["out"], d["lse"], ws)
    for i in range(steps):
        q = torch.randn((B, Hq, D), generator=gen).to(dtype)
        lens = [n + i + 1 for n in first]
        d["q"].copy_(q)
        d["k"].copy_(torch.stack([x[n + i] for x, n in zip(k, first)]))
        d["v"].copy_(torch.stack([x[n + i] for x, n in zip(v, first)]))
        d["slots"].copy_(torch.tensor([slot(b, first[b] + i) for b in range(B)], dtype=torch.int32))
        d["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        b = Batch.__new__(Batch)
        b.nq, b.lens, b.dtype, b.D, b.Hq, b.q = [1] * B, lens, dtype, D, Hq, q
        b.k, b.v = [x[:L] for x, L in zip(held_k, lens)], [x[:L] for x, L in zip(held_v, lens)]
        b.check(d["out"], d["lse"], what=f"step {i}")
        eager, lse = torch.zeros_like(d["out"]), torch.zeros_like(d["lse"])
        step(eager, lse, None)
        assert torch.equal(eager, d["out"]) and torch.equal(lse, d["lse"])


def test_two_streams_with_a_workspace_each():
    P = need_gpu()
    bs = [Batch(P, [1, 1], [3000, 2000], 8, 2, 128, 64, F16, seed=s) for s in (1, 2)]
    args = [(b.q.cuda(), b.table.cuda(), torch.tensor(b.lens, dtype=torch.int32, device="cuda")) for b in bs]
    ws = [P.kv4_attention_workspace(a[0], b.cache, 2, 1, 3000) for a, b in zip(args, bs)]
    outs = [[torch.zeros_like(a[0]) for _ in range(10)] for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(10):
        for s in (0, 1):
            with torch.cuda.stream(streams[s]):
                P.kv4_attention(args[s][0], bs[s].cache, args[s][1], args[s][2], max_kv_len=3000, out=outs[s][i], workspace=ws[s])
    torch.cuda.synchronize()
    for s in (0, 1):
        want = bs[s].gpu(P, cu_q=None)
        bs[s].check(*want)
        assert all(torch.equal(o, want[0]) for o in outs[s])


def test_attention_block_on_int4_weights():
    """An attention block as a decode step runs it: fused q, k, v projection with int4 weights, the new rows into the
    cache, attention, output projection; the chain against 64 bits on the same weights and cache."""
    P = need_gpu()
    Hq, Hkv, D, B, G = 8, 2, 64, 2, 64
    hidden = Hq * D
    gen = torch.Generator("cuda").manual_seed(11)

    def layer(K, N):
        qw = torch.randint(-2 ** 31, 2 ** 31 - 1, (K // 8, N), generator=gen, device="cuda", dtype=torch.int64).int()
        sc = (torch.rand((K // G, N), generator=gen, device="cuda") * 0.004 + 0.002).half()
        return qw, sc

    wqkv, wo = layer(hidden, (Hq + 2 * Hkv) * D), layer(hidden, hidden)
    dense = [P.dequant(q, s, None, fmt="gptq_sym", group_size=G).double() for q, s in (wqkv, wo)]
    cache = P.kv4_cache(8, Hkv, D, 16)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(B, 4)
    keys, vals = [[], []], [[], []]
    for i in range(20):
        x = torch.randn((B, hidden), generator=gen, device="cuda").half()
        qkv = P.gemm(x, wqkv[0], wqkv[1], None, fmt="gptq_sym", group_size=G).view(B, Hq + 2 * Hkv, D)
        slots = (table[:, i // 16] * 16 + i % 16).int()
        P.kv4_write(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], cache, slots)
        lens = torch.full((B,), i + 1, dtype=torch.int32, device="cuda")
        att = P.kv4_attention(qkv[:, :Hq], cache, table, lens)
        y = P.gemm(att.view(B, hidden), wo[0], wo[1], None, fmt="gptq_sym", group_size=G)
        for b in range(B):
            keys[b].append(plain.quantise(qkv[b:b + 1, Hq:Hq + Hkv].cpu())[3])
            vals[b].append(plain.quantise(qkv[b:b + 1, Hq + Hkv:].cpu())[3])
    o = plain.attention(qkv[:, :Hq].double().cpu().numpy(), [np.concatenate(a) for a in keys], [np.concatenate(a) for a in vals],
                        [1] * B, [20] * B)[0]
    want = torch.from_numpy(o).view(B, hidden).cuda() @ dense[1]
    err = (y.double() - want).norm() / want.norm()
    assert err < 2e-3, float(err)
    torch.testing.assert_close(qkv.reshape(B, -1).double(), x.double() @ dense[0], rtol=1e-2, atol=1e-2)
