"""The 8-bit key/value cache on the GPU: rows in and out bit for bit, attention against 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_plain
import kv8_plain as plain
from test_gpu_kv4 import BF16, F16, Batch, need_gpu, rows, same
from test_gpu_layer import NORM_REL

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def random_cache(P, pages, H, D, page, seed=1):
    cache = P.kv8_cache(pages, H, D, page)
    cache.random_(0, 256, generator=torch.Generator("cuda").manual_seed(seed))
    return cache


def read_back(P, cache, table, lens, dtype):
    """(k, v) rows [sum lens, Hkv, D] of whole sequences."""
    page = cache.shape[2] * 16
    slots = [int(table[b, t // page]) * page + t % page for b, n in enumerate(lens) for t in range(n)]
    return P.kv8_read(cache, i32(slots), dtype)


# ------------------------------------------------------------------ rows

@TYPES
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("kind,H,page,steps", [
    ("normal", 1, 16, [[1]]),                                         # one token
    ("wide", 3, 32, [[37, 5, 16], [1, 1, 1], [0, 11, 1], [30, 0, 2]]),    # prompts, single tokens, drafts, more
    ("far", 2, 16, [[3, 17], [1, 2], [1, 1], [1, 1], [15, 9]]),           # scales that grow block after block
    ("constant", 1, 128, [[18], [1], [20]]),
    ("normal", 9, 64, [[130, 1, 0, 77, 33]]),
])
def test_rows_in_and_out(dtype, D, kind, H, page, steps):
    """Appended step by step: every byte of the cache as the definition has it, those that no row owns as they were."""
    P = need_gpu()
    B = len(steps[0])
    total = [sum(s[b] for s in steps) for b in range(B)]
    gen = torch.Generator().manual_seed(sum(total) * 1000 + D)
    per = max(total) // page + 2
    pages = B * per + 1
    table = torch.randperm(pages, generator=gen)[:B * per].view(B, per).int()
    cache = random_cache(P, pages, H, D, page)
    want = cache.cpu().numpy().copy()
    lens = [0] * B
    for i, n in enumerate(steps):
        T = sum(n)
        k, v = rows(gen, T, H, D, dtype, kind), rows(gen, T, H, D, dtype, kind)
        cu = np.cumsum([0] + n)
        for b in range(B):
            plain.append(want, table.numpy(), b, lens[b], k[cu[b]:cu[b + 1]].double().numpy(), v[cu[b]:cu[b + 1]].double().numpy())
            lens[b] += n[b]
        every = all(x == 1 for x in n)
        got = P.kv8_write(k.cuda(), v.cuda(), cache, table.cuda(), i32(lens), cu_q=None if every and i % 2 else i32(cu),
                          max_q_len=None if i % 2 or every else max(n))
        assert got is cache
        diff = np.argwhere(cache.cpu().numpy() != want)
        assert len(diff) == 0, (i, diff[:8])
    back = read_back(P, cache, table, lens, dtype)
    for which, x in enumerate(back):
        exp = np.concatenate([plain.held(want, table.numpy(), b, lens[b])[which] for b in range(B)])
        assert same(x, kv4_plain.rounded(exp, dtype))


@TYPES
def test_rows_rewritten(dtype):
    """Drafts that were not accepted: the sequence goes back, other tokens take their place; a block of which the
    first token is written anew takes a scale of its own again."""
    P = need_gpu()
    H, D, page = 2, 64, 16
    gen = torch.Generator().manual_seed(4)
    table = torch.tensor([[1, 0, 2]], dtype=torch.int32)
    cache = random_cache(P, 3, H, D, page)
    want = cache.cpu().numpy().copy()
    for length, n, size in ((20, 20, 1.0), (24, 4, 300.0), (22, 2, 1.0), (37, 15, 0.1), (33, 1, 5.0), (16, 16, 2.0 ** -8)):
        k, v = ((rows(gen, n, H, D, dtype).float() * size).to(dtype) for _ in range(2))
        plain.append(want, table.numpy(), 0, length - n, k.double().numpy(), v.double().numpy())
        P.kv8_write(k.cuda(), v.cuda(), cache, table.cuda(), i32([length]), cu_q=i32([0, n]))
        assert np.array_equal(cache.cpu().numpy(), want), (length, n)


@TYPES
def test_rows_not_finite(dtype):
    """A row with an infinity or NaN is NaN throughout, does not count for its block's scale, and is fine again when
    it is written anew; its neighbours are as ever."""
    P = need_gpu()
    H, D = 2, 128
    gen = torch.Generator().manual_seed(5)
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    cache = random_cache(P, 2, H, D, 16)
    want = cache.cpu().numpy().copy()
    k, v = rows(gen, 20, H, D, dtype), rows(gen, 20, H, D, dtype)
    k[1, 0, 5], k[2, 1, 127], v[3, 0, 0], v[17, 1, 64] = float("nan"), float("inf"), -float("inf"), float("nan")
    at = 0
    for n in (4, 1, 13, 2):
        plain.append(want, table.numpy(), 0, at, k[at:at + n].double().numpy(), v[at:at + n].double().numpy())
        at += n
        P.kv8_write(k[at - n:at].cuda(), v[at - n:at].cuda(), cache, table.cuda(), i32([at]), cu_q=i32([0, n]))
        assert np.array_equal(cache.cpu().numpy(), want)
    ko, vo = read_back(P, cache, table, [20], dtype)
    exp = plain.held(want, table.numpy(), 0, 20)
    assert same(ko, kv4_plain.rounded(exp[0], dtype)) and same(vo, kv4_plain.rounded(exp[1], dtype))
    assert ko[1, 0].isnan().all() and not ko[1, 1].isnan().any() and vo[17, 1].isnan().all() and int(ko.isnan().sum()) == 2 * D
    fresh = rows(gen, 3, H, D, dtype)
    plain.append(want, table.numpy(), 0, 17, fresh.double().numpy(), fresh.double().numpy())
    P.kv8_write(fresh.cuda(), fresh.cuda(), cache, table.cuda(), i32([20]), cu_q=i32([0, 3]))
    assert np.array_equal(cache.cpu().numpy(), want)


@TYPES
@pytest.mark.parametrize("D", [64, 256])
def test_rows_at_the_ends_of_the_types(dtype, D):
    """The largest values (which a byte rounds beyond), the smallest, zeros, and scales at their least."""
    P = need_gpu()
    most, least = torch.finfo(dtype).max, 2.0 ** -24 if dtype == F16 else 2.0 ** -133
    gen = torch.Generator().manual_seed(6)
    x = rows(gen, 96, 2, D, dtype).double()
    x[:16] = torch.sign(x[:16]) * most
    x[16:32] *= least
    x[32:48] = 0
    x[48:64] = x[48:64] * 2.0 ** -61
    x[64] = most
    x = x.clamp(-most, most).float().to(dtype)
    table = torch.arange(6, dtype=torch.int32)[None]
    cache = random_cache(P, 6, 2, D, 16)
    want = cache.cpu().numpy().copy()
    plain.append(want, table.numpy(), 0, 0, x.double().numpy(), -x.double().numpy())
    P.kv8_write(x.cuda(), -x.cuda(), cache, table.cuda(), i32([96]), cu_q=i32([0, 96]))
    assert np.array_equal(cache.cpu().numpy(), want)
    ko, vo = read_back(P, cache, table, [96], dtype)
    for which, o in enumerate((ko, vo)):
        assert same(o, kv4_plain.rounded(plain.held(want, table.numpy(), 0, 96)[which], dtype)) and torch.isfinite(o).all()


def test_rows_strided_and_repeated():
    """Slices of a fused projection, head-major rows; a slot read into two places, slots that are passed over."""
    P = need_gpu()
    T, H, D = 21, 4, 128
    gen = torch.Generator().manual_seed(8)
    qkv = torch.randn((T, 3 * H, D), generator=gen).half().cuda()
    k, v = qkv[:, H:2 * H], qkv[:, 2 * H:].transpose(0, 1).contiguous().transpose(0, 1)
    a, b = P.kv8_cache(2, H, D, 32), P.kv8_cache(2, H, D, 32)
    table = i32([[1, 0]])
    P.kv8_write(k, v, a, table, i32([T]), cu_q=i32([0, T]))
    P.kv8_write(k.contiguous(), v.contiguous(), b, table, i32([T]), cu_q=i32([0, T]))
    assert torch.equal(a, b)
    slots = i32([32 + t for t in range(T)] + [-1, 32, 33, 64, 2 ** 31 - 1, -2 ** 31, 34])
    big = torch.full((H, T + 7, 2 * D), 7.0, dtype=F16, device="cuda")
    ko, vo = big[..., :D].transpose(0, 1), big[..., D:].transpose(0, 1)
    P.kv8_read(a, slots, k_out=ko, v_out=vo)
    for x, w in ((ko, P.kv8_read(a, slots[:T])[0]), (vo, P.kv8_read(a, slots[:T])[1])):
        assert torch.equal(x[:T], w) and (x[[T, T + 3, T + 4, T + 5]] == 7).all()
        assert torch.equal(x[[T + 1, T + 2, T + 6]], w[:3])


@pytest.mark.parametrize("max_q", [None, 40])
@pytest.mark.parametrize("B", [3, 70])
def test_rows_out_of_bounds(B, max_q):
    """Padding behind the last sequence and before the first, tokens before 0 or beyond the table, pages that do not exist,
    lengths of nonsense, more tokens than max_q_len: passed over, and no byte beside them moves."""
    P = need_gpu()
    H, D, page, dtype = 2, 64, 16, F16
    gen = torch.Generator().manual_seed(B)
    per = 3
    table = torch.randperm(B * per, generator=gen).view(B, per).int()
    table[1, 1], table[2, 0] = -1, B * per
    n = [int(x) for x in torch.randint(0, 8, (B,), generator=gen)]
    n[0], n[1], n[2] = 45, 20, 18
    lens = [x + int(o) for x, o in zip(n, torch.randint(0, 30, (B,), generator=gen))]
    lens[0] = 40                                          # five tokens before 0
    lens[1] = 53                                          # beyond the table's 48
    if B > 5:
        lens[3], lens[4], lens[5] = -7, 2 ** 31 - 1, -2 ** 31
    T = sum(n) + 6
    cu = np.cumsum([2] + n)
    k, v = rows(gen, T, H, D, dtype), rows(gen, T, H, D, dtype)
    cache = random_cache(P, B * per, H, D, page)
    want = cache.cpu().numpy().copy()
    for b in range(B):   # the tokens before the new ones, which a call takes to be there
        if 0 < lens[b] - n[b] < 2 ** 30:
            old = rows(gen, min(lens[b] - n[b], per * page), H, D, dtype)
            plain.append(want, table.numpy(), b, 0, old.double().numpy(), -old.double().numpy())
    cache.copy_(torch.from_numpy(want))
    for b in range(B):
        take = n[b] if max_q is None else min(n[b], max_q)
        if 0 < lens[b] <= 2 ** 30:
            plain.append(want, table.numpy(), b, lens[b] - n[b], k[cu[b]:cu[b] + take].double().numpy(), v[cu[b]:cu[b] + take].double().numpy())
    P.kv8_write(k.cuda(), v.cuda(), cache, table.cuda(), i32(lens), cu_q=i32(cu), max_q_len=max_q)
    diff = np.argwhere(cache.cpu().numpy() != want)
    assert len(diff) == 0, diff[:5]
    # offsets that overlap, run backwards or leave the rows: no fault, no other page
    P.kv8_write(k.cuda(), v.cuda(), cache, i32([[0, 1, 2]] * 3), i32([40, 40, 40]), cu_q=i32([T, 3, -9, 10 ** 6]))
    torch.cuda.synchronize()
    assert np.array_equal(cache[3:].cpu().numpy(), want[3:])


def test_beyond_32_bit_offsets():
    """Rows, and attention, in the pages past 4 GiB of a cache."""
    P = need_gpu()
    Hkv, D, page = 2, 128, 64
    size = P.lib().w4a16_kv8_cache_bytes(1, Hkv, D, page)
    pages = 5 * 2 ** 30 // size
    cache = torch.empty((pages, Hkv, page // 16, 32 * D + 16), dtype=torch.uint8, device="cuda")
    gen = torch.Generator().manual_seed(9)
    L = 150
    k, v = rows(gen, L, Hkv, D, F16), rows(gen, L, Hkv, D, F16)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    assert pages * page < 2 ** 31 and (pages - 2) * size > 2 ** 32
    P.kv8_write(k.cuda(), v.cuda(), cache, table.cuda(), i32([L]), cu_q=i32([0, L]))
    small, few = np.zeros((3, Hkv, 4, 32 * D + 16), np.uint8), np.array([[0, 1, 2]])
    plain.append(small, few, 0, 0, k.double().numpy(), v.double().numpy())
    assert np.array_equal(cache[table[0].long()].cpu().numpy()[:, :, :2], small[:, :, :2])
    hk, hv = plain.held(small, few, 0, L)
    ko, vo = read_back(P, cache, table, [L], F16)
    assert same(ko, kv4_plain.rounded(hk, F16)) and same(vo, kv4_plain.rounded(hv, F16))
    q = torch.randn((1, 4, D), generator=gen).half()
    out = P.kv8_attention(q.cuda(), cache, table.cuda(), i32([L]))
    o = kv4_plain.attention(q.double().numpy(), [hk], [hv], [1], [L])[0]
    assert np.abs(out.double().cpu().numpy() - o).max() <= 2.0 ** -9 * np.abs(o).max()


# ------------------------------------------------------------------ rows that are rotated on the way

@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("D,rot,Hq,Hkv,explicit", [(64, 64, 4, 2, False), (128, 128, 32, 8, False), (128, 50, 3, 1, True), (192, 192, 2, 2, True),
                                                   (256, 62, 8, 1, False), (64, 2, 5, 5, True), (256, 256, 1, 1, False)])
@pytest.mark.parametrize("n,lens", [([1, 1, 1], [30, 1, 17]), ([40, 3, 0, 70], [40, 20, 5, 100])])
def test_rotated_rows(dtype, interleaved, D, rot, Hq, Hkv, explicit, n, lens):
    """Keys are held as their rotation in 64 bits within half a step of e4m3 (2^-4, or 2^-10 scales) and the four fp32 roundings of
    2^-24 of |a| + |b|; values bit for bit; queries with rope's bits. Positions are the tokens' places, or given."""
    P = need_gpu()
    B, page, T = len(n), 32, sum(n) + 3
    gen = torch.Generator().manual_seed(D + rot + T)
    table = torch.randperm(5 * B, generator=gen).view(B, 5).int()
    cu = np.cumsum([1] + n)
    qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=gen).to(dtype).cuda()
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    places = torch.full((T,), -1, dtype=torch.int32)
    for b in range(B):
        places[cu[b]:cu[b + 1]] = torch.arange(lens[b] - n[b], lens[b])
    positions = torch.randint(0, 10 ** 6, (T,), generator=gen).int() if explicit else places
    r = P.Rope(rot, 10000.0, interleaved=interleaved, magnitude=1.1)
    cache, old = random_cache(P, 5 * B, Hkv, D, page), None
    old = cache.cpu().numpy().copy()
    # older tokens, so that there are blocks to append to
    for b in range(B):
        m = lens[b] - n[b]
        if m:
            x = rows(gen, m, Hkv, D, dtype)
            plain.append(old, table.numpy(), b, 0, x.double().numpy(), x.double().numpy())
    cache.copy_(torch.from_numpy(old))
    qo = torch.full((T, Hq, D), 5.0, dtype=dtype, device="cuda")
    P.kv8_write(k, v, cache, table.cuda(), i32(lens), cu_q=i32(cu), max_q_len=max(n), rope=r, positions=positions.cuda() if explicit else None, q=q, q_out=qo)
    mine = (places >= 0).cuda()
    want_q = P.rope(q, positions.cuda(), r, q_out=torch.empty_like(q.contiguous()))
    assert torch.equal(qo[mine], want_q[mine]) and (explicit or (qo[~mine] == 5).all())
    kd, reach = plain.rotate(k.double().cpu().numpy(), positions.numpy(), r.inv_freq.cpu().numpy(), interleaved, 1.1)
    got = cache.cpu().numpy()
    exact = old.copy()
    for b in range(B):
        plain.append(exact, table.numpy(), b, lens[b] - n[b], kd[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]].double().cpu().numpy())
        for t in range(lens[b] - n[b], lens[b]):
            number, blk = int(table[b, t // page]), t % page // 16
            row = cu[b] + t - (lens[b] - n[b])
            for h in range(Hkv):
                s = np.frombuffer(got[number, h, blk, 32 * D:32 * D + 4].tobytes(), np.float32)[0]
                s_exact = np.frombuffer(exact[number, h, blk, 32 * D:32 * D + 4].tobytes(), np.float32)[0]
                assert s == s_exact or s in (2 * s_exact, s_exact / 2)   # (the largest next to 448 scales)
                off = reach[row, h] * (4 * 2.0 ** -24 + 1e6 * 2.0 ** -50)
                x = kd[row, h]
                held = plain.block_rows(got[number, h, blk], D)[0][t % 16]
                assert (np.abs(held - x) <= np.maximum((np.abs(x) + off) / 16, s * 2.0 ** -10) + off).all()
    # values, trailers but the keys' scale, and blocks that are not written: bit for bit
    key_bytes = np.zeros(32 * D + 16, bool)
    key_bytes[:16 * D] = key_bytes[32 * D:32 * D + 4] = True
    assert np.array_equal(got[..., ~key_bytes], exact[..., ~key_bytes])
    share = (got != exact).mean()
    assert share < 1e-4, share    # (a key next to the middle of two numbers falls to either side)
    # in place, the same
    again = torch.from_numpy(old).cuda()
    P.kv8_write(k, v, again, table.cuda(), i32(lens), cu_q=i32(cu), rope=r, positions=positions.cuda() if explicit else None, q=q)
    assert torch.equal(again, cache) and torch.equal(q[mine], want_q[mine])


def test_rotation_of_queries_without_new_lengths():
    """Without cu_q; keys alone, without queries."""
    P = need_gpu()
    B, Hkv, D = 5, 2, 64
    gen = torch.Generator().manual_seed(3)
    k = torch.randn((B, Hkv, D), generator=gen).half().cuda()
    q = torch.randn((B, 6, D), generator=gen).half().cuda()
    lens = i32([1, 9, 16, 17, 30])
    table = i32(torch.arange(10).view(5, 2))
    r = P.Rope(D)
    a, b = P.kv8_cache(10, Hkv, D, 16), P.kv8_cache(10, Hkv, D, 16)
    P.kv8_write(k, k, a, table, lens, rope=r)
    out = torch.empty_like(q)
    P.kv8_write(k, k, b, table, lens, rope=r, q=q, q_out=out)
    assert torch.equal(a, b) and torch.equal(out, P.rope(q, lens - 1, r, q_out=torch.empty_like(q)))


@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("n", [None, [1000, 0, 3, 217], [17] * 70, [1, 0] * 600 + [200] * 3])
def test_rotation_of_many_queries(n, explicit):
    """A row's bits do not depend on how many there are, nor do the keys' and values'; rows of no sequence stay as they are.
    Without cu_q, too."""
    P = need_gpu()
    Hq, Hkv, D = 32, 1, 128
    gen = torch.Generator().manual_seed(11)
    B, before = (1100, 0) if n is None else (len(n), 5)
    T = B if n is None else sum(n) + 12
    assert T * Hq * D >= 4 << 20
    n = n or [1] * B
    lens = [x + int(torch.randint(0, 40, (1,), generator=gen)) for x in n]
    per = -(-max(lens) // 16)
    table = torch.randperm(B * per, generator=gen).view(B, per).int()
    k = torch.randn((T, Hkv, D), generator=gen).bfloat16().cuda()
    q = torch.randn((T, Hq, D), generator=gen).bfloat16().cuda()
    cu = np.cumsum([before] + n)
    places = torch.full((T,), -1, dtype=torch.int32)
    for b in range(B):
        places[cu[b]:cu[b + 1]] = torch.arange(lens[b] - n[b], lens[b])
    r = P.Rope(D, interleaved=explicit)
    kw = dict(rope=r, positions=places.cuda() if explicit else None)
    if T != B:
        kw.update(cu_q=i32(cu), max_q_len=max(n))
    one, two = P.kv8_cache(B * per, Hkv, D, 16), P.kv8_cache(B * per, Hkv, D, 16)
    P.kv8_write(k, k, one, table.cuda(), i32(lens), **kw)
    out = torch.full_like(q, 5.0)
    P.kv8_write(k, k, two, table.cuda(), i32(lens), q=q, q_out=out, **kw)
    assert torch.equal(one, two)
    mine = (places >= 0).cuda()
    want = torch.cat([P.rope(q[i:i + 50], places[i:i + 50].cuda(), r, q_out=torch.empty_like(q[i:i + 50])) for i in range(0, T, 50)])
    assert torch.equal(out[mine], want[mine]) and (explicit or (out[~mine] == 5).all())


# ------------------------------------------------------------------ attention

class Batch8(Batch):
    """Sequences in an 8-bit cache of shuffled pages, with queries, on the GPU and in 64 bits. (Batch.check's bounds hold: a weight is
    rounded by 2^-12, and below fp16's normal range moves by half of 2^-24 where the largest is 2^8 or more, so a key's share by
    2^-33 448 s, with 448 s at most twice the largest value of a block.)"""

    def __init__(self, P, nq, lens, Hq, Hkv, D, page, dtype, seed=0, kscale=1.0, vscale=1.0, spare=1):
        gen = torch.Generator().manual_seed(seed + 7 * D + Hq)
        self.nq, self.lens, self.dtype, self.D, self.Hq = nq, lens, dtype, D, Hq
        B, per = len(lens), max(1, -(-max(lens) // page)) + spare
        self.table = torch.randperm(B * per, generator=gen).view(B, per).int()
        self.cache = random_cache(P, B * per, Hkv, D, page, 3)   # what is not written: anything
        k = torch.cat([(rows(gen, L, Hkv, D, dtype, "wide").float() * kscale).to(dtype) for L in lens])
        v = torch.cat([(rows(gen, L, Hkv, D, dtype).float() * vscale).to(dtype) for L in lens])
        if len(k):
            P.kv8_write(k.cuda(), v.cuda(), self.cache, self.table.cuda(), i32(lens), cu_q=i32(np.cumsum([0] + list(lens))), max_q_len=max(lens))
        self.read()
        self.q = torch.randn((sum(nq), Hq, D), generator=gen).to(dtype)
        self.cu = torch.tensor([0] + nq).cumsum(0).int()

    def read(self):
        """What the cache holds (its bytes are checked by the tests of rows)."""
        cache = self.cache.cpu().numpy()
        both = [plain.held(cache, self.table.numpy(), b, L) for b, L in enumerate(self.lens)]
        self.k, self.v = [x[0] for x in both], [x[1] for x in both]

    def put(self, P, s, t, k, v):
        """Tokens t.. of sequence s anew: k, v [n, Hkv, D]."""
        P.kv8_write(k.cuda(), v.cuda(), self.cache, self.table[s:s + 1].cuda(), i32([t + len(k)]), cu_q=i32([0, len(k)]))
        self.read()

    def gpu(self, P, **over):
        a = dict(cu_q=self.cu.cuda(), max_q_len=max(1, max(self.nq)), max_kv_len=max(self.lens),
                 lse=torch.full((len(self.q), self.Hq), 5.0, device="cuda"))
        a.update(over)
        q = a.pop("q", None)
        out = P.kv8_attention(self.q.cuda() if q is None else q, self.cache, self.table.cuda(), i32(self.lens), **a)
        return out, a["lse"]


HEADS = [(4, 4, 64), (8, 2, 128), (6, 1, 192), (4, 1, 256), (24, 1, 64), (7, 1, 128), (40, 2, 128)]


@TYPES
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("lens,page", [([1], 16), ([0, 1, 15, 16, 17, 33], 16), ([257, 5, 64], 32), ([700, 1300], 128)])
def test_decode(dtype, Hq, Hkv, D, lens, page):
    P = need_gpu()
    b = Batch8(P, [1] * len(lens), lens, Hq, Hkv, D, page, dtype)
    b.check(*b.gpu(P, cu_q=None))


@TYPES
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
    b = Batch8(P, nq, lens, Hq, Hkv, D, 16, dtype)
    b.check(*b.gpu(P, causal=causal, window=window), causal=causal, window=window)


def attention_path(P, T, B, Hq, Hkv, D, max_q, max_kv):
    out = (ctypes.c_int32 * 4)()
    P.lib().w4a16_internal_kv8_path(T, B, Hq, Hkv, D, max_q, max_kv, out)
    return tuple(out)


@TYPES
@pytest.mark.parametrize("nq,lens,Hq,Hkv,D,page,window,path", [
    # few columns (1): one and two column tiles a wave, one chunk a sequence and several, joined by the last workgroup (0)
    # and by a kernel of their own (1), more sequences than a wave has lanes
    ([1] * 3, [100, 128, 7], 8, 2, 128, 16, 0, (1, 1, None, 0)),
    ([1] * 2, [1500, 900], 8, 8, 64, 32, 0, (1, 1, None, 0)),
    ([1], [3000], 4, 1, 128, 64, 0, (1, 1, None, 1)),
    ([1] * 5, [2100, 1, 850, 0, 1300], 24, 1, 128, 16, 0, (1, 2, None, 1)),
    ([5, 5, 3], [1100, 9, 1400], 16, 2, 64, 16, 300, (1, 2, None, 1)),
    ([5], [1000], 4, 1, 64, 16, 0, (1, 2, None, 0)),
    ([8, 2, 8], [1700, 800, 33], 8, 1, 256, 64, 0, (1, 1, None, 1)),
    ([4, 9], [900, 1000], 10, 2, 192, 32, 0, (1, 1, None, 1)),
    ([1] * 130, [(37 * i) % 331 + 600 * (i == 7) for i in range(130)], 2, 1, 64, 16, 0, (1, 1, None, 0)),
    ([1] * 300, [(53 * i) % 200 + 1100 * (i % 97 == 5) for i in range(300)], 2, 1, 64, 16, 0, (1, 1, None, 0)),
    ([1] * 1100, [(29 * i) % 60 + 1000 * (i % 250 == 90) for i in range(1100)], 2, 2, 64, 16, 0, (1, 1, None, 0)),
    # many (2): two groups of waves on a tile, one of them, keys in one chunk and in several
    ([300, 70], [300, 500], 2, 1, 128, 32, 0, (2, 2, 1, 0)),
    ([90], [2500], 4, 2, 64, 16, 0, (2, 2, 5, 0)),
    ([70, 66], [1500, 1030], 1, 1, 256, 64, 700, (2, 1, 3, 0)),
    ([65, 2], [600, 1200], 3, 3, 192, 16, 0, (2, 1, 3, 0)),
    ([129] * 172, [129 + i for i in range(172)], 3, 3, 64, 16, 33, (2, 1, 1, 0)),
])
def test_every_path(dtype, nq, lens, Hq, Hkv, D, page, window, path):
    P = need_gpu()
    got = attention_path(P, sum(nq), len(nq), Hq, Hkv, D, max(nq), max(lens))
    assert all(w is None or g == w for g, w in zip(got, path)), got
    b = Batch8(P, nq, lens, Hq, Hkv, D, page, dtype)
    out, lse = b.gpu(P, window=window)
    b.check(out, lse, window=window)
    again, _ = b.gpu(P, window=window)
    assert torch.equal(out, again), "the same call twice"


@TYPES
@pytest.mark.parametrize("nq,lens,Hq,Hkv,D,window", [
    ([1, 1, 400, 1, 1], [300, 1, 420, 450, 64], 8, 2, 64, 0),                   # whole sequences beside one prompt
    ([1, 500, 16, 1, 0, 17, 2], [2300, 900, 700, 1, 40, 1100, 0], 8, 2, 128, 0),    # 16 queries of 4 heads: the most
    ([300, 1, 3, 32, 33], [2600, 1900, 1200, 800, 33], 4, 2, 256, 500),
    ([1] * 150 + [300, 129, 1], [(31 * i) % 600 + 1 for i in range(150)] + [2100, 140, 9], 4, 1, 128, 0),
])
def test_single_tokens_beside_prompts(dtype, nq, lens, Hq, Hkv, D, window):
    """A batch most of whose sequences are far shorter than the longest runs on both kernels."""
    P = need_gpu()
    path = attention_path(P, sum(nq), len(nq), Hq, Hkv, D, max(nq), max(lens))
    assert path[0] == 2 and path[3] == 64 // (Hq // Hkv)
    b = Batch8(P, nq, lens, Hq, Hkv, D, 16, dtype)
    ws = P.kv8_attention_workspace(b.q.cuda(), b.cache, len(nq), max(nq), max(lens))
    first = None
    for _ in range(3):
        out, lse = b.gpu(P, window=window, workspace=ws)
        b.check(out, lse, window=window)
        first = out if first is None else first
        assert torch.equal(out, first) and int(ws[:P.KV8_COUNTER_BYTES].sum()) == 0


def test_long_sequence_and_workspace_of_many_calls():
    """70,000 keys; one workspace through calls of other shapes, back and forth."""
    P = need_gpu()
    a = Batch8(P, [1, 1], [70000, 300], 8, 2, 64, 128, F16, seed=4)
    b = Batch8(P, [40, 7], [600, 50], 8, 2, 64, 16, F16, seed=5)
    ws = P.kv8_attention_workspace(a.q.cuda(), a.cache, 2, 1, 70000)
    need = P.kv8_attention_workspace(b.q.cuda(), b.cache, 2, 40, 600).numel()
    if ws.numel() < need:
        ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        a.check(*a.gpu(P, cu_q=None, workspace=ws))
        b.check(*b.gpu(P, workspace=ws))
    assert int(ws[:P.KV8_COUNTER_BYTES].sum()) == 0


@TYPES
@pytest.mark.parametrize("nq,lens", [([1, 1], [70, 200]), ([80, 90], [100, 95]), ([3, 2], [40, 700])])
def test_rows_that_are_not_finite(dtype, nq, lens):
    """A key or value row of NaN reaches the queries that see it, whole rows of them, and no other; a query
    with an infinity or NaN itself alone. The sum of exponentials knows of keys only."""
    P = need_gpu()
    b = Batch8(P, nq, lens, 4, 2, 64, 16, dtype)
    gen = torch.Generator().manual_seed(3)
    k, v = rows(gen, 2, 2, 64, dtype), rows(gen, 2, 2, 64, dtype)
    k[0, 1, 5], v[1, 0, 7] = float("nan"), float("inf")
    b.put(P, 0, lens[0] - 1, k[:1], v[:1])       # head 1's key
    b.put(P, 1, lens[1] - 1, k[1:], v[1:])       # head 0's value
    b.q[0, 0, 3] = float("inf")
    if nq[0] > 2:
        b.q[0, 3, 3], b.q[1, 1, 0] = float("nan"), -float("inf")
    out, lse = (x.cpu().double().numpy() for x in b.gpu(P))
    want, wl, *_ = kv4_plain.attention(b.q.double().numpy(), b.k, b.v, nq, lens)
    want[np.isnan(want).any(-1)] = np.nan
    assert (np.isnan(out) == np.isnan(want)).all() and (np.isnan(lse) == np.isnan(wl)).all()
    assert np.isnan(want).any() and not np.isnan(want).all()
    fine = ~np.isnan(want)
    assert np.abs(out[fine] - want[fine]).max() < 0.05


@TYPES
@pytest.mark.parametrize("nq,L,at", [(1, 90, 3), (1, 90, 88), (90, 600, 3), (90, 600, 555)])
def test_value_rows_of_nan_at_no_weight(dtype, nq, L, at):
    """A value row of NaN makes the queries NaN that see it, though its weight is e^-200 and less of the sum's;
    where all queries see a step of keys, and where some do not."""
    P = need_gpu()
    b = Batch8(P, [nq], [L], 4, 2, 64, 16, dtype)
    b.q = (b.q.float().abs() + 1).to(dtype)
    tail = torch.from_numpy(b.k[0][at:]).to(dtype)          # from the row on: it again, and what follows
    tail[0] = -40.0
    v = torch.from_numpy(b.v[0][at:]).to(dtype)
    v[0] = float("nan")
    b.put(P, 0, at, tail, v)
    out, lse = b.gpu(P)
    want = np.arange(nq) + L - nq >= at
    assert (torch.isnan(out).cpu().numpy() == want[:, None, None]).all() and not torch.isnan(lse).any()


@TYPES
@pytest.mark.parametrize("nq,L,window", [(1, 90, 50), (5, 300, 0), (5, 300, 77), (150, 200, 0), (150, 400, 70), (1, 1700, 33)])
def test_what_a_query_does_not_see(dtype, nq, L, window):
    """What masked tokens hold moves no bit of a query's result: any bytes before the window and behind the keys, NaN among
    them, and, for queries that do not see them, keys and values at the type's end, NaN and infinities."""
    P = need_gpu()
    b = Batch8(P, [nq], [L], 4, 2, 64, 16, dtype, seed=6)
    out, lse = b.gpu(P, window=window)
    b.check(out, lse, window=window)
    blocks = b.cache[b.table[0].long()].cpu().numpy()          # pages of 16 tokens
    before = max(0, L - nq + 1 - window) if window else 0     # tokens that no query sees
    kp, vp = plain.places(64)
    for code in (0x7F, 0xFF, 0x7E):
        for t in [*range(before), *range(L, 16 * b.table.shape[1])]:
            blocks[t // 16, :, 0][:, kp[t % 16]] = code
            blocks[t // 16, :, 0][:, vp[t % 16]] = code
        for blk in range(blocks.shape[0]):
            mine = [t for t in range(16 * blk, 16 * blk + 16) if t < before or t >= L]
            tail = blocks[blk, :, 0, 64 * 32 + 8:64 * 32 + 12].copy().view(np.uint32)
            for t in mine:
                tail |= np.uint32(0x10001 << (t % 16))         # said not to be finite
            blocks[blk, :, 0, 64 * 32 + 8:64 * 32 + 12] = tail.view(np.uint8)
            if len(mine) == 16:
                blocks[blk, :, 0, 64 * 32:64 * 32 + 8] = 0x7F if code == 0x7F else 0xFF
        b.cache[b.table[0].long()] = torch.from_numpy(blocks).cuda()
        out2, lse2 = b.gpu(P, window=window)
        assert torch.equal(out, out2) and torch.equal(lse, lse2), code
    if (L - 1) % 16:
        # the last token, which only the last query sees: not finite (its block's scales stay), then large in either
        for x in (float("nan"), float("inf")):
            far = torch.full((1, 2, 64), x, dtype=dtype)
            b.put(P, 0, L - 1, far, far)
            out2, lse2 = b.gpu(P, window=window)
            assert torch.equal(out[:-1], out2[:-1]) and torch.equal(lse[:-1], lse2[:-1]), x
            assert out2[-1].isnan().all()


@pytest.mark.parametrize("dtype,q,k,v", [(F16, 4.0, 40.0, 1.0), (F16, 1e-3, 1e-2, 1e-4), (F16, 1.0, 1.0, 6e4 / 5), (F16, 0.0, 1.0, 1.0), (F16, 1e3, 1e-3, 1.0),
                                         (BF16, 1e4, 1e-4, 1e20), (BF16, 1e-20, 1e18, 1e-12), (BF16, 1e15, 1e-15, 1.0), (BF16, 1e30, 1e-14, 1e-16)])
def test_magnitudes(dtype, q, k, v):
    """Keys, values and queries far from 1; all weight on one key; none of it anywhere."""
    P = need_gpu()
    for nq, lens in (([1, 1], [400, 33]), ([70], [130])):
        b = Batch8(P, nq, lens, 4, 1, 128, 16, dtype, kscale=k, vscale=v)
        b.q = (b.q.float() * q).to(dtype)
        b.check(*b.gpu(P, scale=128 ** -0.5 * min(1.0, 1 / (q * k)) if q * k > 1e10 else None), scale=128 ** -0.5 * min(1.0, 1 / (q * k)) if q * k > 1e10 else None, what=(q, k, v))


def close(b, out, lse, window=0):
    """out and lse of Batch8 b against 64 bits, key by key, where blocks' scales lie far apart:
      logit j off by e_j = (D + 8) 2^-23 (4 sum |q k_j| scale + 4 |lse| + 256): its product's sum in fp32, and the references that
      it is taken from, which hold the exponent of a scale (120 at most) beside it;
      weight p_j s_j rounded to fp16: 2^-12, or 2^-25 below its normal range, where the largest p_j s_j stands at 2^8 or more:
      448 2^-33 of that for a key;
      sums of the keys in fp32; one rounding of the result."""
    q, scale, eps = b.q.double().numpy(), b.D ** -0.5, torch.finfo(b.dtype).eps / 2
    tiny = 2.0 ** -25 if b.dtype == F16 else 2.0 ** -134
    got, gl, at = out.double().cpu().numpy(), lse.double().cpu().numpy(), 0
    for s, (n, L) in enumerate(zip(b.nq, b.lens)):
        G, j = b.Hq // b.k[s].shape[1], np.arange(L)
        st = np.zeros((L, b.k[s].shape[1]))
        for blk in range(-(-L // 16)):
            top = np.abs(b.v[s][16 * blk:16 * blk + 16]).max((0, 2))
            st[16 * blk:16 * blk + 16] = np.maximum(2.0 ** np.ceil(np.log2(np.maximum(top, 2.0 ** -200) / 448) + 1), 2.0 ** -60)
        for i in range(n):
            pos = L - n + i
            see = (j <= pos) & ((j > pos - window) if window else True)
            for a in range(b.Hq):
                k, v, sv = b.k[s][see, a // G], b.v[s][see, a // G], st[see, a // G]
                w = k @ q[at + i, a] * scale
                m = w.max()
                p = np.exp(w - m)
                l = m + np.log(p.sum())
                p = p / p.sum()
                o = p @ v
                e = (b.D + 8) * 2.0 ** -23 * (4 * np.abs(k) @ np.abs(q[at + i, a]) * scale + 4 * abs(l) + 256)
                pe = p * np.minimum(np.expm1(np.minimum(e, 1)) * 2, 1e3)
                sums = len(w) * 2.0 ** -23
                tol = (p * (2.0 ** -12 + sums)) @ np.abs(v) + pe @ np.abs(v) + (pe.sum() + sums) * np.abs(o)
                tol = (tol + len(w) * 448 * 2.0 ** -33 * (p * sv).max()) * (1 + eps) + eps * np.abs(o) + tiny
                bad = ~(np.abs(got[at + i, a] - o) <= tol)
                assert not bad.any(), (s, i, a, got[at + i, a][bad][:4], o[bad][:4], tol[bad][:4])
                assert abs(gl[at + i, a] - l) <= pe.sum() + sums + 2.0 ** -22 * abs(l) + 2.0 ** -20
        at += n


@pytest.mark.parametrize("dtype,low,high", [(BF16, 2.0 ** -50, 2.0 ** 100), (BF16, 2.0 ** -20, 2.0 ** 20), (F16, 2.0 ** -14, 2.0 ** 12)])
@pytest.mark.parametrize("nq,L,window", [(1, 90, 0), (1, 3000, 0), (5, 700, 300), (90, 200, 0), (90, 2500, 1500)])
def test_value_blocks_of_all_scales(dtype, low, high, nq, L, window):
    """Value blocks whose scales run through the type's range over the keys, upwards, downwards and at random: waves and chunks of
    the keys whose references lie further apart than fp32's exponents reach; a large block without weight takes no bits from the others."""
    P = need_gpu()
    for order in ("up", "down", "random", "one"):
        b = Batch8(P, [nq], [L], 4, 2, 64, 16, dtype)
        f = torch.linspace(0, 1, -(-L // 16)).double()
        if order == "down":
            f = f.flip(0)
        elif order == "random":
            f = f[torch.randperm(len(f), generator=torch.Generator().manual_seed(L))]
        elif order == "one":
            f = (torch.arange(len(f)) == len(f) // 2).double()
        f = (low * (high / low) ** f).repeat_interleave(16)[:L]
        k = torch.from_numpy(b.k[0]).to(dtype)
        if order == "one":   # no weight on the large block
            b.q = (b.q.float().abs() + 1).to(dtype)
            k[f == f.max()] = -40.0
        b.put(P, 0, 0, k, (rows(torch.Generator().manual_seed(1), L, 2, 64, dtype).double() * f[:, None, None]).to(dtype))
        close(b, *b.gpu(P, window=window), window=window)


def test_scales_and_no_lse():
    P = need_gpu()
    for scale in (0.0, -0.3, 1.7):
        b = Batch8(P, [1, 4], [50, 300], 4, 4, 64, 32, F16)
        b.check(*b.gpu(P, scale=scale), scale=scale)
    out = b.gpu(P, scale=1.7)[0]
    assert torch.equal(out, b.gpu(P, scale=1.7, lse=None)[0])


def test_queries_of_the_other_type():
    """A cache holds no type: rows written in one, queries in the other."""
    P = need_gpu()
    for dtype, other in ((F16, BF16), (BF16, F16)):
        for nq in ([1, 1], [40, 60]):
            b = Batch8(P, nq, [100, 90], 4, 2, 64, 16, dtype)
            b.q, b.dtype = b.q.to(other), other
            b.check(*b.gpu(P))


@pytest.mark.parametrize("nq,lens", [([1, 1, 1], [100, 260, 64]), ([40, 100, 3], [100, 260, 64])])
def test_pages_that_do_not_exist(nq, lens):
    """Keys in a page whose number is outside the cache are not seen."""
    P = need_gpu()
    b = Batch8(P, nq, lens, 8, 2, 64, 16, F16)
    seen = [np.ones(L, bool) for L in lens]
    for s, at, number in ((0, 2, -1), (1, 0, len(b.cache)), (1, 9, -2 ** 31), (1, 16, 2 ** 31 - 1), (2, 3, -5)):
        b.table[s, at] = number
        seen[s][16 * at:16 * at + 16] = False
    b.cache[0].fill_(0x7F)   # (what a page number of no page must not be taken for)
    for s in range(3):
        for x in np.argwhere(b.table[s].numpy() == 0).flatten():
            seen[s][16 * x:16 * x + 16] = False
            b.table[s, x] = -1
    b.check(*b.gpu(P), seen=seen)


@pytest.mark.parametrize("nq,lens", [([2, 3], [40, 20]), ([70, 80], [90, 100])])
def test_rows_and_lengths_out_of_bounds(nq, lens):
    """Rows outside every sequence stay as they were; lengths are cut to the table and to max_kv_len, negative ones to 0; queries
    beyond max_q_len stay; what the arrays say beyond T is cut."""
    P = need_gpu()
    b = Batch8(P, nq, lens, 4, 2, 64, 16, F16)
    T = sum(nq)
    q = torch.randn((T + 5, 4, 64)).half()
    q[2:2 + T] = b.q
    cu = i32([2, 2 + nq[0], 2 + T])
    out = torch.full((T + 5, 4, 64), 3.0, dtype=F16, device="cuda")
    lse = torch.full((T + 5, 4), 3.0, device="cuda")
    P.kv8_attention(q.cuda(), b.cache, b.table.cuda(), i32([10 ** 9, -7]), cu_q=cu, max_q_len=max(nq), max_kv_len=lens[0], out=out, lse=lse)
    for x in (out, lse):
        assert (x[:2] == 3).all() and (x[2 + T:] == 3).all()
    keep, b.lens = b.lens, [lens[0], 0]
    b.k, b.v = ([x[:L] for x, L in zip(y, b.lens)] for y in (b.k, b.v))
    b.check(out[2:2 + T], lse[2:2 + T])
    b.lens = keep
    out = torch.full((T, 4, 64), 3.0, dtype=F16, device="cuda")
    full, _ = b.gpu(P)
    b.gpu(P, out=out, max_q_len=2)
    for s in (0, 1):
        a = int(b.cu[s])
        assert (out[a + 2:int(b.cu[s + 1])] == 3).all()
        torch.testing.assert_close(out[a:a + 2], full[a:a + 2], rtol=2e-3, atol=2e-3)
    out = b.gpu(P, cu_q=i32([0, nq[0], 10 ** 6]), max_q_len=T)[0]
    torch.testing.assert_close(out[:nq[0]], full[:nq[0]], rtol=2e-3, atol=2e-3)
    b.gpu(P, cu_q=i32([T, 3, -9]), max_q_len=T)
    torch.cuda.synchronize()


@pytest.mark.parametrize("nq", [1, 90])
def test_strided_queries_and_outputs(nq):
    P = need_gpu()
    Hq, Hkv, D = 8, 2, 128
    b = Batch8(P, [nq, nq], [100, 130], Hq, Hkv, D, 16, F16)
    qkv = torch.zeros((2 * nq, Hq + 2 * Hkv, D), dtype=F16, device="cuda")
    qkv[:, :Hq] = b.q.cuda()
    out = torch.zeros((Hq, 2 * nq, D), dtype=F16, device="cuda").transpose(0, 1)
    _, lse = b.gpu(P, q=qkv[:, :Hq], out=out)
    b.check(out, lse)


@pytest.mark.parametrize("nq,lens,D", [([1, 1], [1500, 40], 128), ([9, 2], [900, 1100], 256), ([200, 130], [300, 1500], 64)])
def test_out_in_the_place_of_q(nq, lens, D):
    P = need_gpu()
    b = Batch8(P, nq, lens, 8, 2, D, 16, F16)
    want, _ = b.gpu(P)
    q = b.q.cuda()
    got, _ = b.gpu(P, q=q, out=q)
    assert got is q and torch.equal(got, want)


def test_no_work_and_arguments():
    P = need_gpu()
    cache = P.kv8_cache(2, 2, 64, 16)
    empty, none, table = torch.zeros((0, 2, 64), dtype=F16, device="cuda"), i32([]), torch.zeros((0, 1), dtype=torch.int32, device="cuda")
    P.kv8_write(empty, empty, cache, table, none)
    assert P.kv8_read(cache, none)[0].shape == (0, 2, 64)
    assert P.kv8_attention(torch.zeros((0, 4, 64), dtype=F16, device="cuda"), cache, table, none).shape == (0, 4, 64)
    k, table, lens, r = torch.zeros((1, 2, 64), dtype=F16, device="cuda"), i32([[0, 1]]), i32([1]), P.Rope(64)
    for a, kw in (((k.cpu(), k, cache, table, lens), {}), ((k.float(), k, cache, table, lens), {}), ((k, k.bfloat16(), cache, table, lens), {}), ((k[:, :1], k, cache, table, lens), {}),
                  ((k, k, cache.view(-1), table, lens), {}), ((k, k, cache.int(), table, lens), {}), ((k, k, P.kv4_cache(2, 2, 128, 16), table, lens), {}),
                  ((k, k, cache, table[0], lens), {}), ((k, k, cache, table.long(), lens), {}), ((k, k, cache, table, lens.cpu()), {}), ((k, k, cache, table, i32([1, 2])), {}),
                  ((k, k, cache, table, lens), dict(cu_q=i32([0]))), ((k, k, cache, table, lens), dict(q=k)), ((k, k, cache, table, lens), dict(positions=lens)),
                  ((k, k, cache, table, lens), dict(rope=P.Rope(66))), ((k, k, cache, table, lens), dict(rope=r, q_out=k)), ((k, k, cache, table, lens), dict(rope=r, q=k.bfloat16())),
                  ((k, k, cache, table, lens), dict(rope=r, positions=i32([1, 2]))), ((k, k, cache, table, lens), dict(max_q_len=2)), ((k, k, cache, table, lens), dict(cu_q=i32([0, 1]), max_q_len=2 ** 32 + 1)),
                  ((k.expand(2, 2, 64), k.expand(2, 2, 64), cache, table, lens), {})):
        with pytest.raises((P.InvalidArgument, P.Unsupported)):
            P.kv8_write(*a, **kw)
    for over in (dict(max_kv_len=2 ** 32 + 20), dict(window=2 ** 32 + 1)):
        with pytest.raises(P.InvalidArgument, match="32-bit"):
            P.kv8_attention(k, cache, table, lens, **over)


# ------------------------------------------------------------------ as a program uses them

def test_steps_of_a_program():
    """A prompt, then token by token: rotated, written, attended over, on a captured graph that is replayed with new lengths and
    rows; every step against 64 bits on what the cache holds, and the eager calls on a cache of their own between them."""
    P = need_gpu()
    B, Hq, Hkv, D, page, dtype = 3, 8, 2, 128, 16, F16
    gen = torch.Generator().manual_seed(2)
    first, steps, per = [40, 15, 700], 5, 46
    table = torch.randperm(B * per, generator=gen).view(B, per).int()
    r = P.Rope(D, 10000.0)
    caches = [P.kv8_cache(B * per, Hkv, D, page) for _ in range(2)]
    T = sum(first)
    prompt = torch.randn((T, Hq + 2 * Hkv, D), generator=gen).to(dtype).cuda()
    for c in caches:
        P.kv8_write(prompt[:, Hq:Hq + Hkv], prompt[:, Hq + Hkv:], c, table.cuda(), i32(first), cu_q=i32(np.cumsum([0] + first)), rope=r)
    d = {"qkv": torch.zeros((B, Hq + 2 * Hkv, D), dtype=dtype, device="cuda"), "lens": i32([1] * B), "out": torch.zeros((B, Hq, D), dtype=dtype, device="cuda"),
         "lse": torch.zeros((B, Hq), device="cuda"), "q": torch.zeros((B, Hq, D), dtype=dtype, device="cuda"), "table": table.cuda()}
    ws = P.kv8_attention_workspace(d["q"], caches[0], B, 1, per * page)

    def step(cache, qkv, lens, q, out, lse, ws):
        P.kv8_write(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], cache, d["table"], lens, rope=r, q=qkv[:, :Hq], q_out=q)
        P.kv8_attention(q, cache, d["table"], lens, out=out, lse=lse, workspace=ws)

    warm = P.kv8_cache(B * per, Hkv, D, page)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, d["qkv"], d["lens"], d["q"], d["out"], d["lse"], ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(caches[0], d["qkv"], d["lens"], d["q"], d["out"], d["lse"], ws)
    for i in range(steps):
        qkv = (torch.randn((B, Hq + 2 * Hkv, D), generator=gen) * 2.0 ** i).to(dtype)   # (scales grow)
        lens = [n + i + 1 for n in first]
        d["qkv"].copy_(qkv)
        d["lens"].copy_(i32(lens))
        g.replay()
        torch.cuda.synchronize()
        b = Batch8.__new__(Batch8)
        b.nq, b.lens, b.dtype, b.D, b.Hq, b.q, b.table, b.cache = [1] * B, lens, dtype, D, Hq, d["q"].cpu(), table, caches[0]
        b.read()
        b.check(d["out"], d["lse"], what=f"step {i}")
        eager, lse, q = torch.zeros_like(d["out"]), torch.zeros_like(d["lse"]), torch.zeros_like(d["q"])
        step(caches[1], qkv.cuda(), i32(lens), q, eager, lse, None)
        assert torch.equal(eager, d["out"]) and torch.equal(lse, d["lse"]) and torch.equal(q, d["q"]) and torch.equal(*caches)


def test_two_streams_with_a_workspace_each():
    P = need_gpu()
    bs = [Batch8(P, [1, 1], [3000, 2000], 8, 2, 128, 64, F16, seed=s) for s in (1, 2)]
    args = [(b.q.cuda(), b.table.cuda(), i32(b.lens)) for b in bs]
    ws = [P.kv8_attention_workspace(a[0], b.cache, 2, 1, 3000) for a, b in zip(args, bs)]
    outs = [[torch.zeros_like(a[0]) for _ in range(10)] for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(10):
        for s in (0, 1):
            with torch.cuda.stream(streams[s]):
                P.kv8_attention(args[s][0], bs[s].cache, args[s][1], args[s][2], max_kv_len=3000, out=outs[s][i], workspace=ws[s])
    torch.cuda.synchronize()
    for s in (0, 1):
        want = bs[s].gpu(P, cu_q=None)
        bs[s].check(*want)
        assert all(torch.equal(o, want[0]) for o in outs[s])


@pytest.mark.parametrize("chunk", [1, 7, 20])
def test_decoder_layer_on_int4_weights(chunk):
    """A decoder layer as a program runs it, tokens by the piece: norm, fused q, k, v projection with int4 weights, rotation and
    cache, attention, output projection, residual and norm, gated feed-forward; the chain's parts against 64 bits."""
    P = need_gpu()
    Hq, Hkv, D, B, G, inter = 8, 2, 64, 2, 64, 768
    hidden, total = Hq * D, 20
    gen = torch.Generator("cuda").manual_seed(11)

    def layer(K, N):
        qw = torch.randint(-2 ** 31, 2 ** 31 - 1, (K // 8, N), generator=gen, device="cuda", dtype=torch.int64).int()
        return qw, (torch.rand((K // G, N), generator=gen, device="cuda") * 0.004 + 0.002).half()

    def linear(x, w):
        return P.gemm(x, w[0], w[1], None, fmt="gptq_sym", group_size=G)

    wqkv, wo, w13, w2 = layer(hidden, (Hq + 2 * Hkv) * D), layer(hidden, hidden), layer(hidden, 2 * inter), layer(inter, hidden)
    dense = [P.dequant(q, s, None, fmt="gptq_sym", group_size=G).double() for q, s in (wqkv, wo, w13, w2)]
    n1, n2 = (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).half(), (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).half()
    cache, r = P.kv8_cache(8, Hkv, D, 16), P.Rope(D, 10000.0)
    table = i32(torch.arange(8).view(B, 4))
    tokens = torch.randn((B, total, hidden), generator=gen, device="cuda").half()
    for at in range(0, total, chunk):
        n = min(chunk, total - at)
        x = tokens[:, at:at + n].reshape(B * n, hidden)
        res = x.clone()
        cu, lens = i32([i * n for i in range(B + 1)]), i32([at + n] * B)
        y1 = P.rms_norm(x, n1, 1e-5)
        qkv = linear(y1, wqkv).view(B * n, Hq + 2 * Hkv, D)
        before = qkv.clone()
        P.kv8_write(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], cache, table, lens, cu_q=cu, max_q_len=n, rope=r, q=qkv[:, :Hq])
        att = P.kv8_attention(qkv[:, :Hq], cache, table, lens, cu_q=cu, max_q_len=n)
        y2 = P.rms_norm(linear(att.view(B * n, hidden), wo), n2, 1e-5, residual=res)
        gu = linear(y2, w13)
        act = torch.empty((B * n, inter), dtype=F16, device="cuda")
        P.fused_silu_mul_interleaved_f16(gu, act, inter, B * n * inter)
        out = linear(act, w2)
    # the last piece, from its tokens, in 64 bits but for what the cache holds
    h = plain.norm(x, n1, 1e-5)[1]
    assert ((y1.double().cpu() - h).abs() <= h.abs() * (2.0 ** -11 + NORM_REL) + 2.0 ** -25).all()
    pos = np.tile(np.arange(at, at + n), B)
    qd = plain.rotate(before[:, :Hq].double().cpu().numpy(), pos, r.inv_freq.cpu().numpy(), False)[0]
    both = [plain.held(cache.cpu().numpy(), table.cpu().numpy(), b, total) for b in range(B)]
    o = kv4_plain.attention(qd, [x[0] for x in both], [x[1] for x in both], [n] * B, [total] * B)[0]
    kd = plain.rotate(before[:, Hq:Hq + Hkv].double().cpu().numpy(), pos, r.inv_freq.cpu().numpy(), False)[0]
    got = np.concatenate([x[0][total - n:] for x in both])
    assert np.linalg.norm(got - kd) < 2.0 ** -4 * np.linalg.norm(kd)
    want = x.double().cpu() + torch.from_numpy(o).view(B * n, hidden) @ dense[1].cpu()
    assert float((res.double().cpu() - want).norm() / want.norm()) < 2e-3
    y = want / torch.sqrt((want * want).mean(-1, keepdim=True) + 1e-5) * n2.double().cpu()
    g, u = (y @ dense[2].cpu()).split(inter, -1)
    final = (g * torch.sigmoid(g) * u) @ dense[3].cpu()
    assert float((out.double().cpu() - final).norm() / final.norm()) < 5e-3
