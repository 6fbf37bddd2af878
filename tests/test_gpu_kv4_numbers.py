"""The 4-bit key/value cache at the ends of its numbers' range: rows near the type's largest value, value
rows and queries many powers of two apart, infinities. Compared with 64 bits (kv4_plain.py)."""
import numpy as np
import pytest
import torch

import kv4_plain as plain
from test_gpu_kv4 import BF16, F16, Batch, need_gpu, rows, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_rows_across_the_whole_range(dtype, D):
    """Rows from the type's lowest to its largest value: zero point times scale passes the largest finite
    number, what a nibble holds does not."""
    P = need_gpu()
    most = torch.finfo(dtype).max
    gen = torch.Generator().manual_seed(D)
    T, H = 40, 2
    x = (torch.rand((2, T, H, D), generator=gen).double() * 2 - 1) * most
    x[..., 0] = -most                                      # the range that a row spans: from the lowest value
    x[..., 1] *= torch.rand((2, T, H), generator=gen).double()
    x[:, ::2, :, 2] = most                                 # to the largest one, or less
    x[:, ::4, :, 3:] = 0
    x[:, 1::4, :, 3:20] *= 1e-6
    k, v = x.float().to(dtype)
    cache = P.kv4_cache(3, H, D, 16)
    slots = torch.randperm(48, generator=gen)[:T].int().cuda()
    P.kv4_write(k.cuda(), v.cuda(), cache, slots)
    for want, got in zip((k, v), P.kv4_read(cache, slots, dtype)):
        want = plain.rounded(plain.quantise(want)[3], dtype)
        assert (want == 0).any() and (want > 0).any() and (want < 0).any()
        assert same(got, want)


def close(b, out, lse, window=0, scale=None, but=()):
    """out and lse of Batch b against 64 bits, every query row (those in `but` aside) within what the operator's
    definition allows, key by key:
      logit j off by e_j = (D + 8) 2^-23 (4 sum |q k_j| scale + 4 |lse| + 16): its product's sum in fp32, and the
      references that it is taken from, which hold the logarithm of a value scale beside the logit;
      weight p_j s_j rounded to fp16: 2^-11, or 2^-25 below its normal range, where the largest p_j s_j
      stands at 2^7 or more: 15 2^-32 of that for a key, (n - zero) being 15 at most;
      sums of the keys in fp32; one rounding of the result.
    So a value row counts by p_j s_j: one of any scale that has no weight leaves the result alone. Scales below 2^-60
    count as 2^-60 there. s_j is at most a 14th of what the row spans (15 steps, one lost to rounding)."""
    q = b.q.double().numpy()
    scale = b.D ** -0.5 if scale is None else scale
    eps = torch.finfo(b.dtype).eps / 2
    tiny = 2.0 ** -25 if b.dtype == F16 else 2.0 ** -134
    got, gl, at = out.double().cpu().numpy(), lse.double().cpu().numpy(), 0
    for s, (n, L) in enumerate(zip(b.nq, b.lens)):
        G = b.Hq // b.k[s].shape[1]
        j = np.arange(L)
        steps = np.maximum((b.v[s].max(-1).clip(min=0) - b.v[s].min(-1).clip(max=0)) / 14, 2.0 ** -60)   # [L, Hkv]
        for i in range(n):
            pos = L - n + i
            see = (j <= pos) & ((j > pos - window) if window else True)
            for a in range(b.Hq):
                if (at + i, a) in but:
                    continue
                k, v, st = b.k[s][see, a // G], b.v[s][see, a // G], steps[see, a // G]
                w = k @ q[at + i, a] * scale
                m = w.max()
                p = np.exp(w - m)
                l = m + np.log(p.sum())
                p = p / p.sum()
                o = p @ v
                e = (b.D + 8) * 2.0 ** -23 * (4 * np.abs(k) @ np.abs(q[at + i, a]) * abs(scale) + 4 * abs(l) + 16)
                # (p_j off by e^e_j - 1: where that is large, all of it)
                pe = p * np.minimum(np.expm1(np.minimum(e, 1)) * 2, 1e3)
                sums = len(w) * 2.0 ** -23
                tol = (p * (2.0 ** -11 + sums)) @ np.abs(v) + pe @ np.abs(v) + (pe.sum() + sums) * np.abs(o)
                tol = (tol + len(w) * 15 * 2.0 ** -32 * (p * st).max()) * (1 + eps) + eps * np.abs(o) + tiny
                bad = ~(np.abs(got[at + i, a] - o) <= tol)
                assert not bad.any(), (s, i, a, got[at + i, a][bad][:4], o[bad][:4], tol[bad][:4])
                lt = pe.sum() + sums + 2.0 ** -22 * abs(l) + 2.0 ** -20
                assert abs(gl[at + i, a] - l) <= lt, (s, i, a, gl[at + i, a], l, lt)
        at += n


def put_row(P, b, s, t, k, v):
    """Token t of sequence s anew: k, v [Hkv, D]."""
    page = b.cache.shape[2] * 16
    slot = (b.table[s, t // page:t // page + 1] * page + t % page).cuda()
    P.kv4_write(k[None].cuda(), v[None].cuda(), b.cache, slot)
    b.k[s][t], b.v[s][t] = plain.quantise(k)[3], plain.quantise(v)[3]


@pytest.mark.parametrize("dtype,base,ratio", [(BF16, 1.0, 2.0 ** 20), (BF16, 1.0, 2.0 ** 32), (BF16, 1.0, 2.0 ** 100), (BF16, 2.0 ** -50, 2.0 ** 150),
                                              (F16, 2.0 ** -8, 2.0 ** 18), (F16, 2.0 ** -11, 2.0 ** 22), (F16, 2.0 ** -14, 2.0 ** 26)])
@pytest.mark.parametrize("nq,L,window", [(1, 90, 0), (1, 3000, 0), (5, 700, 400), (90, 200, 0), (90, 2500, 1500)])
def test_a_large_value_row_of_no_weight(dtype, base, ratio, nq, L, window):
    """A value row far larger than the others that no query gives weight to: the others' weights keep their bits, on
    either kernel, whether the row comes first or last, in a step of keys that all see or some."""
    P = need_gpu()
    for at in (L // 3 + 3, L - nq):
        b = Batch(P, [nq], [L], 4, 2, 64, 16, dtype, vscale=base)
        b.q = (b.q.float().abs() + 1).to(dtype)
        big = rows(torch.Generator().manual_seed(at), 1, 2, 64, dtype)[0].float()
        put_row(P, b, 0, at, torch.full((2, 64), -40.0, dtype=dtype), (big * (base * ratio / 2)).to(dtype))
        close(b, *b.gpu(P, window=window), window=window)


@pytest.mark.parametrize("dtype,low,high", [(BF16, 2.0 ** -55, 2.0 ** 100), (BF16, 2.0 ** -20, 2.0 ** 20), (F16, 2.0 ** -14, 2.0 ** 12)])
@pytest.mark.parametrize("nq,L", [(1, 90), (1, 3000), (5, 700), (90, 200), (90, 2500)])
def test_value_rows_of_all_scales(dtype, low, high, nq, L):
    """Value rows whose scales run through the type's range over the keys, upwards, downwards and at random:
    waves and chunks of the keys whose references lie further apart than fp32's exponents reach."""
    P = need_gpu()
    for order in ("up", "down", "random"):
        b = Batch(P, [nq], [L], 4, 2, 64, 16, dtype)
        f = torch.linspace(0, 1, L).double()
        if order == "down":
            f = f.flip(0)
        elif order == "random":
            f = f[torch.randperm(L, generator=torch.Generator().manual_seed(L))]
        f = low * (high / low) ** f
        v = rows(torch.Generator().manual_seed(1), L, 2, 64, dtype).double() * f[:, None, None]
        t = torch.arange(L)
        slots = (b.table[0, t // 16] * 16 + t % 16).int().cuda()
        k16, _ = P.kv4_read(b.cache, slots, dtype)
        P.kv4_write(k16, v.to(dtype).cuda(), b.cache, slots)
        b.k[0], b.v[0] = plain.quantise(k16.cpu())[3], plain.quantise(v.to(dtype))[3]
        close(b, *b.gpu(P))


@pytest.mark.parametrize("q,k,scale", [(2.0 ** 114, 2.0 ** -116, 0.125), (2.0 ** 120, 2.0 ** -122, 0.125), (1.5 * 2.0 ** 125, 2.0 ** -128, 0.125),
                                       (2.0 ** 122, 1.0, 2.0 ** -124), (2.0 ** 60, 2.0 ** -120, 2.0 ** 60), (2.0 ** -110, 2.0 ** 108, 0.125),
                                       (2.0 ** -125, 2.0 ** 100, 2.0 ** 24), (0.25, 2.0 ** 12, 2.0 ** -14), (1.0, 2.0 ** -40, 2.0 ** 38)])
@pytest.mark.parametrize("nq,L", [(1, 90), (1, 1500), (90, 200)])
def test_queries_of_any_magnitude(q, k, scale, nq, L):
    """bfloat16 queries up to the type's end, whose logits are ordinary numbers."""
    P = need_gpu()
    b = Batch(P, [nq], [L], 4, 2, 64, 16, BF16, kscale=k)
    b.q = (b.q.double().clamp(-1.9, 1.9) * q).to(BF16)
    assert torch.isfinite(b.q).all() and torch.isfinite(torch.tensor(b.k[0])).all()
    out, lse = b.gpu(P, scale=scale)
    assert torch.isfinite(out).all()
    close(b, out, lse, scale=scale)


@pytest.mark.parametrize("nq,L", [(1, 90), (90, 200)])
def test_keys_orthogonal_to_large_queries(nq, L):
    """q . k = 0 exactly, beside a factor that passes fp32's range: a logit of 0."""
    P = need_gpu()
    b = Batch(P, [nq], [L], 4, 2, 64, 16, BF16)
    b.q[:] = 0
    b.q[..., 0] = 2.0 ** 126
    t = torch.arange(L)
    slots = (b.table[0, t // 16] * 16 + t % 16).int().cuda()
    k = rows(torch.Generator().manual_seed(2), L, 2, 64, BF16).float() * 2.0 ** 110
    k[..., 0] = 0
    _, v16 = P.kv4_read(b.cache, slots, BF16)
    P.kv4_write(k.to(BF16).cuda(), v16, b.cache, slots)
    b.k[0], b.v[0] = plain.quantise(k.to(BF16))[3], plain.quantise(v16.cpu())[3]
    close(b, *b.gpu(P))


@pytest.mark.parametrize("far", [2.0 ** 30, 2.0 ** 60, 2.0 ** 115, 2.0 ** -30, 2.0 ** -100])
@pytest.mark.parametrize("nq,L,Hq", [(1, 90, 8), (1, 1500, 24), (5, 300, 8), (90, 200, 4)])
def test_queries_of_many_magnitudes(far, nq, L, Hq):
    """One query row many powers of two larger or smaller than its neighbours costs them no bits."""
    P = need_gpu()
    b = Batch(P, [nq], [L], Hq, 2, 64, 16, BF16)
    odd = (nq // 2, 1)
    b.q[odd] = (b.q[odd].double() * far).to(BF16)
    close(b, *b.gpu(P), but=(odd,) if far > 1 else ())   # (its own logits are far beyond what exp tells apart)
    # and the others' results do not depend on it
    first = b.gpu(P)
    b.q[odd] = b.q[odd] * 0 + 1
    second = b.gpu(P)
    keep = torch.ones(first[1].shape, dtype=torch.bool)
    keep[odd] = False
    tol = 2.0 ** -7 * first[0].double().abs().max()
    assert float((first[0].double() - second[0].double()).abs()[keep.cuda()].max()) <= tol


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("nq,L", [(1, 1), (1, 90), (1, 1500), (90, 200)])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_queries_are_nan(dtype, nq, L, sign):
    """An infinite query has no softmax: its logits are infinities of either sign or NaN. Also where all of them
    are -infinity, which is not a row that sees nothing."""
    P = need_gpu()
    b = Batch(P, [nq], [L], 4, 2, 64, 16, dtype)
    t = torch.arange(L)
    slots = (b.table[0, t // 16] * 16 + t % 16).int().cuda()
    k = rows(torch.Generator().manual_seed(2), L, 2, 64, dtype)
    k[..., 7] = -3.0
    _, v16 = P.kv4_read(b.cache, slots, dtype)
    P.kv4_write(k.cuda(), v16, b.cache, slots)
    b.k[0], b.v[0] = plain.quantise(k)[3], plain.quantise(v16.cpu())[3]
    b.q[nq // 2, 1, 7] = sign * float("inf")
    out, lse = b.gpu(P)
    assert torch.isnan(out[nq // 2, 1]).all() and torch.isnan(lse[nq // 2, 1])
    assert int(torch.isnan(out).sum()) == 64
    close(b, out, lse, but=((nq // 2, 1),))


@pytest.mark.parametrize("dtype,k,v,scale", [(BF16, 2.0 ** 120, 1.0, 2.0 ** -122), (BF16, 1.0, 2.0 ** 125, 0.125), (F16, 300.0, 1.0, 2.0 ** -9),
                                             (F16, 1.0, 1.2e4, 0.125), (F16, 2.0 ** -12, 2.0 ** -12, 2.0 ** 9), (BF16, 2.0 ** -124, 2.0 ** -50, 2.0 ** 121)])
@pytest.mark.parametrize("nq,L", [(1, 90), (1, 1500), (90, 200)])
def test_keys_and_values_at_the_ends(dtype, k, v, scale, nq, L):
    P = need_gpu()
    b = Batch(P, [nq], [L], 4, 2, 64, 16, dtype, kscale=k, vscale=v)
    assert np.isfinite(b.k[0]).all() and np.isfinite(b.v[0]).all()
    out, lse = b.gpu(P, scale=scale)
    assert torch.isfinite(out).all()
    close(b, out, lse, scale=scale)
