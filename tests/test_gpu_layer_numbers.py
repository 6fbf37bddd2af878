"""Norm and rotary positions where a rounding or fp32's range decides: numbers next to the middle of two of e4m3, an eps that
outweighs rows, rows of several waves that are zero or not finite, magnitudes that take products past fp32."""
import numpy as np
import pytest
import torch

import kv8_plain as plain
from test_gpu_layer import BF16, E4M3, F16, NORM_REL, TYPES, need_gpu, rounded_once

pytestmark = pytest.mark.gpu


def near_the_middle(dtype):
    """[groups, 32] positive weights, the first of each the largest m, the others next to the middle between two numbers of e4m3
    times m / 448: 21 is one, and 21 / 448 is 3 / 64, so 3 m / 64 of any m that holds it is one but for the scale's rounding."""
    bits = 11 if dtype == F16 else 8
    first = np.arange(1, 2 ** bits // 3, 2, dtype=np.float64)
    powers = 2.0 ** np.concatenate((np.arange(0, -11, -1), np.arange(0, -11, -1), np.arange(0, -9, -1)))   # (21 2^4 is the largest middle)
    return torch.from_numpy(np.concatenate((first[:, None], 0.75 * first[:, None] * powers), 1)).to(dtype)


@TYPES
def test_8bit_next_to_the_middle(dtype):
    """Rows of 1 and -1 and no eps: y is the weight itself, exactly. Each number is the fp32 quotient of it and the scale (itself an
    fp32 quotient) rounded to nearest even, bit for bit: once a group, once a row."""
    P = need_gpu()
    w = near_the_middle(dtype)
    assert torch.equal(w[:, 1].double() * 4, w[:, 0].double() * 3)
    K = w.numel()
    x = torch.where(torch.rand((3, K), generator=torch.Generator().manual_seed(0)) < 0.5, -1.0, 1.0).to(dtype)
    assert torch.equal(P.rms_norm(x.cuda(), w.flatten().cuda(), 0.0).cpu(), x * w.flatten())
    scale = w[:, 0].float() / 448.0
    want = (w.float() / scale[:, None]).to(E4M3).float().flatten()
    q, s = P.rms_norm_8bit(x.cuda(), w.flatten().cuda(), 0.0, group=32)
    assert torch.equal(s.cpu(), scale.expand(3, -1)) and torch.equal(q.float().cpu(), x.float() * want)
    for i in range(0, len(w), 7):
        row = torch.cat((w[i], w[i, 1:20]))   # (of no width that a group has)
        q, s = P.rms_norm_8bit(x[:, :51].contiguous().cuda(), row.cuda(), 0.0)
        assert (s.cpu() == scale[i]).all() and torch.equal(q.float().cpu(), x[:, :51].float() * torch.cat((want[32 * i:32 * i + 32], want[32 * i + 1:32 * i + 20])))


@pytest.mark.parametrize("K", [64, 3000])
def test_8bit_beyond_fp32(K):
    """y beyond fp32 in a group: its scale is infinite, what is finite of it 0, what is not NaN; its neighbours are as ever."""
    P = need_gpu()
    x = torch.ones((2, K), dtype=BF16)
    x[0, 40] = 2.0 ** 20                        # y of about sqrt(K) 2^126 there, and beside it about 2^-20
    w = torch.ones(K, dtype=BF16)
    w[40] = 2.0 ** 127
    w = w.cuda()
    for group in (32, 0) if K == 64 else (0,):
        q, s = P.rms_norm_8bit(x.cuda(), w, 1e-6, group=group)
        q, s = q.float().cpu(), s.cpu()
        at = 40 // (group or K)
        part = slice(at * (group or K), (at + 1) * (group or K))
        assert s[0, at] == float("inf") and torch.isfinite(s[1]).all()
        assert q[0, 40].isnan() and not q[0, part].nan_to_num(0).any() and int(q[0].isnan().sum()) == 1
        if group:
            y = plain.norm(x, w, 1e-6)[1][0, :32]
            assert torch.isfinite(s[0, 0]) and ((q[0, :32].double() * s[0, 0] - y).abs() <= y.abs() * (2.0 ** -4 + NORM_REL + 2.0 ** -22)).all()


@TYPES
@pytest.mark.parametrize("K", [700, 2100, 5003, 20000, 40000, 65536])
def test_8bit_rows_without_a_scale_of_their_own(dtype, K):
    """Rows of several waves that are zero, infinite or NaN, a scale a row, beside ordinary ones: many of each."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(K)
    T = 300 if K < 30000 else 60
    x = torch.randn((T, K), generator=gen).to(dtype)
    w = (1 + 0.3 * torch.randn(K, generator=gen)).to(dtype)
    want, ws = (y[::6] for y in P.rms_norm_8bit(x.cuda(), w.cuda()))   # (as many rows: how a row is split may depend on that)
    x[1::6] = 0
    x[2::6, K - 1] = float("inf")
    x[3::6, K // 3] = float("nan")
    x[4::6] = -float("inf")
    for _ in range(3):
        q, s = P.rms_norm_8bit(x.cuda(), w.cuda())
        q, s = q.float().cpu(), s.cpu()
        assert torch.equal(q[::6], want.float().cpu()) and torch.equal(s[::6], ws.cpu()) and torch.isfinite(ws).all()
        assert (s[1::6] == 2.0 ** -100).all() and not q[1::6].any()
        for first in (2, 3, 4):
            assert s[first::6].isnan().all() and q[first::6].isnan().all()


@pytest.mark.parametrize("K", [8, 300, 5000])
@pytest.mark.parametrize("eps", [1e-3, 1.0, 2.0 ** 26, 2.0 ** 30, 1e20, 3e38])
def test_norm_of_small_rows_under_a_large_eps(eps, K):
    """Rows whose squares fp32 does not hold beside an eps that is all of the root: y = h / sqrt(eps), which bf16 holds."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(K)
    x = torch.stack([(torch.rand(K, generator=gen) + 0.4) * 2.0 ** e for e in (-60, -50, -47, -40, 0, 50, 62)]).bfloat16()
    w = (torch.rand(K, generator=gen) + 0.5).bfloat16()
    y = plain.norm(x, w, eps)[1]
    rounded_once(P.rms_norm(x.cuda(), w.cuda(), eps), y, BF16, NORM_REL)


@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("magnitude", [1.0, 1.5, -2.0, 1000.0, 3e38, 1e-3])
def test_rope_of_the_largest_values(dtype, interleaved, magnitude):
    """Pairs at the type's end, whose products with the magnitude pass fp32 and whose sums may be anything from 0 to beyond the
    type: the formula's value, to the largest finite one beyond that, and never NaN."""
    P = need_gpu()
    T, H, D = 200, 2, 64
    gen = torch.Generator().manual_seed(3)
    most = torch.finfo(dtype).max
    x = torch.where(torch.rand((T, H, D), generator=gen) < 0.5, -most, most)
    x[:, 1] *= torch.rand((T, D), generator=gen)
    x = x.to(dtype).clamp(-most, most)
    positions = torch.randint(-3000, 3000, (T,), generator=gen).int()
    r = P.Rope(D, 10000.0, interleaved=interleaved, magnitude=magnitude)
    got = P.rope(x.cuda(), positions.cuda(), r, q_out=torch.empty_like(x.cuda())).double().cpu()
    want, reach = plain.rotate(x.double().numpy(), positions.numpy(), r.inv_freq.cpu().numpy(), interleaved, float(np.float32(magnitude)))
    # four fp32 roundings of |a| + |b|, and the angle's in fp64, 2^-50 of it; then one to the type, below its largest value
    want, off = torch.from_numpy(want), torch.from_numpy(reach * (4 * 2.0 ** -24 + 3000 * 2.0 ** -50))
    eps = torch.finfo(dtype).eps / 2
    low, high = (want - off).clamp(-most, most), (want + off).clamp(-most, most)
    tiny = 2.0 ** -25 if dtype == F16 else 2.0 ** -134
    assert torch.isfinite(got).all()
    assert (got >= low - low.abs() * eps - tiny).all() and (got <= high + high.abs() * eps + tiny).all()
    # the same bits where rows are appended to a cache
    cache, out = P.kv8_cache(T // 16 + 1, 1, D, 16), torch.empty_like(x.cuda())
    k = torch.zeros((T, 1, D), dtype=dtype, device="cuda")
    table = torch.arange(T // 16 + 1, dtype=torch.int32, device="cuda")[None]
    P.kv8_write(k, k, cache, table, torch.tensor([T], dtype=torch.int32, device="cuda"), cu_q=torch.tensor([0, T], dtype=torch.int32, device="cuda"),
                rope=r, positions=positions.cuda(), q=x.cuda(), q_out=out)
    assert torch.equal(out.double().cpu(), got)
