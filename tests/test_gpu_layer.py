"""Norm and rotary positions on the GPU against 64 bits (kv8_plain.py)."""
import numpy as np
import pytest
import torch

import kv8_plain as plain
from helpers import pkg

pytestmark = pytest.mark.gpu
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
TYPES = pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])


def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return pkg()


def tiny(dtype):
    """Half a step of the type's smallest numbers."""
    return 2.0 ** -25 if dtype == F16 else 2.0 ** -134


def rounded_once(got, want, dtype, relative, absolute=0.0, what=""):
    """got is `want`, computed in fp32 within `relative` of itself and `absolute`, and rounded to its type."""
    got, want = got.double().cpu(), torch.as_tensor(want)
    eps = torch.finfo(dtype).eps / 2
    off = want.abs() * relative + absolute
    tol = off + (want.abs() + off) * eps + tiny(dtype)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, torch.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


# fp32: h one rounding, its square and the sum of at most 64 of a thread and a tree of ten levels (each term passes
# at most 75 additions), division, eps, root (2 units) and two products: under 100 roundings of 2^-24, half of the
# sum's counting
NORM_REL = 100 * 2.0 ** -24


def normed(P, x, w, eps, residual=None, **over):
    """(y, h) of rms_norm with new outputs."""
    total = None if residual is None else torch.full_like(residual, 9.0)
    out = P.rms_norm(x, w, eps, residual=residual, residual_out=total, **over)
    return out, total


@TYPES
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (5, 8), (33, 128), (2, 129), (17, 255), (3, 256), (4, 500), (4, 513), (9, 1024), (2, 1031),
                                 (3, 2048), (2, 2500), (5, 4096), (2, 4101), (1, 8192), (2, 9001), (1, 16384), (2, 16391), (1, 32768), (1, 40000),
                                 (2, 65535), (1, 65536), (700, 96)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(dtype, T, K, residual):
    P = need_gpu()
    gen = torch.Generator().manual_seed(T * 100 + K)
    x = torch.randn((T, K), generator=gen).to(dtype).cuda()
    r = (torch.randn((T, K), generator=gen) * 5).to(dtype).cuda() if residual else None
    w = (1 + 0.3 * torch.randn(K, generator=gen)).to(dtype).cuda()
    out, total = normed(P, x, w, 1e-5, r)
    h, y = plain.norm(x, w, 1e-5, r)
    rounded_once(out, y, dtype, NORM_REL)
    if residual:
        rounded_once(total, h, dtype, 2.0 ** -24)
    q, s = P.rms_norm_8bit(x, w, 1e-5, residual=r, residual_out=total)
    assert s.shape == (T, 1)
    check_8bit(q, s, y, 0)


@TYPES
@pytest.mark.parametrize("T,K,group", [(2100, 513, 0), (1100, 1031, 0), (600, 4096, 128), (300, 5003, 0), (333, 4608, 512), (130, 8191, 0)])
def test_norm_of_many_rows(dtype, T, K, group):
    """Rows that run with more elements a thread than a few rows of their width; in place."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(T + K)
    x = torch.randn((T, K), generator=gen).to(dtype).cuda()
    r = (torch.randn((T, K), generator=gen) * 5).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(K, generator=gen)).to(dtype).cuda()
    h, y = plain.norm(x, w, 1e-5, r)
    q, s = P.rms_norm_8bit(x, w, 1e-5, group=group, residual=r, residual_out=torch.empty_like(r))
    check_8bit(q, s, y, group)
    assert P.rms_norm(x, w, 1e-5, residual=r, out=x) is x
    rounded_once(x, y, dtype, NORM_REL)
    rounded_once(r, h, dtype, 2.0 ** -24)


def check_8bit(q, s, y, group):
    """Scales are max |y| / 448 (2^-100 at least) within the norm's roundings and two more; numbers are half a step
    of e4m3 from y / scale, which is off by as much and three more."""
    y = y.reshape(*y.shape[:-1], -1, group or y.shape[-1])
    want = (y.abs().amax(-1) / 448).clamp(min=2.0 ** -100)
    s, q = s.double().cpu(), q.cpu().double().reshape(y.shape)
    assert ((s - want).abs() <= want * (NORM_REL + 2.0 ** -22)).all()
    x = y / s[..., None]
    off = x.abs() * (NORM_REL + 2.0 ** -22)
    assert ((q - x).abs() <= off + torch.maximum((x.abs() + off) * 2.0 ** -4, torch.tensor(2.0 ** -10))).all()
    assert (q.abs().amax(-1) == torch.where(want > 2.0 ** -100, 448.0, q.abs().amax(-1))).all()


@TYPES
@pytest.mark.parametrize("group", [32, 64, 128, 256, 512])
@pytest.mark.parametrize("K", [32, 128, 256, 512, 1536, 4096, 11264, 66560 - 1024])
def test_norm_8bit_groups(dtype, group, K):
    P = need_gpu()
    if K % group:
        with pytest.raises(P.InvalidArgument):
            P.rms_norm_8bit(torch.zeros((1, K), dtype=dtype, device="cuda"), torch.zeros(K, dtype=dtype, device="cuda"), group=group)
        return
    gen = torch.Generator().manual_seed(K + group)
    x = (torch.randn((5, K), generator=gen) * torch.randn((5, K), generator=gen).exp()).to(dtype).cuda()
    x[3, :group] = 0
    w = torch.randn(K, generator=gen).to(dtype).cuda()
    q, s = P.rms_norm_8bit(x, w, 1e-6, group=group)
    assert q.dtype == E4M3 and s.shape == (5, K // group)
    check_8bit(q, s, plain.norm(x, w, 1e-6)[1], group)
    assert s[3, 0] == 2.0 ** -100 and not q[3, :group].float().any()


@TYPES
@pytest.mark.parametrize("T,H,K", [(3, 5, 128), (40, 3, 64), (2, 2, 200), (2, 3, 4096)])
def test_norm_strides(dtype, T, H, K):
    """Heads out of a fused projection; rows of odd strides at odd addresses; results into wider rows."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(K)
    wide = torch.randn((T, H + 3, K), generator=gen).to(dtype).cuda()
    x = wide[:, 1:H + 1]
    w = torch.randn(K, generator=gen).to(dtype).cuda()
    want = plain.norm(x, w, 1e-6)[1]
    rounded_once(P.rms_norm(x, w), want, dtype, NORM_REL)
    odd = torch.zeros(T * H * (K + 3) + 1, dtype=dtype, device="cuda")[1:].view(T, H, K + 3)[..., 1:K + 1]
    odd.copy_(x)
    out = torch.full((H, T, K + 5), 3.0, dtype=dtype, device="cuda")
    rounded_once(P.rms_norm(odd, w, out=out.transpose(0, 1)[..., 2:K + 2]).cpu(), want, dtype, NORM_REL)
    assert (out[..., :2] == 3).all() and (out[..., K + 2:] == 3).all()
    q8 = torch.full((T, H, K + 3), 7, dtype=torch.uint8, device="cuda").view(E4M3)
    q, s = P.rms_norm_8bit(odd, w, out=q8[..., 1:K + 1])
    check_8bit(q, s, want, 0)
    assert (q8.view(torch.uint8)[..., 0] == 7).all() and (q8.view(torch.uint8)[..., K + 1:] == 7).all()
    r = torch.randn((T, H, K), generator=gen).to(dtype).cuda()
    h, y = plain.norm(x, w, 1e-6, r)
    out, total = normed(P, x, w, 1e-6, r)
    rounded_once(out, y, dtype, NORM_REL)
    rounded_once(total, h, dtype, 2.0 ** -24)


@TYPES
@pytest.mark.parametrize("K", [100, 2048, 9000])
def test_norm_in_place(dtype, K):
    """The residual takes the sum in place; x and the result may share a buffer; broadcast rows are read."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(K)
    x, r = (torch.randn((6, K), generator=gen).to(dtype).cuda() for _ in range(2))
    w = torch.randn(K, generator=gen).to(dtype).cuda()
    want, total = normed(P, x, w, 1e-6, r)
    a, b = x.clone(), r.clone()
    assert P.rms_norm(a, w, residual=b, out=a) is a
    assert torch.equal(a, want) and torch.equal(b, total)
    a, b = x.clone(), r.clone()
    P.rms_norm(a, w, residual=b, residual_out=a)   # the sum into x's place
    assert torch.equal(a, total) and torch.equal(b, r)
    one = x[:1].expand(6, K)
    assert torch.equal(P.rms_norm(one, w), P.rms_norm(one.contiguous(), w))


@TYPES
@pytest.mark.parametrize("K", [8, 120, 300, 2000, 5000, 20000])
def test_norm_of_any_magnitude(dtype, K):
    """Rows whose squares fp32 does not hold, upwards and downwards, beside ordinary ones; zeros; eps 0."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(K)
    powers = [-14, -10, 0, 14] if dtype == F16 else [-125, -100, -60, -50, -40, 0, 50, 62, 64, 100, 126]
    x = torch.stack([(torch.rand(K, generator=gen) + 0.4) * 2.0 ** e for e in powers]).to(dtype).cuda()
    w = torch.randn(K, generator=gen).to(dtype).cuda()
    for eps in (0.0, 1e-6, 1e-30):
        y = plain.norm(x, w, eps)[1]
        # (an eps of 1e-30 beside rows of 2^-125: what is far below eps has a y near 0)
        rounded_once(P.rms_norm(x, w, eps), y, dtype, NORM_REL, 2.0 ** -100 if dtype == BF16 else 0.0, eps)
        q, s = P.rms_norm_8bit(x, w, eps)
        keep = y.abs().amax(-1) > 2.0 ** -80
        check_8bit(q[keep.cuda()].contiguous(), s[keep.cuda()], y[keep], 0)
    z = torch.zeros((2, K), dtype=dtype, device="cuda")
    assert not P.rms_norm(z, w, 1e-6).any()
    q, s = P.rms_norm_8bit(z, w, 1e-6)
    assert not q.float().any() and (s == 2.0 ** -100).all()


@TYPES
@pytest.mark.parametrize("K", [64, 1000, 4096])
def test_norm_of_rows_that_are_not_finite(dtype, K):
    """A row with a NaN is NaN throughout; with an infinity NaN there and 0 elsewhere; its neighbours are as ever."""
    P = need_gpu()
    gen = torch.Generator().manual_seed(K)
    x = torch.randn((5, K), generator=gen).to(dtype).cuda()
    w = torch.randn(K, generator=gen).to(dtype).cuda()
    want = P.rms_norm(x, w)
    x[1, K // 2], x[3, 5] = float("nan"), -float("inf")
    got = P.rms_norm(x, w)
    assert torch.equal(got[[0, 2, 4]], want[[0, 2, 4]]) and got[1].isnan().all()
    assert got[3].isnan().nonzero().flatten().tolist() == [5] and not got[3].nan_to_num(0).any()
    q, s = P.rms_norm_8bit(x, w, group=32 if K % 32 == 0 else 0)
    assert s[1].isnan().all() and s[3, 0].isnan() and not s[[0, 2, 4]].isnan().any()
    assert K % 32 or not s[3, 1:].isnan().any()


def test_norm_many_rows():
    """More workgroups than one dimension of a launch holds here; offsets past 32 bits of bytes."""
    P = need_gpu()
    x = torch.randn((70001, 1024), dtype=F16, device="cuda")
    w = torch.ones(1024, dtype=F16, device="cuda")
    out = P.rms_norm(x, w)
    for i in (0, 65535, 65536, 70000):
        rounded_once(out[i:i + 1], plain.norm(x[i:i + 1], w, 1e-6)[1], F16, NORM_REL)
    del x, out
    big = torch.empty(5 * 2 ** 30, dtype=torch.uint8, device="cuda").view(F16)
    rows = big.as_strided((3, 4096), (2 ** 30, 1))
    rows.copy_(torch.randn((3, 4096)).half())
    w = torch.ones(4096, dtype=F16, device="cuda")
    want = plain.norm(rows, w, 1e-6)[1]
    rounded_once(P.rms_norm(rows, w, out=rows), want, F16, NORM_REL)


def test_norm_without_work():
    P = need_gpu()
    w = torch.ones(64, dtype=F16, device="cuda")
    assert P.rms_norm(torch.zeros((0, 64), dtype=F16, device="cuda"), w).shape == (0, 64)
    q, s = P.rms_norm_8bit(torch.zeros((0, 3, 64), dtype=F16, device="cuda"), w, group=32)
    assert q.shape == (0, 3, 64) and s.shape == (0, 3, 2)


def test_norm_arguments():
    P = need_gpu()
    x, w = torch.zeros((2, 64), dtype=F16, device="cuda"), torch.ones(64, dtype=F16, device="cuda")
    for a, kw in (((x.cpu(), w), {}), ((x, w.cpu()), {}), ((x.float(), w), {}), ((x, w.bfloat16()), {}), ((x, w[:32]), {}), ((x[0], w), {}),
                  ((x.t(), torch.ones(2, dtype=F16, device="cuda")), {}), ((x, w), dict(residual=x[:1])), ((x, w), dict(residual_out=x)),
                  ((x, w), dict(out=x.float())), ((x, w), dict(out=x[:, :32])), ((x, w), dict(out=x[:1].expand(2, 64))), ((x, w, -1.0), {}),
                  ((x, w), dict(residual=x.float()))):
        with pytest.raises(P.InvalidArgument):
            P.rms_norm(*a, **kw)
    for kw in (dict(group=48), dict(group=-3), dict(group=128), dict(scales=torch.zeros((2, 2), device="cuda")), dict(out=x), dict(scales=torch.zeros((2, 1), device="cuda").half())):
        with pytest.raises(P.InvalidArgument):
            P.rms_norm_8bit(x, w, **kw)


# ------------------------------------------------------------------ rotary positions

def turned(out, x, positions, r, dtype, what=""):
    """Sine and cosine rounded to fp32, two products and their sum: four roundings of 2^-24 of |a| + |b| at most; then
    one to the type."""
    want, reach = plain.rotate(x.double().cpu().numpy(), positions.cpu().numpy(), r.inv_freq.cpu().numpy(), r.interleaved, r.magnitude)
    # (the angle: position times frequency in fp64, an error of 2^-52 of it, the same in either computation)
    far = float(np.abs(positions.cpu().numpy().astype(np.float64)).max(initial=0)) * float(r.inv_freq.abs().max()) * 2.0 ** -50
    rounded_once(out, torch.from_numpy(want), dtype, 0.0, torch.from_numpy(reach * (4 * 2.0 ** -24 + far)), what)
    assert torch.equal(out[..., r.rot:].cpu(), x[..., r.rot:].cpu()), what


@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", [(1, 1, 0, 2, 2), (1, 32, 8, 128, 128), (7, 3, 1, 64, 64), (33, 4, 4, 80, 80), (5, 2, 1, 128, 32), (9, 5, 2, 96, 90),
                                            (3, 2, 2, 100, 50), (4, 1, 1, 33, 6), (2, 1, 1, 1024, 1024), (3, 2, 1, 1024, 2), (6, 9, 0, 256, 14), (4500, 3, 2, 64, 48)])
def test_rope(dtype, interleaved, T, Hq, Hkv, D, rot):
    P = need_gpu()
    gen = torch.Generator().manual_seed(T + D + rot)
    q = torch.randn((T, Hq, D), generator=gen).to(dtype).cuda()
    k = (torch.randn((T, Hkv, D), generator=gen) * 3).to(dtype).cuda() if Hkv else None
    positions = torch.randint(-5, 5000, (T,), generator=gen).int().cuda()
    r = P.Rope(rot, 10000.0, interleaved=interleaved, magnitude=1.3)
    qo = torch.full_like(q, 9.0)
    if Hkv:
        a, b = P.rope(q, positions, r, k=k, q_out=qo, k_out=torch.full_like(k, 9.0))
        turned(b, k, positions, r, dtype)
    else:
        a = P.rope(q, positions, r, q_out=qo)
    assert a is qo
    turned(a, q, positions, r, dtype)
    # in place, the same bits
    q2, k2 = q.clone(), k.clone() if Hkv else None
    P.rope(q2, positions, r, k=k2)
    assert torch.equal(q2, a) and (not Hkv or torch.equal(k2, b))


@TYPES
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_rope_far_positions(dtype, interleaved):
    """Positions to the ends of int32, either sign: angles that fp32 would have off by whole turns."""
    P = need_gpu()
    positions = torch.tensor([0, 1, -1, 4095, 99999, 10 ** 6 + 1, -10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    gen = torch.Generator().manual_seed(1)
    q = torch.randn((len(positions), 3, 64), generator=gen).to(dtype).cuda()
    for kw in (dict(), dict(scaling="linear", factor=16.0), dict(scaling="base", factor=4.0), dict(scaling="ramp", factor=8.0, original_length=4096, slow=1, fast=4)):
        r = P.Rope(64, 500000.0, interleaved=interleaved, **kw)
        turned(P.rope(q, positions.cuda(), r, q_out=torch.empty_like(q)), q, positions, r, dtype, kw)


def test_rope_back_and_forth():
    """A position and its negative undo each other, but for two roundings to the type."""
    P = need_gpu()
    q = torch.randn((50, 4, 128), dtype=torch.float32).half().cuda()
    positions = torch.randint(0, 100000, (50,), dtype=torch.int32, device="cuda")
    r = P.Rope(128)
    back = P.rope(P.rope(q, positions, r, q_out=torch.empty_like(q)), -positions, r)
    size = torch.maximum(q[..., :64].abs(), q[..., 64:].abs()).double().repeat(1, 1, 2)
    assert ((back.double() - q.double()).abs() <= size * 4 * 2.0 ** -11).all()


@TYPES
def test_rope_strides_and_ends(dtype):
    """Slices of a fused projection, head-major results, rows at odd addresses; the type's largest values, infinities, NaN."""
    P = need_gpu()
    T, H, D = 12, 3, 64
    gen = torch.Generator().manual_seed(2)
    qkv = torch.randn((T, 3 * H, D), generator=gen).to(dtype).cuda()
    positions = torch.arange(T, dtype=torch.int32, device="cuda") + 1000
    r = P.Rope(D)
    out = torch.zeros((H, T, D), dtype=dtype, device="cuda").transpose(0, 1)
    odd = torch.zeros(T * H * (D + 1) + 1, dtype=dtype, device="cuda")[1:].view(T, H, D + 1)[..., :D]
    P.rope(qkv[:, :H], positions, r, k=qkv[:, H:2 * H], q_out=out, k_out=odd)
    turned(out, qkv[:, :H], positions, r, dtype)
    turned(odd, qkv[:, H:2 * H], positions, r, dtype)
    before = qkv.clone()
    P.rope(qkv[:, :H], positions, r, k=qkv[:, H:2 * H])
    assert torch.equal(qkv[:, :H], out) and torch.equal(qkv[:, H:2 * H], odd) and torch.equal(qkv[:, 2 * H:], before[:, 2 * H:])
    most = torch.finfo(dtype).max
    q = torch.full((4, 1, 64), most, dtype=dtype, device="cuda")
    q[1], q[2, 0, 7], q[3, 0, 7] = -most, float("inf"), float("nan")
    got = P.rope(q, torch.tensor([1, 1, 0, 5], dtype=torch.int32, device="cuda"), r, q_out=torch.empty_like(q))
    assert torch.isfinite(got[:2]).all() and got[0, 0].abs().max() == most       # saturated, not infinite
    nan = got.isnan().nonzero()[:, [0, 2]].tolist()
    assert [3, 7] in nan and [3, 39] in nan and all(n[1] in (7, 39) for n in nan)


def test_rope_of_more_tokens_than_a_launch_has_threads_along_x():
    P = need_gpu()
    T = (1 << 25) + 70001   # two tokens a workgroup of 256: 2^32 threads and some
    r = P.Rope(2)
    positions = torch.arange(T, dtype=torch.int32, device="cuda") % 1000
    q = torch.zeros((T, 1, 2), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    P.rope(q, positions, r)
    w = positions.double()
    want = torch.stack([w.cos(), w.sin()], 1)
    assert ((q[:, 0].double() - want).abs().max() <= 2.0 ** -11 + 2.0 ** -22).item()   # (values of 1 at most: half a step of fp16, and fp32's)


def test_rope_arguments():
    P = need_gpu()
    q, pos, r = torch.zeros((2, 4, 64), dtype=F16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), P.Rope(64)
    for a, kw in (((q.cpu(), pos, r), {}), ((q.float(), pos, r), {}), ((q[0], pos, r), {}), ((q, pos[:1], r), {}), ((q, pos.long(), r), {}), ((q, pos.cpu(), r), {}),
                  ((q, pos, P.Rope(66)), {}), ((q, pos, P.Rope(64, device="cpu")), {}), ((q, pos, r), dict(k=q.bfloat16())), ((q, pos, r), dict(k=q[:1])),
                  ((q, pos, r), dict(k_out=q)), ((q, pos, r), dict(q_out=q[:, :2])), ((q, pos, r), dict(k=q[..., :32])), ((q.transpose(1, 2), pos, r), {})):
        with pytest.raises(P.InvalidArgument):
            P.rope(*a, **kw)
    assert P.rope(q[:0], pos[:0], r).shape == (0, 4, 64)


def test_streams_and_captured_calls():
    """On another stream than the current one's default, and captured: each replay equals the eager call on its inputs."""
    P = need_gpu()
    T, K, H = 5, 512, 4
    w, r = torch.rand(K, device="cuda").half(), P.Rope(128, scaling="linear", factor=2.0)
    d = {"x": torch.zeros((T, K), dtype=F16, device="cuda"), "res": torch.zeros((T, K), dtype=F16, device="cuda"), "pos": torch.zeros(T, dtype=torch.int32, device="cuda")}

    def step(x, res, pos):
        y = P.rms_norm(x, w, residual=res)
        P.rope(y.view(T, H, 128), pos, r)
        return y, *P.rms_norm_8bit(y, w, group=128)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(**d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = step(**d)
    for i in range(4):
        x, res, pos = torch.randn((T, K)).half().cuda(), torch.randn((T, K)).half().cuda(), torch.randint(0, 9999, (T,)).int().cuda()
        for name, t in (("x", x), ("res", res), ("pos", pos)):
            d[name].copy_(t)
        g.replay()
        torch.cuda.synchronize()
        want = step(x, res, pos)
        assert torch.equal(res, d["res"])
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want)), i
