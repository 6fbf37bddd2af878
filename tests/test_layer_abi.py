"""Norm, rotary positions and the 8-bit cache without a GPU: refusals before any HIP call, sizes, frequencies, the
choice of an attention kernel, and the plain implementation that the GPU tests compare with."""
import ctypes
import math

import numpy as np
import pytest
import torch

import kv8_plain as plain
from helpers import pkg

P16 = 1 << 20   # a 16-byte aligned address that nothing reads


def _err(P):
    return P.lib().w4a16_last_error().decode()


def _refused(P, rc, needle, unsupported=False):
    assert rc == (P.ERR_UNSUPPORTED if unsupported else P.ERR_INVALID_ARG), _err(P)
    assert needle in _err(P)


def _norm(P, **over):
    a = dict(elem=0, x=P16, xst=64, xsh=64, r=None, rst=0, rsh=0, ro=None, rost=0, rosh=0, w=P16, out=P16, ost=64, osh=64,
             scales=P16, T=4, H=1, K=64, group=None, eps=1e-6)
    a.update(over)
    head = (None, a["elem"], a["x"], a["xst"], a["xsh"], a["r"], a["rst"], a["rsh"], a["ro"], a["rost"], a["rosh"], a["w"], a["out"], a["ost"], a["osh"])
    if a["group"] is None:
        return P.lib().w4a16_rms_norm(*head, a["T"], a["H"], a["K"], a["eps"])
    return P.lib().w4a16_rms_norm_8bit(*head, a["scales"], a["T"], a["H"], a["K"], a["group"], a["eps"])


@pytest.mark.parametrize("group", [None, 0], ids=["16 bits", "8 bits"])
@pytest.mark.parametrize("over,needle,unsupported", [
    (dict(elem=3), "element type", False),
    (dict(T=-1), "bad sizes", False),
    (dict(H=0), "bad sizes", False),
    (dict(K=0), "bad sizes", False),
    (dict(K=65537), "at most 65536", True),
    (dict(T=2 ** 20, H=2 ** 11), "2^30", True),
    (dict(eps=-1e-6), "eps", False),
    (dict(eps=float("nan")), "eps", False),
    (dict(eps=float("inf")), "eps", False),
    (dict(x=None), "null pointer argument (x)", False),
    (dict(w=None), "null pointer", False),
    (dict(out=None), "null pointer argument (out)", False),
    (dict(x=P16 + 1), "2-byte aligned", False),
    (dict(w=P16 + 1), "2-byte aligned", False),
    (dict(r=P16), "both or neither", False),
    (dict(ro=P16), "both or neither", False),
    (dict(r=P16, ro=P16, rst=64, rost=60), "residual_out: rows", False),
    (dict(r=P16 + 1, ro=P16, rst=64, rost=64), "2-byte aligned", False),
    (dict(xst=-64), "non-negative", False),
    (dict(ost=63), "over each other", False),
    (dict(H=2, osh=32, ost=128), "over each other", False),
])
def test_norm_refusals(group, over, needle, unsupported):
    P = pkg()
    _refused(P, _norm(P, group=group, **over), needle, unsupported)


@pytest.mark.parametrize("over,needle", [
    (dict(group=-1), "group -1"), (dict(group=16), "group 16"), (dict(group=48, K=96), "group 48"), (dict(group=1024, K=2048), "group 1024"),
    (dict(group=128), "a multiple"), (dict(group=0, scales=None), "scales"), (dict(group=0, scales=P16 + 2), "4-byte")])
def test_norm_8bit_refusals(over, needle):
    P = pkg()
    _refused(P, _norm(P, **over), needle)


def test_norm_without_rows_is_no_call():
    P = pkg()
    assert _norm(P, T=0, x=None, out=None) == 0 and _norm(P, T=0, group=0, scales=None) == 0


def _rope(P, **over):
    a = dict(elem=0, q=P16, qst=256, qsh=64, qo=P16, qost=256, qosh=64, k=P16, kst=128, ksh=64, ko=P16, kost=128, kosh=64, pos=P16, f=P16,
             mag=1.0, T=4, Hq=4, Hkv=2, D=64, rot=64, inter=0)
    a.update(over)
    return P.lib().w4a16_rope(None, *a.values())


@pytest.mark.parametrize("over,needle,unsupported", [
    (dict(elem=9), "element type", False),
    (dict(T=-1), "bad sizes", False),
    (dict(Hq=0), "bad sizes", False),
    (dict(D=0), "bad sizes", False),
    (dict(D=1040), "at most 1024 of 1024", True),
    (dict(T=2 ** 30 // 4 + 1), "2^30", True),
    (dict(Hq=1025), "at most 1024", True),
    (dict(rot=0), "rot=0", False),
    (dict(rot=33), "rot=33", False),
    (dict(rot=66), "rot=66", False),
    (dict(mag=float("inf")), "magnitude", False),
    (dict(k=None), "all or none", False),
    (dict(ko=None), "all or none", False),
    (dict(Hkv=0), "all or none", False),
    (dict(q=None), "null pointer argument (q)", False),
    (dict(qo=None), "null pointer argument (q_out)", False),
    (dict(pos=None), "null pointer", False),
    (dict(f=None), "null pointer", False),
    (dict(pos=P16 + 2), "4-byte", False),
    (dict(f=P16 + 4), "8-byte", False),
    (dict(q=P16 + 1), "2-byte aligned", False),
    (dict(qost=200), "q_out: rows", False),
    (dict(kosh=63), "k_out: rows", False),
])
def test_rope_refusals(over, needle, unsupported):
    P = pkg()
    _refused(P, _rope(P, **over), needle, unsupported)


def test_rope_without_rows_is_no_call():
    P = pkg()
    assert _rope(P, T=0, q=None) == 0 and _rope(P, T=0, k=None, ko=None, Hkv=0) == 0


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("base", 8.0), ("ramp", 8.0), ("ramp", 0.5)])
@pytest.mark.parametrize("rot,base", [(2, 10000.0), (96, 10000.0), (128, 5e5), (1024, 1e4)])
def test_frequencies(rot, base, scaling, factor):
    """Within a few roundings of fp64: a power's error is that of its exponent, at most ln(base factor^2) 2^-51."""
    P = pkg()
    r = P.Rope(rot, base, scaling=scaling, factor=factor, original_length=8192, slow=1.0, fast=4.0, device="cpu")
    want = plain.frequencies(rot, base, scaling, factor, 8192, 1.0, 4.0)
    assert r.rot == rot and np.abs(r.inv_freq.numpy() / want - 1).max() < 2.0 ** -44
    if scaling == "ramp":   # both ends of the ramp are there
        plain_f = plain.frequencies(rot, base)
        assert r.inv_freq[0] == plain_f[0]
        assert rot == 2 or abs(r.inv_freq[-1].item() / (plain_f[-1] / factor) - 1) < 2.0 ** -44


@pytest.mark.parametrize("a,needle", [
    ((3, 1e4, 0, 1, 0, 0, 1), "rot=3"), ((0, 1e4, 0, 1, 0, 0, 1), "rot=0"), ((1026, 1e4, 0, 1, 0, 0, 1), "rot=1026"), ((64, 0.0, 0, 1, 0, 0, 1), "base"),
    ((64, math.nan, 0, 1, 0, 0, 1), "base"), ((64, 1e4, 4, 1, 0, 0, 1), "scaling 4"), ((64, 1e4, -1, 1, 0, 0, 1), "scaling -1"), ((64, 1e4, 1, 0.0, 0, 0, 1), "factor"),
    ((64, 1e4, 2, math.inf, 0, 0, 1), "factor"), ((64, 1e4, 3, 2, 0.0, 1, 4), "original_length"), ((64, 1e4, 3, 2, 8192, 4, 4), "slow < fast"),
    ((64, 1e4, 3, 2, 8192, -1, 4), "slow < fast")])
def test_frequency_refusals(a, needle):
    P = pkg()
    _refused(P, P.lib().w4a16_rope_frequencies(*a, (ctypes.c_double * 512)()), needle)


def test_frequencies_need_room():
    P = pkg()
    _refused(P, P.lib().w4a16_rope_frequencies(64, 1e4, 0, 1.0, 0.0, 0.0, 1.0, None), "null pointer")


def test_rope_handles():
    P = pkg()
    r = P.Rope(inv_freq=[1.0, 0.5, 0.1], interleaved=True, magnitude=1.5, device="cpu")
    assert (r.rot, r.interleaved, r.magnitude) == (6, True, 1.5) and r.inv_freq.dtype == torch.float64
    for bad in (dict(), dict(rot=64, scaling="other"), dict(rot=8, inv_freq=[1.0]), dict(inv_freq=[]), dict(inv_freq=[[1.0]]), dict(rot=-2), dict(rot=2 ** 33)):
        with pytest.raises(P.InvalidArgument):
            P.Rope(device="cpu", **bad)


# ------------------------------------------------------------------ 8-bit cache

def _write(P, **over):
    a = dict(elem=0, k=P16, kst=256, ksh=64, v=P16, vst=256, vsh=64, q=None, qst=0, qsh=0, qo=None, qost=0, qosh=0, pos=None, f=None, mag=1.0,
             rot=0, inter=0, cache=P16, table=P16, lens=P16, cu=P16, T=8, B=2, Hq=0, Hkv=4, D=64, pages=4, page=16, per=2, mq=8)
    a.update(over)
    return P.lib().w4a16_kv8_write(None, *a.values())


TURN = dict(f=P16, rot=64, q=P16, qst=512, qsh=64, qo=P16, qost=512, qosh=64, Hq=8)


@pytest.mark.parametrize("over,needle,unsupported", [
    (dict(elem=7), "element type", False),
    (dict(k=None), "null pointer argument (k)", False),
    (dict(v=None), "null pointer argument (v)", False),
    (dict(cache=None), "null pointer", False),
    (dict(table=None), "null pointer", False),
    (dict(lens=None), "null pointer", False),
    (dict(k=P16 + 8), "16-byte aligned", False),
    (dict(cache=P16 + 8), "16-byte aligned", False),
    (dict(table=P16 + 2), "4-byte", False),
    (dict(cu=P16 + 1), "4-byte", False),
    (dict(kst=252), "multiples of 8", False),
    (dict(vsh=-64), "multiples of 8", False),
    (dict(pages=0), "must be positive", False),
    (dict(T=-1), "bad sizes", False),
    (dict(B=-1), "bad sizes", False),
    (dict(mq=0), "bad sizes", False),
    (dict(per=0), "bad sizes", False),
    (dict(D=96), "head dimension 96", True),
    (dict(page=24), "page_size 24", True),
    (dict(Hkv=1025), "1025 heads", True),
    (dict(pages=2 ** 31 - 1), "slots are int32", True),
    (dict(T=2 ** 22 + 1), "tokens: at most", True),
    (dict(B=65536), "sequences", True),
    (dict(cu=None), "one token", False),
    (dict(cu=None, B=8), "max_q_len is 1", False),
    (dict(pos=P16), "for a rotation", False),
    (dict(q=P16, qo=P16, Hq=8), "for a rotation", False),
    ({**TURN, "qo": None}, "all or none", False),
    ({**TURN, "Hq": 0}, "all or none", False),
    ({**TURN, "Hq": 1025}, "1025 heads", True),
    ({**TURN, "rot": 66}, "rot=66", False),
    ({**TURN, "rot": 31}, "rot=31", False),
    ({**TURN, "rot": 0}, "rot=0", False),
    ({**TURN, "mag": float("nan")}, "magnitude", False),
    ({**TURN, "f": P16 + 4}, "8-byte", False),
    ({**TURN, "pos": P16 + 2}, "4-byte", False),
    ({**TURN, "q": P16 + 1}, "2-byte aligned", False),
    ({**TURN, "qost": 500}, "q_out: rows", False),
])
def test_write_refusals(over, needle, unsupported):
    P = pkg()
    _refused(P, _write(P, **over), needle, unsupported)


def test_write_without_tokens_is_no_call():
    P = pkg()
    assert _write(P, T=0, k=None, cache=None) == 0 and _write(P, T=0, B=0, cu=None, mq=1) == 0


def _read(P, **over):
    a = dict(elem=0, cache=P16, slots=P16, k=P16, kst=256, ksh=64, v=P16, vst=256, vsh=64, pages=4, T=8, Hkv=4, D=64, page=16)
    a.update(over)
    return P.lib().w4a16_kv8_read(None, *a.values())


@pytest.mark.parametrize("over,needle,unsupported", [
    (dict(elem=7), "element type", False),
    (dict(k=None), "null pointer", False),
    (dict(v=None), "null pointer", False),
    (dict(slots=None), "null pointer", False),
    (dict(cache=None), "null pointer", False),
    (dict(v=P16 + 8), "16-byte aligned", False),
    (dict(cache=P16 + 4), "16-byte aligned", False),
    (dict(slots=P16 + 2), "4-byte", False),
    (dict(kst=252), "multiples of 8", False),
    (dict(ksh=56), "over each other", False),
    (dict(T=-1), "must not be negative", False),
    (dict(D=80), "head dimension 80", True),
    (dict(page=8), "page_size 8", True),
    (dict(T=2 ** 31 - 1), "at most", True),
])
def test_read_refusals(over, needle, unsupported):
    P = pkg()
    _refused(P, _read(P, **over), needle, unsupported)


def test_cache_bytes():
    P = pkg()
    f = P.lib().w4a16_kv8_cache_bytes
    assert f(3, 8, 128, 64) == 3 * 8 * 4 * (32 * 128 + 16)
    assert f(1, 1, 64, 16) == 2064
    assert f(2 ** 21, 8, 128, 64) == 2 ** 21 * 8 * 4 * 4112
    for bad in ((0, 8, 128, 64), (1, 0, 128, 64), (1, 8, 80, 64), (1, 8, 128, 48), (2 ** 27, 8, 128, 16), (1, 1025, 128, 16)):
        assert f(*bad) == 0, bad
    with pytest.raises(P.Unsupported):
        P.kv8_cache(4, 2, 80, 16, device="cpu")
    assert P.kv8_cache(4, 2, 64, 32, device="cpu").shape == (4, 2, 2, 2064)


def _attention(P, **over):
    a = dict(elem=0, q=P16, qst=512, qsh=64, cache=P16, table=P16, lens=P16, cu=P16, out=P16, ost=512, osh=64, lse=None, T=8,
             B=2, Hq=8, Hkv=4, D=64, pages=4, page=16, per=2, mq=4, mkv=32, scale=0.1, causal=1, window=0, ws=P16, wsb=1 << 30)
    a.update(over)
    return P.lib().w4a16_kv8_attention(None, *a.values())


@pytest.mark.parametrize("over,needle,unsupported", [
    (dict(elem=1), "element type", False),
    (dict(q=None), "null pointer", False),
    (dict(out=None), "null pointer", False),
    (dict(cache=None), "null pointer", False),
    (dict(Hq=6), "multiple of 4", False),
    (dict(T=-1), "bad sizes", False),
    (dict(mq=0), "bad sizes", False),
    (dict(per=0), "pages_per_seq", False),
    (dict(window=-1), "window", False),
    (dict(scale=float("nan")), "finite", False),
    (dict(cu=None), "one query", False),
    (dict(q=P16 + 2), "16-byte aligned", False),
    (dict(ost=504), "over each other", False),
    (dict(ws=None), "workspace too small", False),
    (dict(wsb=1024), "workspace too small", False),
    (dict(ws=P16 + 16), "256-byte aligned", False),
    (dict(D=80), "head dimension 80", True),
    (dict(page=40), "page_size 40", True),
    (dict(mkv=2 ** 30 + 1), "max_kv_len", True),
    (dict(B=65, mkv=2 ** 30), "2^36 keys", True),
])
def test_attention_refusals(over, needle, unsupported):
    P = pkg()
    _refused(P, _attention(P, **over), needle, unsupported)


def test_workspace_covers_every_split():
    """Partial results of as many chunks as a launch may have fit; a smaller max_kv_len needs no more."""
    P = pkg()
    out = (ctypes.c_int32 * 4)()
    rng = np.random.RandomState(3)
    for _ in range(1500):
        Hkv, G, D = int(rng.choice([1, 2, 8, 12, 64])), int(rng.choice([1, 3, 4, 8, 24])), int(rng.choice([64, 128, 192, 256]))
        if Hkv * G > 1024:
            continue
        B, mq, mkv = int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 17))
        a = (min(B * mq, 4096), B, Hkv * G, Hkv, D, mq)
        n = P.lib().w4a16_kv8_attention_workspace_size(*a, mkv)
        P.lib().w4a16_internal_kv8_path(*a, mkv, out)
        kind, _, parts, few_q = out
        cols = min(mq, a[0]) * G
        assert (kind == 2) == (cols > 64) and n >= 65536
        if kind == 1 and n > 65536:
            assert n >= 65536 + 4 * parts * Hkv * min(cols, 32) * (D + 2) // 2
        assert P.lib().w4a16_kv8_attention_workspace_size(*a, max(1, mkv // 2)) <= n


# ------------------------------------------------------------------ the plain implementation

def test_plain_e4m3_is_torchs():
    """All codes, all ties between neighbours, and random numbers."""
    codes = np.arange(256, dtype=np.uint8)
    values = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(values, plain.VALUES, equal_nan=True)
    ties = (plain.TABLE[1:] + plain.TABLE[:-1]) / 2
    rng = np.random.RandomState(0)
    x = np.concatenate((ties, -ties, plain.TABLE, -plain.TABLE, rng.uniform(-448, 448, 100000), rng.standard_normal(100000) * 2.0 ** rng.randint(-14, 8, 100000)))
    x = np.clip(x, -448, 448).astype(np.float32).astype(np.float64)
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(plain.e4m3(x)[0], want)


@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_plain_layout_has_a_byte_for_everything(D):
    k, v = plain.places(D)
    assert sorted(np.concatenate((k.ravel(), v.ravel()))) == list(range(32 * D))


def test_plain_append_and_held():
    """What is appended in pieces is held within a step of e4m3 at the scale of its block's final content."""
    rng = np.random.RandomState(1)
    table = np.array([[2, 0]])
    cache = rng.randint(0, 256, (3, 2, 2, 32 * 64 + 16)).astype(np.uint8)
    k, v = (rng.standard_normal((50, 2, 64)) * 2.0 ** rng.randint(-3, 9, (50, 1, 1)) for _ in range(2))
    at = 0
    for n in (1, 5, 3, 20, 1, 1, 19):
        plain.append(cache, table, 0, at, k[at:at + n], v[at:at + n])
        at += n
    for x, y in zip((k, v), plain.held(cache, table, 0, 50)):
        for blk in range(4):
            top = np.abs(x[16 * blk:16 * blk + 16]).max((0, 2), keepdims=True)
            err = np.abs(x[16 * blk:16 * blk + 16] - y[16 * blk:16 * blk + 16])
            # (once or, with the scale raised, again as a subnormal: a step of 2^-9 of a scale of at most top / 224)
            assert (err <= np.abs(x[16 * blk:16 * blk + 16]) / 16 + top / 224 * 2.0 ** -9).all()
