"""The 4-bit key/value cache without a GPU: sizes, refusals before any HIP call, the choice of an attention
kernel, and the plain implementation that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_plain as plain
from helpers import pkg

P16 = 1 << 20   # a 16-byte aligned address that nothing reads


def _err(P):
    return P.lib().w4a16_last_error().decode()


def _rows(P, read=False, **over):
    a = dict(elem=0, k=P16, v=P16, kst=256, ksh=64, vst=256, vsh=64, slots=P16, cache=P16, pages=4, T=8, Hkv=4, D=64, page=16)
    a.update(over)
    s = (a["kst"], a["ksh"], a["vst"], a["vsh"])
    if read:
        return P.lib().w4a16_kv4_read(None, a["elem"], a["cache"], a["slots"], a["k"], a["v"], *s, a["pages"], a["T"], a["Hkv"], a["D"], a["page"])
    return P.lib().w4a16_kv4_write(None, a["elem"], a["k"], a["v"], *s, a["slots"], a["cache"], a["pages"], a["T"], a["Hkv"], a["D"], a["page"])


@pytest.mark.parametrize("read", [False, True], ids=["write", "read"])
@pytest.mark.parametrize("over,needle,unsupported", [
    (dict(elem=7), "element type", False),
    (dict(k=None), "null pointer", False),
    (dict(v=None), "null pointer", False),
    (dict(slots=None), "null pointer", False),
    (dict(cache=None), "null pointer", False),
    (dict(k=P16 + 8), "16-byte aligned", False),
    (dict(cache=P16 + 4), "16-byte aligned", False),
    (dict(slots=P16 + 2), "4-byte", False),
    (dict(kst=252), "multiples of 8", False),
    (dict(vsh=-64), "multiples of 8", False),
    (dict(pages=0), "must be positive", False),
    (dict(Hkv=0), "must be positive", False),
    (dict(T=-1), "must not be negative", False),
    (dict(D=96), "head dimension 96", True),
    (dict(page=24), "page_size 24", True),
    (dict(page=8), "page_size 8", True),
    (dict(page=2048), "page_size 2048", True),
    (dict(Hkv=1025), "1025 heads", True),
    (dict(pages=2 ** 31 - 1), "slots are int32", True),
    (dict(T=2 ** 31 - 1), "at most", True),
])
def test_row_refusals(read, over, needle, unsupported):
    P = pkg()
    assert _rows(P, read, **over) == (P.ERR_UNSUPPORTED if unsupported else P.ERR_INVALID_ARG)
    assert needle in _err(P)


@pytest.mark.parametrize("over", [dict(ksh=56), dict(kst=248), dict(vst=64, vsh=64), dict(kst=0)])
def test_read_refuses_rows_over_each_other(over):
    P = pkg()
    assert _rows(P, True, **over) == P.ERR_INVALID_ARG and "over each other" in _err(P)


def test_no_rows_is_no_call():
    P = pkg()
    assert _rows(P, T=0, k=None, slots=None) == 0 and _rows(P, True, T=0, cache=None) == 0


def test_cache_bytes():
    P = pkg()
    f = P.lib().w4a16_kv4_cache_bytes
    assert f(3, 8, 128, 64) == 3 * 8 * 4 * (16 * 128 + 128)
    assert f(1, 1, 64, 16) == 1152
    assert f(2 ** 21, 8, 128, 64) == 2 ** 21 * 8 * 4 * 2176
    for bad in ((0, 8, 128, 64), (1, 0, 128, 64), (1, 8, 80, 64), (1, 8, 128, 48), (2 ** 27, 8, 128, 16), (1, 1025, 128, 16)):
        assert f(*bad) == 0, bad


def _attention(P, **over):
    a = dict(elem=0, q=P16, qst=512, qsh=64, cache=P16, table=P16, lens=P16, cu=P16, out=P16, ost=512, osh=64, lse=None, T=8,
             B=2, Hq=8, Hkv=4, D=64, pages=4, page=16, per=2, mq=4, mkv=32, scale=0.1, causal=1, window=0, ws=P16, wsb=1 << 30)
    a.update(over)
    return P.lib().w4a16_kv4_attention(None, *a.values())


@pytest.mark.parametrize("over,needle,unsupported", [
    (dict(elem=1), "element type", False),
    (dict(q=None), "null pointer", False),
    (dict(out=None), "null pointer", False),
    (dict(cache=None), "null pointer", False),
    (dict(table=None), "null pointer", False),
    (dict(lens=None), "null pointer", False),
    (dict(Hq=6), "multiple of 4", False),
    (dict(Hq=0), "multiple of", False),
    (dict(T=-1), "bad sizes", False),
    (dict(B=-1), "bad sizes", False),
    (dict(mq=0), "bad sizes", False),
    (dict(mkv=-1), "bad sizes", False),
    (dict(per=0), "pages_per_seq", False),
    (dict(window=-1), "window", False),
    (dict(scale=float("nan")), "finite", False),
    (dict(scale=float("inf")), "finite", False),
    (dict(scale=3e38), "finite", False),      # (times log2 e it is not)
    (dict(cu=None), "one query", False),
    (dict(cu=None, T=2), "max_q_len is 1", False),
    (dict(q=P16 + 2), "16-byte aligned", False),
    (dict(qsh=60), "multiples of 8", False),
    (dict(ost=504), "over each other", False),
    (dict(osh=0), "over each other", False),
    (dict(lse=P16 + 2), "4-byte aligned", False),
    (dict(lens=P16 + 1), "4-byte aligned", False),
    (dict(ws=None), "workspace too small", False),
    (dict(wsb=1024), "workspace too small", False),
    (dict(ws=P16 + 16), "256-byte aligned", False),
    (dict(D=80), "head dimension 80", True),
    (dict(page=40), "page_size 40", True),
    (dict(Hq=2048, Hkv=4), "2048 heads", True),
    (dict(B=70000), "sequences", True),
    (dict(mkv=2 ** 30 + 1), "max_kv_len", True),
    (dict(B=65, mkv=2 ** 30), "2^36 keys", True),
    (dict(T=2 ** 27, mq=2 ** 27, qst=512), "at most", True),
])
def test_attention_refusals(over, needle, unsupported):
    P = pkg()
    assert _attention(P, **over) == (P.ERR_UNSUPPORTED if unsupported else P.ERR_INVALID_ARG), _err(P)
    assert needle in _err(P)


def test_attention_without_work_is_no_call():
    P = pkg()
    assert _attention(P, T=0, q=None) == 0
    assert _attention(P, T=0, B=0, cu=None, mq=1) == 0


def test_workspace_covers_every_split():
    """Partial results of as many chunks as a launch may have fit, whatever the lengths are."""
    P = pkg()
    out = (ctypes.c_int32 * 4)()
    rng = np.random.RandomState(3)
    for _ in range(2000):
        Hkv, G, D = int(rng.choice([1, 2, 8, 12, 64])), int(rng.choice([1, 3, 4, 8, 24])), int(rng.choice([64, 128, 192, 256]))
        if Hkv * G > 1024:
            continue
        B, mq, mkv = int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 11)), int(2 ** rng.uniform(0, 17))
        T = min(B * mq, 4096)
        a = (T, B, Hkv * G, Hkv, D, mq, mkv)
        n = P.lib().w4a16_kv4_attention_workspace_size(*a)
        P.lib().w4a16_internal_kv4_path(*a, out)
        C = min(mq, T) * G
        assert (out[0] == 2) == (C > 64)
        if out[0] == 2:
            rows = -(-C // 128) * B
            if 1 < B <= 1024 and 2 * max(1, (T * G + 127 * B) // 128) < rows:
                rows = max(1, (T * G + 127 * B) // 128)      # one row of tiles: no more than T rows of q make
            slots = 0 if out[2] == 1 else rows * Hkv * out[2] * 128
            assert out[2] == 1 or rows * Hkv <= 4096
            assert out[3] == (64 // G if B > 1 and 4 * T < B * mq else 0)
            if out[3]:           # and the partial results of what runs on the other kernel
                few = P.lib().w4a16_kv4_attention_workspace_size(T, B, Hkv * G, Hkv, D, out[3], mkv) - 65536
                assert n >= 65536 + slots * (D + 2) * 4 + few
        else:
            tiles = -(-C // (32 * out[1]))
            whole = mkv <= 512 or tiles * B * Hkv > 16384
            slots = 0 if whole else tiles * Hkv * out[2] * (-(-min(C, 32 * out[1]) // 16) * 16)
            assert out[2] >= B
            # the rule of the kernel: chunks of c 128 keys, at most `places` of them for any lengths
            if not whole and B <= 64:
                at_once = max(1, 256 * {(64, 1): 4, (128, 1): 4, (192, 1): 3, (256, 1): 2, (64, 2): 3, (128, 2): 2}[D, out[1]] // (Hkv * tiles))
                budget = max(2 * B, min(128 * B, -(-2 * B // at_once) * at_once))
                for _ in range(4):
                    steps = [-(-int(x) // 32) for x in rng.randint(0, mkv + 1, B)]
                    chunks = lambda c: sum(1 if s <= max(16, 4 * c) else -(-s // (4 * c)) for s in steps)
                    for rest in (0, 2, 4):
                        c = max(1, -(-sum(steps) // (4 * budget - rest * B)))
                        if rest == 4 or chunks(c) <= budget:
                            break
                    assert chunks(c) <= out[2], (a, c)
        assert n >= 65536 + slots * (D + 2) * 4 if out[0] == 2 else n == 65536 + slots * (D + 2) * 4
        less = a[:6] + (int(mkv * rng.uniform(0, 1)),)
        assert P.lib().w4a16_kv4_attention_workspace_size(*less) <= n, "a smaller max_kv_len fits too"


def test_python_refusals_without_a_gpu():
    P = pkg()
    cpu = torch.zeros((1, 2, 1, 16 * 64 + 128), dtype=torch.uint8)
    rows = torch.zeros((3, 2, 64), dtype=torch.float16)
    ids = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: P.kv4_write(rows, rows, cpu, ids), lambda: P.kv4_read(cpu, ids),
                 lambda: P.kv4_attention(rows, cpu, ids.view(3, 1), ids), lambda: P.kv4_write(rows, rows, None, ids)):
        with pytest.raises(P.InvalidArgument, match="cache"):
            call()
    for shape in ((2, 8, 96, 64), (2, 8, 128, 20), (0, 8, 128, 16)):
        with pytest.raises(P.Unsupported):
            P.kv4_cache(*shape, device="cpu")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_plain_quantisation(dtype):
    """What is held is within half a step, and the rounding of the scale and of the zero point, of the row; ends, zero
    and constants."""
    gen = torch.Generator().manual_seed(1)
    x = (torch.randn((50, 64), generator=gen) * torch.randn((50, 1), generator=gen).exp() + torch.randn((50, 1), generator=gen)).to(dtype)
    n, s, z, held = plain.quantise(x)
    d, sd = x.double().numpy(), s.double().numpy()[:, None]
    eps = torch.finfo(dtype).eps / 2
    # a value at an end may be clamped by the half step that rounding the zero point moved the grid
    assert (np.abs(held - d) <= sd * (1.0 + 16 * eps)).all()
    inner = (n > 0) & (n < 15)
    assert (np.abs(held - d)[inner] <= (sd * np.ones_like(d))[inner] * 0.5 * (1 + 1e-9)).all()
    assert n.max() == 15 and n.min() == 0
    for v in (0.0, 3.0, -2.5):
        n, s, z, held = plain.quantise(torch.full((1, 64), v).to(dtype))
        assert np.abs(held - v).max() <= abs(v) * eps * 2
    n, s, z, held = plain.quantise(torch.tensor([[0.5] * 63 + [15.0]]).to(dtype))
    assert (n[0, :63] == 0).all() and n[0, 63] == 15   # 0.5 is a tie: to even
    bad = torch.zeros((1, 64), dtype=dtype)
    bad[0, 1] = float("inf")
    assert np.isnan(plain.quantise(bad)[3]).all()


def test_plain_layout():
    """A row's nibbles are where the header puts them."""
    cache = np.zeros((2, 3, 2, 16 * 128 + 128), np.uint8)
    n = (np.arange(128) % 16).astype(np.uint8)
    plain.pack(cache, 32 + 21, 1, 0, n, torch.tensor(1.5, dtype=torch.float16), 7)
    plain.pack(cache, 32 + 21, 1, 1, n, torch.tensor(2.5, dtype=torch.float16), 9)
    block = cache[1, 1, 1]
    t = 5
    assert list(block[t * 64:t * 64 + 4]) == [0x10, 0x32, 0x54, 0x76]
    # values: quad 1, pair 0, second of it: dimensions 8..11 are column 1, h 0
    at = 8 * 128 + 256 + 16 + 2
    assert list(block[at:at + 2]) == [0x98, 0xBA] and list(block[at + 4:at + 6]) == [0xDC, 0xFE]
    words = block[16 * 128:].view(np.uint32)
    assert words[t] == (7 << 16 | 0x3E00) and words[16 + t] == (9 << 16 | 0x4100)
