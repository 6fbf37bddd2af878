"""How large a workspace 4-bit cache attention asks for: no more than its launches can write."""
import ctypes

import numpy as np
import pytest

from helpers import pkg

COUNTERS = 65536


def ask(P, *shape):
    """(bytes, path) of T, B, Hq, Hkv, D, max_q, max_kv."""
    out = (ctypes.c_int32 * 4)()
    P.lib().w4a16_internal_kv4_path(*shape, out)
    return P.lib().w4a16_kv4_attention_workspace_size(*shape), tuple(out)


@pytest.mark.parametrize("shape,least", [
    ((570, 480, 32, 8, 128, 90, 32768), 1 << 30),     # single tokens and short prompts: tiles enough without a split
    ((1055, 32, 32, 8, 128, 1024, 4096), 1 << 25),    # a chunk of a prompt among single tokens
    ((2048, 1, 32, 8, 128, 2048, 2048), 1 << 20),     # one prompt
])
def test_prompts_in_one_chunk_have_no_partial_results(shape, least):
    """What is left is that of the sequences which run on the kernel for few columns."""
    P = pkg()
    n, (kind, _, splits, few_q) = ask(P, *shape)
    assert kind == 2 and splits == 1
    few = ask(P, *shape[:5], few_q, shape[6])[0] if few_q else COUNTERS
    assert n == few < least


def test_partial_results_are_at_most_the_tiles_times_their_chunks():
    P = pkg()
    rng = np.random.RandomState(4)
    seen = [0, 0, 0]
    for _ in range(4000):
        Hkv, G, D = int(rng.choice([1, 2, 8, 12, 32])), int(rng.choice([1, 3, 4, 8, 24])), int(rng.choice([64, 128, 192, 256]))
        if Hkv * G > 1024:
            continue
        B, mq, mkv = int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 17))
        T = max(1, int(min(B * mq, 2 ** rng.uniform(0, 14))))
        n, (kind, nt, splits, few_q) = ask(P, T, B, Hkv * G, Hkv, D, mq, mkv)
        if kind == 2:
            few = ask(P, T, B, Hkv * G, Hkv, D, few_q, mkv)[0] - COUNTERS if few_q else 0
            tiles = -(-min(mq, T) * G // 128) * B
            # (a smaller max_kv_len never has more chunks than this one may: one more than these where they are rounded up)
            most = 0 if splits == 1 else min(-(-mkv // 512), 2 * splits) * tiles * Hkv * 128
            assert n <= COUNTERS + few + most * (D + 2) * 4
            seen[0 if splits == 1 else 1] += 1
        else:
            tiles = -(-min(mq, T) * G // (32 * nt))
            assert n <= COUNTERS + tiles * Hkv * splits * 64 * (D + 2) * 4
            seen[2] += 1
    assert min(seen) > 100, seen
