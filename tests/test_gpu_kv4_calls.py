"""Calls of the 4-bit key/value cache that the other tests do not make."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import BF16, F16, Batch, attention_path, need_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,B", [(3, 0), (0, 3), (3, 2)])
def test_queries_without_sequences_are_refused(T, B):
    """Without cu_q there is a query for each sequence, also where either is none at all: the result would be memory
    that nothing wrote."""
    P = need_gpu()
    cache = P.kv4_cache(2, 2, 64, 16)
    q = torch.zeros((T, 4, 64), dtype=F16, device="cuda")
    with pytest.raises(P.InvalidArgument, match="one query"):
        P.kv4_attention(q, cache, torch.zeros((B, 1), dtype=torch.int32, device="cuda"),
                        torch.zeros(B, dtype=torch.int32, device="cuda"))


def check_some(b, out, lse, which):
    """Batch.check of the sequences `which` of b alone."""
    some = Batch.__new__(Batch)
    some.dtype, some.D, some.Hq = b.dtype, b.D, b.Hq
    some.nq, some.lens, some.k, some.v = ([x[s] for s in which] for x in (b.nq, b.lens, b.k, b.v))
    rows = torch.cat([torch.arange(int(b.cu[s]), int(b.cu[s + 1])) for s in which])
    some.q = b.q[rows]
    some.check(out[rows.cuda()], lse[rows.cuda()])


@pytest.mark.parametrize("dtype,D,Hkv,nq,lens,page,path", [
    # many columns, one group of waves a tile: every D of up to 128 in one chunk of the keys and in several
    (BF16, 128, 16, [65] * 17, [300 - i for i in range(17)], 64, ("many", 1, 1)),
    (BF16, 128, 16, [65] * 16, [1030 - 9 * i for i in range(16)], 64, ("many", 1, 2)),
    (F16, 128, 16, [65, 1] * 8, [1100 - 30 * i for i in range(16)], 16, ("many", 1, 2)),
    (F16, 64, 16, [65] * 16, [1030 - 9 * i for i in range(16)], 32, ("many", 1, 3)),
    # few columns, more heads and sequences than there are counters: no sequence is split, however long
    (F16, 64, 16, [1] * 1100, [(31 * i) % 90 + 1400 * (i % 400 == 7) for i in range(1100)], 16, ("few", 1, 1100, 0)),
])
def test_instances_that_large_batches_run(dtype, D, Hkv, nq, lens, page, path):
    P = need_gpu()
    b = Batch(P, nq, lens, Hkv, Hkv, D, page, dtype)
    assert attention_path(P, sum(nq), len(nq), Hkv, Hkv, D, max(nq), max(lens)) == path
    out, lse = b.gpu(P)
    n = len(nq)
    check_some(b, out, lse, (0, 3, n // 2, n - 1) if n < 100 else (0, 7, 407, 408, 600, n - 1))
    # the others: the same as in a call of a few of them
    for s in range(0, n, max(1, n // 16)):
        rows = slice(int(b.cu[s]), int(b.cu[s + 1]))
        alone = P.kv4_attention(b.q[rows].cuda(), b.cache, b.table[s:s + 1].cuda(), torch.tensor([lens[s]], dtype=torch.int32, device="cuda"),
                                cu_q=torch.tensor([0, nq[s]], dtype=torch.int32, device="cuda"), max_q_len=max(nq), max_kv_len=max(lens))
        # either is off by the weights' and the results' rounding: 2^-11 and half a step of the largest value
        most = float(np.abs(b.v[s]).max()) if lens[s] else 0.0
        assert float((alone.double() - out[rows].double()).abs().max()) <= 2 * most * (2.0 ** -10 + torch.finfo(dtype).eps)
    again, _ = b.gpu(P)
    assert torch.equal(out, again)
