"""Calls of the norm, rotary positions and the caches that a program may make besides the ordinary ones: no sequences, tensors that
gradients are computed of, memory that is not there, sizes beyond 32 bits."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import BF16, F16, need_gpu, rows
from test_gpu_kv8 import TYPES, Batch8, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("per", [0, 3])
def test_queries_at_given_positions_without_sequences(per):
    """Rows of no sequence are rotated at the positions that are given, also where there is no sequence at all; without
    positions they stay as they are."""
    P = need_gpu()
    T, D = 5, 64
    q = torch.randn((T, 3, D)).half().cuda()
    k = torch.randn((T, 2, D)).half().cuda()
    cache = P.kv8_cache(2, 2, D, 16)
    before = cache.random_(0, 256).clone()
    table, lens, pos, r = torch.zeros((0, per), dtype=torch.int32, device="cuda"), i32([]), i32([5, 0, -3, 10 ** 6, 77]), P.Rope(D)
    out = torch.full_like(q, 3.0)
    P.kv8_write(k, k, cache, table, lens, cu_q=i32([0]), rope=r, positions=pos, q=q, q_out=out)
    assert torch.equal(out, P.rope(q, pos, r, q_out=torch.empty_like(q)))
    out.fill_(3.0)
    P.kv8_write(k, k, cache, table, lens, cu_q=i32([0]), rope=r, q=q, q_out=out)
    P.kv8_write(k, k, cache, table, lens, cu_q=i32([0]), rope=r, positions=pos)
    P.kv8_write(k, k, cache, table, lens)
    assert (out == 3).all() and torch.equal(cache, before)
