"""Calls of the 4-bit key/value cache that the other tests do not make."""
import pytest
import torch

from test_gpu_kv4 import F16, need_gpu

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
