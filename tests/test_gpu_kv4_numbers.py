"""The 4-bit key/value cache at the ends of its numbers' range: rows near the type's largest value. Compared with
64 bits (kv4_plain.py)."""
import pytest
import torch

import kv4_plain as plain
from test_gpu_kv4 import BF16, F16, need_gpu, same

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
