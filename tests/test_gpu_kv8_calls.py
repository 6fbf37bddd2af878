"""Calls of the norm, rotary positions and the caches that a program may make besides the ordinary ones: no sequences, tensors that
gradients are computed of, memory that is not there, sizes beyond 32 bits."""
import numpy as np
import pytest
import torch

from test_gpu_kv4 import F16, need_gpu, rows
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


@TYPES
@pytest.mark.parametrize("nq,L", [(3, 33), (5, 97), (5, 1601), (90, 129), (150, 401), (80, 2497)])
def test_a_largest_row_that_others_do_not_see(dtype, nq, L):
    """A block whose one token only the last query sees, its key, then its value, at the type's end: finite, so it counts for the
    block's scale and reaches every product of its step, yet moves no bit of the other queries' results.
    (The last query's own scale q . k may be more than fp32 holds.)"""
    P = need_gpu()
    assert L % 16 == 1
    b = Batch8(P, [nq], [L], 4, 2, 64, 16, dtype, seed=6)
    last = [torch.from_numpy(x[0][-1:]).to(dtype) for x in (b.k, b.v)]
    out, lse = b.gpu(P)
    most = torch.finfo(dtype).max
    sign = torch.where(torch.rand((1, 2, 64), generator=torch.Generator().manual_seed(1)) < 0.5, -most, most).to(dtype)
    for key, value in ((sign, last[1]), (last[0], sign), (sign, -sign)):
        b.put(P, 0, L - 1, key, value)
        out2, lse2 = b.gpu(P)
        assert torch.equal(out[:-1], out2[:-1]) and torch.equal(lse[:-1], lse2[:-1])
    b.put(P, 0, L - 1, *last)
    out2, lse2 = b.gpu(P)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_memory_that_is_not_there():
    """An output or workspace that cannot be had is torch's own error, so that a program that waits for it (to take a smaller
    batch) sees it. (The process's share of the card is lowered: torch refuses before it asks the device.)"""
    P = need_gpu()
    one = torch.zeros((1, 1, 256), dtype=F16, device="cuda")
    x, w = torch.zeros((1, 65536), dtype=F16, device="cuda"), torch.ones(65536, dtype=F16, device="cuda")
    c4, c8, heads4, heads8 = (f(1, n, 256, 16) for n in (1, 128) for f in (P.kv4_cache, P.kv8_cache))
    rows_ = x.expand(1 << 17, 65536)                        # 16 GiB of results, 8 in 8 bits
    q = one.expand(1 << 22, 8, 256)                         # 16 GiB of results
    many = one.expand(512, 1024, 256)                       # 1 GiB of workspace
    table, lens = i32([[0]]), i32([1])
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (256 << 20)) / total)
    try:
        for call in (lambda: P.rms_norm(rows_, w), lambda: P.rms_norm_8bit(rows_, w),
                     lambda: P.kv4_attention(q, c4, table, lens, cu_q=i32([0, 1]), max_q_len=1), lambda: P.kv8_attention(q, c8, table, lens, cu_q=i32([0, 1]), max_q_len=1),
                     lambda: P.kv4_attention_workspace(many, heads4, 64, 8, 1 << 16), lambda: P.kv8_attention_workspace(many, heads8, 64, 8, 1 << 16)):
            with pytest.raises(torch.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert not P.rms_norm(x, w).any()


def test_workspace_of_any_queries():
    """Only the number of rows and heads counts: queries of either side of the bus, numpy's, or without a head dimension."""
    P = need_gpu()
    for cache, workspace in ((P.kv4_cache(2, 2, 64, 16), P.kv4_attention_workspace), (P.kv8_cache(2, 2, 64, 16), P.kv8_attention_workspace)):
        want = workspace(torch.zeros((6, 4, 64), dtype=F16, device="cuda"), cache, 2, 3, 5000).numel()
        for q in (torch.zeros((6, 4)), np.zeros((6, 4, 64)), torch.zeros((6, 4, 1, 64), device="cuda")):
            assert workspace(q, cache, 2, 3, 5000).numel() == want


def test_sizes_below_32_bits():
    """Python's integers beyond either end of 32 bits are refused, not cut."""
    P = need_gpu()
    q, table, lens = torch.zeros((1, 2, 64), dtype=F16, device="cuda"), i32([[0, 1]]), i32([1])
    for cache, call, workspace in ((P.kv4_cache(2, 2, 64, 16), P.kv4_attention, P.kv4_attention_workspace), (P.kv8_cache(2, 2, 64, 16), P.kv8_attention, P.kv8_attention_workspace)):
        for over in (dict(max_q_len=1 - 2 ** 32), dict(max_kv_len=16 - 2 ** 32), dict(window=-2 ** 32), dict(window=8 - 2 ** 32)):
            with pytest.raises(P.InvalidArgument):
                call(q, cache, table, lens, **over)
        for a in ((1 - 2 ** 32, 1, 32), (1, 1 - 2 ** 32, 32), (1, 1, 32 - 2 ** 32)):
            with pytest.raises(P.InvalidArgument):
                workspace(q, cache, *a)


def test_read_from_what_is_no_cache():
    P = need_gpu()
    slots = i32([0])
    for bad in (torch.zeros((1, 1, 1, 8), dtype=torch.uint8, device="cuda"), torch.zeros((1, 1, 1, 100), dtype=torch.uint8, device="cuda"),
                torch.zeros((1, 1, 1, 2064), dtype=torch.uint8), torch.zeros((1, 1, 2064), dtype=torch.uint8, device="cuda")):
        with pytest.raises(P.InvalidArgument):
            P.kv8_read(bad, slots)


@TYPES
def test_scale_stays_behind_drafts(dtype):
    """A draft that raised its block's scale and is not accepted: the older rows stay as they were rounded for it, and what takes its
    place is held at that scale; neither is further from its row than half a step there, 2^-4 of a number or 2^-10 scales."""
    P = need_gpu()
    H, D = 2, 64
    gen = torch.Generator().manual_seed(12)
    table, slots = i32([[0]]), i32(range(16))
    k = [rows(gen, n, H, D, dtype) for n in (5, 3, 2)]
    k[1] = (k[1].float() * 4096).to(dtype)
    cache = P.kv8_cache(1, H, D, 16)
    scales = []
    for n, x in zip((5, 8, 7), k):
        P.kv8_write(x.cuda(), x.cuda(), cache, table, i32([n]), cu_q=i32([0, len(x)]))
        scales.append(cache[0, :, 0, 32 * D:32 * D + 8].contiguous().view(torch.float32).cpu())
    assert (scales[1] > 256 * scales[0]).all() and torch.equal(scales[1], scales[2])
    want = torch.cat((k[0], k[2])).double()
    for which, got in enumerate(P.kv8_read(cache, slots, dtype)):
        s = scales[2][:, which].double()[:, None]
        err = (got[:7].double().cpu() - want).abs()
        # (the older rows twice: at their own scale, then at this one)
        step = torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10)
        assert (err[5:] <= step[5:]).all() and (err[:5] <= step[:5] * (2 + 2.0 ** -4)).all()
        assert (err > want.abs() * 2.0 ** -4).any()      # as said: coarser
    P.kv8_write(k[0].cuda(), k[0].cuda(), cache, table, i32([5]), cu_q=i32([0, 5]))
    assert torch.equal(cache[0, :, 0, 32 * D:32 * D + 8].contiguous().view(torch.float32).cpu(), scales[0])


# ------------------------------------------------------------------ gradients: there are none

def calls_that_write(P):
    """name -> (the call, tensors that it writes)"""
    x, res, w = (torch.randn((4, 128), device="cuda").half() for _ in range(3))
    w = w[0].contiguous()
    q, k, v = (torch.randn((4, 2, 64), device="cuda").half() for _ in range(3))
    cache, table, lens, r = P.kv8_cache(4, 2, 64, 16), i32([[0], [1], [2], [3]]), i32([1, 2, 3, 4]), P.Rope(64)
    out, out8, scales = torch.empty_like(x), torch.empty((4, 128), dtype=P.E4M3, device="cuda"), torch.empty((4, 4), device="cuda")
    total, qo, ko, lse = torch.empty_like(x), torch.empty_like(q), torch.empty_like(k), torch.empty((4, 2), device="cuda")
    c4 = P.kv4_cache(4, 2, 64, 16)
    return {
        "norm": (lambda: P.rms_norm(x, w, residual=res, out=out), [res, out]),
        "norm beside": (lambda: P.rms_norm(x, w, residual=res, residual_out=total), [total]),
        "8 bits": (lambda: P.rms_norm_8bit(x, w, group=32, residual=res, out=out8, scales=scales), [res, out8, scales]),
        "rope": (lambda: P.rope(q, lens, r, k=k), [q, k]),
        "rope beside": (lambda: P.rope(q, lens, r, k=k, q_out=qo, k_out=ko), [qo, ko]),
        "write": (lambda: P.kv8_write(k, v, cache, table, lens, rope=r, q=q), [cache, q]),
        "write beside": (lambda: P.kv8_write(k, v, cache, table, lens, rope=r, q=q, q_out=qo), [cache, qo]),
        "read": (lambda: P.kv8_read(cache, i32([0, 1, 2, 3]), k_out=ko, v_out=qo), [ko, qo]),
        "attention": (lambda: P.kv8_attention(q, cache, table, lens, out=qo, lse=lse), [qo, lse]),
        "4 bits": (lambda: P.kv4_attention(q, c4, table, lens, out=qo, lse=lse), [qo, lse]),
    }, (x, res, w, q, k, v)


def test_written_tensors_are_seen_as_changed():
    """A backward pass that has saved a tensor which a call then writes raises torch's error; it does not run on the new values."""
    P = need_gpu()
    calls, _ = calls_that_write(P)
    for name, (call, written) in calls.items():
        for i, t in enumerate(written):
            if not t.dtype.is_floating_point or t.dtype == P.E4M3:
                before = t._version
                call()
                assert t._version > before, (name, i)
                continue
            leaf = torch.ones(t.shape, dtype=t.dtype, device="cuda", requires_grad=True)
            y = (leaf * t.detach()).sum()     # saves t
            call()
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()


def test_inference_tensors_are_written_anywhere():
    P = need_gpu()
    with torch.inference_mode():
        calls, _ = calls_that_write(P)
        for call, _ in calls.values():
            call()
    for call, _ in calls.values():
        call()


def test_in_place_where_gradients_flow():
    """The operators have no backward pass. In place on a tensor of a graph the rotation or the sum would be missing from the
    gradients behind it, without an error: refused, as long as gradients are recorded. Out of place a result has no graph."""
    P = need_gpu()
    calls, (x, res, w, q, k, v) = calls_that_write(P)
    for t in (res, q, k):
        t.requires_grad_()
    for name in ("norm", "8 bits", "rope", "write"):
        with pytest.raises(P.InvalidArgument, match="no backward"):
            calls[name][0]()
        with torch.no_grad():
            calls[name][0]()
    for name in ("norm beside", "rope beside", "write beside", "attention", "4 bits"):
        calls[name][0]()
    for t in (x, w, v):
        t.requires_grad_()
    with torch.no_grad():
        for t in (res, q, k):
            t.requires_grad_(False)
    assert not P.rms_norm(x, w, residual=res).requires_grad
    for name in calls:
        calls[name][0]()
    # a tensor that is no leaf, as a projection's result is
    h = (x[:, None] * 1.0).view(4, 2, 64)
    with pytest.raises(P.InvalidArgument, match="no backward"):
        P.rope(h, i32([0, 1, 2, 3]), P.Rope(64))
