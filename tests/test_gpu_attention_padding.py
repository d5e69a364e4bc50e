"""Padded batches: tokens outside every sequence, as a captured call has them.
Their rows are zeros in a new output, whatever the allocator left there, and
cost about what writing them costs."""
import math

import pytest
import torch

import cabi
import cmp_ext_b200 as cx
from seq_reference import U, attend, check

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def cu(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def qkv(tokens, hq, hkv, d, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, hq + 2 * hkv, d, generator=g, device="cuda").to(dtype)
    return x[:, :hq], x[:, hq : hq + hkv], x[:, hq + hkv :]


@pytest.mark.parametrize("path", ["tc", "skinny", "simt"])
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (7, 1, 128), (128, 1, 64), (6, 2, 64)])
@pytest.mark.parametrize("first,used,total", [(0, 300, 1500), (700, 130, 1001), (5, 0, 777), (900, 1, 901)])
def test_rows_outside_are_zeros(cuda, first, used, total, hq, hkv, d, path):
    q, k, v = qkv(total, hq, hkv, d, BF16, total)
    at = cu(first, first + used)
    size = total * hq * d
    junk = torch.full((size,), math.nan, dtype=BF16, device="cuda")  # what the next allocation of that size gets
    cx._set_path(path)
    try:
        del junk
        out = cx.attention_varlen(q, k, v, at)
    finally:
        cx._set_path("auto")
    torch.cuda.synchronize()
    assert cabi.device_error() == 0
    assert not out[:first].any() and not out[first + used :].any()
    sees = slice(first, first + min(used, 40))
    rows = out[sees]
    want, tol = attend(q[sees], k[sees], v[sees], 1 / math.sqrt(d), True, U[BF16], U[BF16])
    check(rows, want, tol, "the sequence")


@pytest.mark.parametrize("total,used", [(16384, 300), (65536, 64)])
def test_padding_costs_what_writing_it_costs(cuda, total, used):
    q, k, v = qkv(total, 32, 8, 128, BF16, 1)
    at = cu(0, used)

    def best(f):
        times = []
        for _ in range(7):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            f()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    out = torch.empty(total, 32, 128, dtype=BF16, device="cuda")
    written = best(lambda: out.zero_())
    whole = best(lambda: cx.attention_varlen(q, k, v, at))
    alone = best(lambda: cx.attention_varlen(q, k, v, at, out=out))  # rows outside are left as they were
    print(f"{total} tokens, {used} used: {whole:.3f} ms, {alone:.3f} without zeros, writing zeros {written:.3f}")
    assert whole <= alone + 4 * written + 0.05


@pytest.mark.parametrize("path", ["tc", "skinny", "simt"])
@pytest.mark.parametrize("batch,width", [(9, 40), (400, 40), (100000, 1024)])
def test_offsets_that_do_not_ascend(cuda, batch, width, path):
    """The same 64 tokens named again and again, with more work in them than 32
    bits count: no access outside, no endless call, and later calls are right."""
    hq, hkv, d, page, t = 32, 8, 64, 64, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    kc, vc = (torch.randn(width, hkv, page, d, generator=g, device="cuda").to(F16) for _ in range(2))
    q = torch.randn(t, hq, d, generator=g, device="cuda").to(F16)
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, width).expand(batch, width)
    lens = torch.full((batch,), width * page, dtype=torch.int32, device="cuda")
    at = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    at[1::2] = t
    cx._set_path(path)
    try:
        cx.attention_paged(q, kc, vc, table, lens, cu_seqlens_q=at)
        cx.attention_varlen(q, *(x.reshape(-1, hkv, d)[:t].contiguous() for x in (kc, vc)), at)
        torch.cuda.synchronize()
        assert cabi.device_error() == 0
        out = cx.attention_paged(q[:3], kc, vc, table[:3, :2], torch.tensor([100, 5, 128], dtype=torch.int32, device="cuda"))
    finally:
        cx._set_path("auto")
    torch.cuda.synchronize()
    keys = kc[:2].transpose(1, 2).reshape(-1, hkv, d), vc[:2].transpose(1, 2).reshape(-1, hkv, d)
    for i, n in enumerate((100, 5, 128)):
        want, tol = attend(q[i : i + 1], keys[0][:n], keys[1][:n], 1 / math.sqrt(d), True, U[F16], U[F16])
        check(out[i : i + 1], want, tol, f"row {i}")


@pytest.mark.parametrize("path", ["tc", "skinny", "simt"])
def test_a_captured_padded_batch(cuda, path):
    """One graph, replayed with other lengths: rows that a longer batch wrote are zeros again in a shorter one."""
    total = 700
    q, k, v = qkv(total, 8, 2, 64, BF16, 3)
    at = cu(0, 300, 650)
    cx._set_path(path)
    try:
        cx.attention_varlen(q, k, v, at)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = cx.attention_varlen(q, k, v, at)
        for offsets in ((0, 300, 650), (0, 10, 11), (200, 200, 700), (0, 0, 0), (50, 400, 401), (0, 699, 700)):
            at.copy_(torch.tensor(offsets, dtype=torch.int32))
            g.replay()
            torch.cuda.synchronize()
            assert cabi.device_error() == 0
            assert torch.equal(out, cx.attention_varlen(q, k, v, at))
            assert not out[: offsets[0]].any() and not out[offsets[2] :].any()
            for a, b in zip(offsets, offsets[1:]):
                n = min(b - a, 20)
                want, tol = attend(q[a : a + n], k[a : a + n], v[a : a + n], 1 / 8, True, U[BF16], U[BF16])
                check(out[a : a + n], want, tol, f"{offsets}")
    finally:
        cx._set_path("auto")
