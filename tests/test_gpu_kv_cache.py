"""kv_cache_write and kv_cache_read on the GPU against the definition in 64
bits: codes and scales are whole facts, so everything has to be equal."""
import math

import pytest
import torch

import cabi
import cmp_ext_b200 as cx
from seq_reference import e8m0, quantise

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def caches(pages, heads, page, d, dtype, fill=0):
    kc, vc = (torch.full((pages, heads, page, d), float(fill), device="cuda").to(dtype) for _ in range(2))
    if dtype != E4M3:
        return kc, vc, None, None
    ks, vs = (torch.full((pages, heads, page), 9, dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2))
    return kc, vc, ks, vs


def values(x, dtype):
    """What an 8-bit cache gives back for x: e4m3's value times the scale, held to dtype's finite range."""
    code, byte = quantise(x)
    top = torch.finfo(dtype).max
    return (code * e8m0(byte).unsqueeze(-1)).clamp(-top, top).to(dtype)


def same(a, b):
    a, b = a.double(), b.double()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("q8", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("tokens,heads,d,page", [(1, 1, 64, 16), (100, 2, 128, 16), (37, 3, 96, 1), (64, 8, 128, 64),
                                                 (9, 2, 7, 5), (33, 1, 512, 8), (50, 5, 80, 48), (300, 2, 256, 128)])
def test_write_and_read(cuda, tokens, heads, d, page, dtype, q8):
    pages = -(-tokens // page) + 2
    g = gen(tokens + d)
    qkv = torch.randn(tokens, 4 * heads, d, generator=g, device="cuda")
    qkv = (qkv * 2.0 ** torch.randint(-12, 6, (tokens, 4 * heads, 1), generator=g, device="cuda")).to(dtype)
    k, v = qkv[:, heads : 2 * heads], qkv[:, 3 * heads :]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    kc, vc, ks, vs = caches(pages, heads, page, d, E4M3 if q8 else dtype, fill=2)
    before = [x.clone() if x is not None else None for x in (kc, vc, ks, vs)]
    cx.kv_cache_write(k, v, kc, vc, slots, ks, vs)
    back = cx.kv_cache_read(kc, vc, slots, ks, vs, dtype=dtype)
    torch.cuda.synchronize()
    page_of, row = slots // page, slots % page
    untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    untouched[page_of, row] = False
    for x, cache, scale, old, old_scale, got in ((k, kc, ks, before[0], before[2], back[0]),
                                                 (v, vc, vs, before[1], before[3], back[1])):
        held = cache.view(torch.uint8 if q8 else cache.dtype).transpose(1, 2)[page_of, row].view(cache.dtype)
        if q8:
            code, byte = quantise(x)
            assert same(held, code)
            assert torch.equal(scale.view(torch.uint8).transpose(1, 2)[page_of, row], byte)
            assert same(got, values(x, dtype))
            assert torch.equal(scale.view(torch.uint8).transpose(1, 2)[untouched],
                               old_scale.view(torch.uint8).transpose(1, 2)[untouched])
        else:
            assert torch.equal(held, x) and torch.equal(got, x)
        assert torch.equal(cache.view(torch.uint8).transpose(1, 2)[untouched], old.view(torch.uint8).transpose(1, 2)[untouched])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_scale_borders_and_bad_values(cuda, dtype):
    """Largest magnitudes on both sides of each border of the scale, ties of
    e4m3, zeros, subnormals, the type's ends, infinities and NaN."""
    info = torch.finfo(dtype)
    tops = [448.0, 449.0 if dtype == F32 else 450.0, 1.75, 1.76, 0.875, 1.0, 2.0**-9 * 1.75, info.max, info.tiny,
            info.tiny / 4, 0.0, 2.0**-120 if dtype != F16 else 2.0**-24, 3.5, 3.51]
    x = torch.zeros(len(tops) + 4, 1, 64, device="cuda", dtype=dtype)
    ramp = torch.linspace(-1, 1, 63, device="cuda", dtype=torch.float64)
    for i, t in enumerate(tops):
        x[i, 0, 1:] = (ramp * t).to(dtype)
        x[i, 0, 0] = t
    n = len(tops)
    x[n, 0, :32] = torch.arange(32, device="cuda") * 2.0**-5 + 16  # half-way cases of 4 significant bits
    x[n, 0, 32] = 448
    x[n + 1, 0, 3], x[n + 2, 0, 60], x[n + 3, 0, 0] = math.nan, math.inf, -math.inf
    x[n + 1 :, 0, 7] = 1.5
    kc, vc, ks, vs = caches(8, 1, 4, 64, E4M3)
    slots = torch.arange(len(x), device="cuda")
    cx.kv_cache_write(x, -x, kc, vc, slots, ks, vs)
    for out, want in zip(cx.kv_cache_read(kc, vc, slots, ks, vs, dtype=dtype), (x, -x)):
        assert same(out, values(want, dtype))
        assert out[n + 1 :].isnan().all()
    assert torch.equal(ks.view(torch.uint8).view(-1)[: len(x)], quantise(x)[1].view(-1))
    assert same(kc.view(-1, 64)[: len(x)], quantise(x)[0].view(-1, 64))


@pytest.mark.parametrize("dtype,held", [(BF16, E4M3), (F16, F16)])
def test_slots_outside_the_cache(cuda, dtype, held):
    kc, vc, ks, vs = caches(3, 2, 8, 64, held, fill=1)
    x = torch.randn(6, 2, 64, generator=gen(1), device="cuda").to(dtype)
    slots = torch.tensor([-1, 5, 24, 2**40, -(2**40), 23], device="cuda")
    cx.kv_cache_write(x, x, kc, vc, slots, ks, vs)
    k, v = cx.kv_cache_read(kc, vc, slots, ks, vs, dtype=dtype)
    torch.cuda.synchronize()
    out = torch.tensor([0, 2, 3, 4], device="cuda")
    assert not k[out].any() and not v[out].any()
    assert k[[1, 5]].any() and (kc.float() == 1).sum() == kc.numel() - 2 * 2 * 64 + (kc[[0, 2], :, [5, 7]].float() == 1).sum()


@pytest.mark.parametrize("held", [E4M3, BF16])
def test_strided_caches(cuda, held):
    """Token-major pages and both caches in one tensor; an odd address and row length."""
    x, y = (torch.randn(20, 2, 64, generator=gen(s), device="cuda").to(BF16) for s in (1, 2))
    slots = torch.randperm(32, generator=gen(3), device="cuda")[:20]
    plain = caches(4, 2, 8, 64, held)
    cx.kv_cache_write(x, y, plain[0], plain[1], slots, plain[2], plain[3])
    want = cx.kv_cache_read(plain[0], plain[1], slots, plain[2], plain[3])
    for room in (torch.zeros(4, 8, 2, 2, 64, device="cuda").to(held).permute(3, 0, 2, 1, 4),
                 torch.zeros(2, 4, 2, 8, 67, device="cuda").to(held)[..., 3:]):
        kc, vc = room[0], room[1]
        ks, vs = (t.transpose(1, 2).contiguous().transpose(1, 2) if t is not None else None for t in plain[2:])
        cx.kv_cache_write(x, y, kc, vc, slots, ks, vs)
        got = cx.kv_cache_read(kc, vc, slots, ks, vs)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    flat = x.transpose(1, 2).contiguous().transpose(1, 2)  # stride of the last dimension is not 1
    other = caches(4, 2, 8, 64, held)
    cx.kv_cache_write(flat, y, other[0], other[1], slots, other[2], other[3])
    torch.cuda.synchronize()
    assert torch.equal(other[0].view(torch.uint8), plain[0].view(torch.uint8))


def test_empty_and_default_dtype(cuda):
    kc, vc, ks, vs = caches(2, 2, 8, 64, E4M3)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    cx.kv_cache_write(torch.empty(0, 2, 64, dtype=F16, device="cuda"), torch.empty(0, 2, 64, dtype=F16, device="cuda"),
                      kc, vc, none, ks, vs)
    k, v = cx.kv_cache_read(kc, vc, none, ks, vs)
    assert k.shape == v.shape == (0, 2, 64) and k.dtype == BF16
    x = torch.ones(3, 2, 64, dtype=F16, device="cuda")
    slots = torch.arange(3, device="cuda")
    cx.kv_cache_write(x, x, kc[:0], vc[:0], slots, ks[:0], vs[:0])  # no pages: every slot is outside
    assert not cx.kv_cache_read(kc[:0], vc[:0], slots, ks[:0], vs[:0])[0].any()
    torch.cuda.synchronize()
    assert cabi.device_error() == 0


def test_graph_and_side_stream(cuda):
    kc, vc, ks, vs = caches(8, 2, 16, 128, E4M3)
    x = torch.randn(40, 2, 128, generator=gen(4), device="cuda").to(BF16)
    slots = torch.arange(40, device="cuda")
    cx.kv_cache_write(x, x, kc, vc, slots, ks, vs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cx.kv_cache_write(x, x, kc, vc, slots, ks, vs)
        k, v = cx.kv_cache_read(kc, vc, slots, ks, vs)
    x.mul_(3)
    slots.add_(50)
    g.replay()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        k2, v2 = cx.kv_cache_read(kc, vc, slots, ks, vs)
    torch.cuda.synchronize()
    assert torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(k, v)
    assert same(k, values(x, BF16))
