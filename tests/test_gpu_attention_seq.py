"""attention_varlen and attention_paged on the GPU against softmax attention
in 64 bits (seq_reference.attend, which derives the bound on rounding), on
every kernel that takes the case; lengths, masks, layouts, streams and graphs
where such kernels go wrong."""
import contextlib
import math
import random

import pytest
import torch

import cabi
import cmp_ext_b200 as cx
from seq_reference import U, attend, check, e8m0, quantise

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


PATHS = ["auto", "simt", "tc", "skinny"]


def takes(path, dtype, d, page=8):
    """Whether a forced kernel takes the case (the tensor-core ones: 16-bit, D 64 or 128, pages of 8, 16, 32, ... keys)."""
    return path in ("auto", "simt") or (dtype != F32 and d in (64, 128) and page >= 8 and page & (page - 1) == 0)


@contextlib.contextmanager
def forced(path):
    cx._set_path(path)
    try:
        yield
    finally:
        cx._set_path("auto")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def cu_of(lens, first=0):
    out = [first]
    for x in lens:
        out.append(out[-1] + x)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def finish():
    torch.cuda.synchronize()
    assert cabi.device_error() == 0


# ---------------------------------------------------------------- packed sequences
def qkv(tokens, hq, hkv, d, dtype, seed):
    x = torch.randn(tokens, hq + 2 * hkv, d, generator=gen(seed), device="cuda").to(dtype)
    return x[:, :hq], x[:, hq : hq + hkv], x[:, hq + hkv :]  # views of one projection, as models have them


def check_varlen(got, q, k, v, cu_q, cu_k, causal, scale, what):
    a, b = cu_q.tolist(), cu_k.tolist()
    for i in range(len(a) - 1):
        want, tol = attend(q[a[i] : a[i + 1]], k[b[i] : b[i + 1]], v[b[i] : b[i + 1]], scale, causal,
                           0.0 if q.dtype == F32 else U[q.dtype], U[q.dtype])
        check(got[a[i] : a[i + 1]], want, tol, f"{what}, sequence {i} of {a[i + 1] - a[i]} tokens")


LENS = {
    "one": [1],
    "edges": [0, 1, 127, 128, 129, 0, 2],
    "tiles": [256, 257, 63, 64, 65],
    "long": [700],
    "many": [3] * 40 + [17, 0, 31],
}


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d,hq,hkv", [(F16, 64, 4, 4), (BF16, 128, 8, 2), (BF16, 64, 7, 1), (F16, 128, 6, 2),
                                            (F32, 64, 2, 1), (BF16, 80, 4, 2), (F16, 128, 5, 1)])
@pytest.mark.parametrize("lens", list(LENS))
def test_varlen(cuda, lens, dtype, d, hq, hkv, causal, path):
    lens = LENS[lens]
    if not takes(path, dtype, d):
        pytest.skip("not this kernel's")
    q, k, v = qkv(sum(lens), hq, hkv, d, dtype, seed=sum(lens) + d)
    cu = cu_of(lens)
    with forced(path):
        out = cx.attention_varlen(q, k, v, cu, causal=causal)
    finish()
    check_varlen(out, q, k, v, cu, cu, causal, 1 / math.sqrt(d), "varlen")


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F32, 40)])
@pytest.mark.parametrize("causal", [True, False])
def test_varlen_other_key_lengths(cuda, dtype, d, causal, path):
    """More keys than queries, fewer (rows that see nothing), none."""
    if not takes(path, dtype, d):
        pytest.skip("not this kernel's")
    n, length = [5, 130, 40, 3, 200, 1], [300, 7, 0, 3, 129, 1000]
    q, _, _ = qkv(sum(n), 4, 2, d, dtype, 1)
    _, k, v = qkv(sum(length), 4, 2, d, dtype, 2)
    cu_q, cu_k = cu_of(n), cu_of(length)
    with forced(path):
        out = cx.attention_varlen(q, k, v, cu_q, cu_k, causal=causal, scale=-0.2)
    finish()
    check_varlen(out, q, k, v, cu_q, cu_k, causal, -0.2, "varlen")
    assert not out[cu_q[2] : cu_q[3]].any()  # no keys: zeros


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F32, 64)])
def test_varlen_rest_and_garbage_between(cuda, dtype, d):
    """Tokens before the first and behind the last sequence: zeros in a new
    output, left alone in a given one; NaN there never reaches a sequence."""
    lens, first, total = [100, 3, 250], 9, 420
    q, k, v = (x.clone() for x in qkv(total, 8, 2, d, dtype, 3))
    cu = cu_of(lens, first)
    end = first + sum(lens)
    for x in (q, k, v):
        x[:first] = math.nan
        x[end:] = math.inf
    k[end + 1 :] = math.nan
    out = cx.attention_varlen(q, k, v, cu)
    finish()
    check_varlen(out, q, k, v, cu, cu, True, 1 / math.sqrt(d), "varlen")
    assert not out[:first].any() and not out[end:].any()
    given = torch.full_like(out, 7.0)
    assert cx.attention_varlen(q, k, v, cu, out=given) is not None
    finish()
    assert torch.equal(given[first:end], out[first:end])
    assert (given[:first] == 7).all() and (given[end:] == 7).all()


@pytest.mark.parametrize("dtype,d,hq,hkv", [(F16, 64, 4, 4), (BF16, 128, 8, 1), (F32, 64, 2, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("path", PATHS)
def test_varlen_bad_values_stay_with_their_keys(cuda, dtype, d, hq, hkv, bad, path):
    """A key or value that is not finite reaches the rows that see it and no
    other.  Other sequences, and every row a bad key is hidden from, keep their
    bits; rows a bad value is hidden from may be summed in another order (the
    bound holds for them)."""
    lens, at = [150, 60], 97
    if not takes(path, dtype, d):
        pytest.skip("not this kernel's")

    def run():
        with forced(path):
            return cx.attention_varlen(q, k, v, cu_of(lens))

    q, k, v = (x.clone() for x in qkv(210, hq, hkv, d, dtype, 4))
    clean = run()
    v[at, 0, 5] = bad
    out = run()
    finish()
    check_varlen(out, q, k, v, cu_of(lens), cu_of(lens), True, 1 / math.sqrt(d), "value")
    assert out[:at].isfinite().all() and torch.equal(out[150:], clean[150:])
    v[at, 0, 5] = 0
    k[at] = bad
    out = run()
    finish()
    assert torch.equal(out[:at], clean[:at]) and torch.equal(out[150:], clean[150:])


def test_varlen_strides_and_out(cuda):
    """Heads-first storage, an odd address, a strided output."""
    q, k, v = qkv(90, 4, 2, 64, BF16, 5)
    cu = cu_of([90])
    want = cx.attention_varlen(q, k, v, cu)
    turned = [x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v)]
    assert torch.equal(cx.attention_varlen(*turned, cu), want)
    shifted = []
    for x in (q, k, v):
        room = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        shifted.append(room[1:].view(x.shape).copy_(x))
    assert torch.equal(cx.attention_varlen(*shifted, cu), want)
    last = [x.permute(0, 2, 1).contiguous().permute(0, 2, 1) for x in (q, k, v)]
    assert torch.equal(cx.attention_varlen(*last, cu), want)
    room = torch.full((90, 3, 4, 65), 3.0, dtype=BF16, device="cuda")
    out = room[:, 1, :, 1:]
    got = cx.attention_varlen(q, k, v, cu, out=out)
    finish()
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    assert (room[:, 0] == 3).all() and (room[:, 2] == 3).all() and (room[:, 1, :, 0] == 3).all()


def test_varlen_refusals(cuda):
    q, k, v = qkv(8, 4, 2, 64, BF16, 6)
    cu = cu_of([8])
    with pytest.raises(RuntimeError, match="out must not overlap an input"):
        cx.attention_varlen(q, k, v, cu, out=q)
    with pytest.raises(RuntimeError, match="out must have the query's dtype"):
        cx.attention_varlen(q, k, v, cu, out=torch.empty(8, 4, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="out must not overlap itself"):
        cx.attention_varlen(q, k, v, cu, out=torch.empty(1, 4, 64, dtype=BF16, device="cuda").expand(8, 4, 64))
    with pytest.raises(RuntimeError, match="Device mismatch"):
        cx.attention_varlen(q, k, v, cu.cpu())
    wide = torch.zeros(8, 2, 520, device="cuda")
    with pytest.raises(RuntimeError, match="unsupported"):
        cx.attention_varlen(wide, wide, wide, cu)


def test_varlen_empty(cuda):
    q, k, v = qkv(0, 4, 2, 64, BF16, 7)
    assert cx.attention_varlen(q, k, v, cu_of([0, 0])).shape == (0, 4, 64)
    q, k, v = qkv(5, 4, 2, 64, BF16, 7)
    assert not cx.attention_varlen(q, k, v, cu_of([])).any()  # no sequences: every row is outside
    assert not cx.attention_varlen(q, k[:0], v[:0], cu_of([5]), cu_of([0])).any()
    finish()


def test_varlen_lengths_out_of_range_are_clamped(cuda):
    q, k, v = qkv(64, 4, 2, 64, BF16, 8)
    for cu in ([0, 1000], [-5, 64], [40, 10], [-(2**31), 2**31 - 1], [70, 90]):
        out = cx.attention_varlen(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        finish()
        assert out.isfinite().all()
    want = cx.attention_varlen(q, k, v, cu_of([64]))
    assert torch.equal(cx.attention_varlen(q, k, v, torch.tensor([0, 1000], dtype=torch.int32, device="cuda")), want)


# ---------------------------------------------------------------- paged cache
class Paged:
    """A cache whose unused slots hold `rest`, with K / V of each sequence."""

    def __init__(self, lens, page, hkv, d, dtype, kv="same", seed=0, rest=math.nan, nhd=False, extra=3):
        g = gen(seed)
        need = [-(-x // page) for x in lens]
        pages = sum(need) + extra
        order = torch.randperm(pages, generator=g, device="cuda")
        self.table = torch.full((len(lens), max(need + [0]) + 1), -7, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        shape = (pages, hkv, page, d)
        held = torch.float32 if kv == "e4m3" else dtype
        kc, vc = (torch.full(shape, rest, device="cuda", dtype=held) for _ in range(2))
        self.keys, self.values, at = [], [], 0
        for b, x in enumerate(lens):
            mine = order[at : at + need[b]]
            at += need[b]
            self.table[b, : need[b]] = mine.int()
            k, v = (torch.randn(x, hkv, d, generator=g, device="cuda").to(dtype) for _ in range(2))
            v *= 2.0 ** torch.randint(-3, 4, (x, hkv, 1), generator=g, device="cuda")  # scales that differ
            j = torch.arange(x, device="cuda")
            kc[mine[j // page], :, j % page], vc[mine[j // page], :, j % page] = k.to(held), v.to(held)
            self.keys.append(k)
            self.values.append(v)
        self.ks = self.vs = None
        if kv == "e4m3":
            (kc, self.ks), (vc, self.vs) = (self.coded(x) for x in (kc, vc))
            back = [(quantise(k), quantise(v)) for k, v in zip(self.keys, self.values)]
            self.keys = [a[0] * e8m0(a[1]).unsqueeze(-1) for a, _ in back]
            self.values = [b[0] * e8m0(b[1]).unsqueeze(-1) for _, b in back]
        if nhd:
            kc, vc = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))
        self.kc, self.vc = kc, vc

    @staticmethod
    def coded(x):
        y, b = quantise(x)
        return y.float().to(E4M3), b.view(E8M0)

    def run(self, q, **kw):
        return cx.attention_paged(q, self.kc, self.vc, self.table, self.lens, key_scale=self.ks, value_scale=self.vs, **kw)

    def check(self, got, q, cu, causal, scale, what="paged", sequences=None):
        a = cu.tolist()
        u_w = 0.0 if q.dtype == F32 else max(U[q.dtype], U[BF16] if self.ks is not None else 0.0)
        for b in sequences if sequences is not None else range(len(a) - 1):
            want, tol = attend(q[a[b] : a[b + 1]], self.keys[b], self.values[b], scale, causal, u_w, U[q.dtype])
            check(got[a[b] : a[b + 1]], want, tol, f"{what}, sequence {b}")


def queries(n, hq, d, dtype, seed=1):
    return torch.randn(n, hq, d, generator=gen(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("kv", ["same", "e4m3"])
@pytest.mark.parametrize("dtype,d,hq,hkv,page", [(F16, 64, 4, 4, 16), (BF16, 128, 8, 2, 32), (BF16, 128, 16, 1, 64),
                                                 (F16, 128, 6, 2, 128), (BF16, 64, 32, 2, 256), (F16, 64, 5, 1, 8),
                                                 (F32, 64, 4, 2, 16), (BF16, 96, 4, 2, 16), (F16, 128, 4, 2, 48),
                                                 (BF16, 64, 3, 3, 1)])
def test_paged_single_tokens(cuda, dtype, d, hq, hkv, page, kv):
    lens = [1, 15, 16, 17, 63, 64, 65, 128, 300, 0, 777, 2]
    c = Paged(lens, page, hkv, d, dtype, kv, seed=page + d)
    q = queries(len(lens), hq, d, dtype)
    out = c.run(q)
    finish()
    c.check(out, q, cu_of([1] * len(lens)), True, 1 / math.sqrt(d))
    assert not out[9].any()
    # with the offsets spelled out, and with a longest length that is not true: the same rows
    assert torch.equal(c.run(q, cu_seqlens_q=cu_of([1] * len(lens)), max_seqlen_q=1), out)


@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("kv", ["same", "e4m3"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d,hq,hkv,page", [(F16, 64, 4, 4, 16), (BF16, 128, 8, 2, 32), (F16, 128, 7, 1, 64),
                                                 (BF16, 64, 6, 2, 128), (F32, 64, 4, 2, 16), (F16, 128, 4, 2, 24)])
def test_paged_chunks(cuda, dtype, d, hq, hkv, page, causal, kv, path):
    """Chunks of several lengths in one call: a first chunk (all keys new),
    later ones, single tokens, none, more queries than keys."""
    if not takes(path, dtype, d, page):
        pytest.skip("not this kernel's")
    n = [40, 1, 130, 0, 3, 70, 20, 1]
    lens = [40, 500, 333, 64, 1030, 71, 5, 1]
    c = Paged(lens, page, hkv, d, dtype, kv, seed=d + hq)
    q, cu = queries(sum(n), hq, d, dtype), cu_of(n)
    with forced(path):
        out = c.run(q, cu_seqlens_q=cu, causal=causal, max_seqlen_q=max(n))
        finish()
        c.check(out, q, cu, causal, 1 / math.sqrt(d))
        for hint in (None, 1, 1000):  # a hint changes the kernel at most, never what is right
            got = c.run(q, cu_seqlens_q=cu, causal=causal, max_seqlen_q=hint)
            finish()
            c.check(got, q, cu, causal, 1 / math.sqrt(d), f"hint {hint}")


@pytest.mark.parametrize("kv", ["same", "e4m3"])
@pytest.mark.parametrize("n", [1, 2, 5, 33])
def test_paged_long_context(cuda, n, kv):
    """One sequence over many thread blocks' keys, and short ones beside it."""
    lens = [9001, 33, 4000, 40]
    c = Paged(lens, 64, 2, 128, BF16, kv, seed=n)
    q, cu = queries(n * 4, 8, 128, BF16), cu_of([n] * 4)
    out = c.run(q)
    finish()
    c.check(out, q, cu, True, 1 / math.sqrt(128))
    for _ in range(3):  # the same bits each time
        assert torch.equal(c.run(q), out)


@pytest.mark.parametrize("kv", ["same", "e4m3"])
@pytest.mark.parametrize("n", [1, 30])
def test_paged_rest_values_do_not_matter(cuda, n, kv):
    """Unused slots of the last page hold anything: the same bits come out."""
    lens = [45, 129, 700]
    outs = []
    for rest in (0.0, math.nan, math.inf):
        c = Paged(lens, 32, 2, 128, F16, kv, seed=5, rest=rest)
        outs.append(c.run(queries(3 * n, 4, 128, F16)))
    finish()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("kv", ["same", "e4m3"])
@pytest.mark.parametrize("n", [1, 20])
def test_paged_layouts(cuda, n, kv):
    """Token-major pages, a strided page table, a cache that is a slice of a larger one."""
    lens = [100, 31, 260]
    c = Paged(lens, 16, 4, 64, BF16, kv, seed=6)
    q = queries(3 * n, 8, 64, BF16)
    want = c.run(q)
    t = Paged(lens, 16, 4, 64, BF16, kv, seed=6, nhd=True)
    assert torch.equal(t.run(q), want)
    both = torch.stack((c.kc.view(torch.uint8), c.vc.view(torch.uint8)), 1)
    c.kc, c.vc = (both[:, i].view(c.kc.dtype) for i in range(2))
    wide = torch.full((3, 2 * c.table.shape[1]), 5, dtype=torch.int32, device="cuda")
    wide[:, ::2] = c.table
    c.table = wide[:, ::2]
    assert torch.equal(c.run(q), want)
    finish()


@pytest.mark.parametrize("n", [1, 24])
def test_paged_bad_pages_read_as_zeros(cuda, n):
    c = Paged([200, 64], 16, 2, 64, F16, seed=7)
    q = queries(2 * n, 4, 64, F16)
    c.table[0, 3], c.table[0, 7] = -1, 10**6
    for x in (c.keys, c.values):
        x[0][48:64] = 0
        x[0][112:128] = 0
    out = c.run(q)
    finish()
    c.check(out, q, cu_of([n, n]), True, 1 / 8)


def test_paged_lengths_out_of_range_are_clamped(cuda):
    c = Paged([64, 64], 16, 2, 64, F16, seed=8, rest=0.0)
    q = queries(2, 4, 64, F16)
    room = c.table.shape[1] * 16
    for bad in ([-1, 64], [2**31 - 1, 64], [room + 5, 64]):
        lens = torch.tensor(bad, dtype=torch.int32, device="cuda")
        out = cx.attention_paged(q, c.kc, c.vc, c.table, lens)
        finish()
        assert torch.equal(out[1], c.run(q)[1]) and out.isfinite().all()


@pytest.mark.parametrize("dtype,kv", [(F16, "same"), (BF16, "same"), (BF16, "e4m3"), (F16, "e4m3")])
@pytest.mark.parametrize("n", [1, 40])
def test_paged_extreme_values(cuda, dtype, kv, n):
    """Large scores of both signs, keys of the type's lowest value, values far
    from one, rows whose scores are all -inf."""
    lens = [300, 90]
    c = Paged(lens, 16, 2, 64, dtype, kv, seed=9, rest=0.0)
    q = queries(2 * n, 4, 64, dtype) * 8
    cu = cu_of([n, n])
    for scale in (1.0, -1.0, 0.0):
        out = c.run(q, scale=scale)
        finish()
        c.check(out, q, cu, True, scale, f"scale {scale}")
    if kv == "same":
        low = torch.finfo(dtype).min
        ones = torch.ones_like(q)
        page = int(c.table[0, 2])
        c.kc[page] = low
        c.keys[0][32:48] = low
        out = c.run(ones, scale=0.125)
        finish()
        c.check(out, ones, cu, True, 0.125, "lowest values")
        c.kc.fill_(-math.inf)
        assert not c.run(ones, scale=0.125).any()
        finish()


def test_paged_beyond_32_bit_offsets(cuda):
    """Pages whose first element lies past 2^32."""
    page, hkv, d = 64, 8, 128
    pages = 2**32 // (page * hkv * d) + 40
    kc, vc = (torch.zeros(pages, hkv, page, d, dtype=torch.uint8, device="cuda").view(E4M3) for _ in range(2))
    ks, vs = (torch.full((pages, hkv, page), 127, dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2))
    small = Paged([600], page, hkv, d, BF16, "e4m3", seed=10, rest=0.0)
    used = int((small.lens[0] + page - 1) // page)
    rows = small.table[0, :used].long()
    far = torch.arange(pages - used, pages, device="cuda")
    for big, src in ((kc, small.kc), (vc, small.vc), (ks, small.ks), (vs, small.vs)):
        big.view(torch.uint8)[far] = src.view(torch.uint8)[rows]
    # a table of the same width: the split of the keys, and with it the bits, may depend on that
    table = torch.full_like(small.table, -7)
    table[0, :used] = far.int()
    for n in (1, 50):
        q = queries(n, 16, d, BF16)
        got = cx.attention_paged(q, kc, vc, table, small.lens, key_scale=ks, value_scale=vs)
        finish()
        small.check(got, q, cu_of([n]), True, 1 / math.sqrt(d))
        assert torch.equal(got, small.run(q))
    slots = far[0] * page + torch.arange(70, device="cuda")
    k, v = cx.kv_cache_read(kc, vc, slots, ks, vs)
    cx.kv_cache_write(v, k, kc, vc, slots, ks, vs)
    k2, v2 = cx.kv_cache_read(kc, vc, slots, ks, vs)
    finish()
    assert torch.equal(k2, v) and torch.equal(v2, k)


@pytest.mark.parametrize("n", [1, 6, 40])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_paged_bad_tokens_of_an_8_bit_cache(cuda, n, dtype, bad):
    """A token whose key or value held a NaN or an infinity reads back as NaN:
    rows that see it are NaN in that kv head, the others keep the bound."""
    length, at, hkv = 210, 205, 2
    c = Paged([length], 16, hkv, 64, dtype, "e4m3", seed=14, rest=0.0)
    q = queries(n, 4, 64, dtype)
    slot = c.table[0, at // 16].long() * 16 + at % 16
    k, v = (torch.randn(1, hkv, 64, generator=gen(15), device="cuda").to(dtype) for _ in range(2))
    for side in range(2):
        kk, vv = k.clone(), v.clone()
        (kk, vv)[side][0, 1, 7] = bad
        cx.kv_cache_write(kk, vv, c.kc, c.vc, slot.view(1), c.ks, c.vs)
        for x, held in ((kk, c.keys), (vv, c.values)):
            code, byte = quantise(x)
            held[0][at] = (code * e8m0(byte).unsqueeze(-1))[0]
        out = c.run(q)
        finish()
        sees = torch.arange(n, device="cuda") + length - n >= at
        assert out[sees][:, 2:].isnan().all() and out[sees][:, :2].isfinite().all()
        assert out[~sees].isfinite().all()
        c.check(out, q, cu_of([n]), True, 1 / 8)


def test_workspace_errors_of_the_c_abi(cuda):
    import ctypes

    q = torch.zeros(1, 8, 128, dtype=BF16, device="cuda")
    kc = torch.zeros(64, 2, 64, 128, dtype=BF16, device="cuda")
    table, lens = torch.arange(64, dtype=torch.int32, device="cuda"), torch.tensor([4000], dtype=torch.int32, device="cuda")
    a = cabi.AttentionSeqArgs()
    a.dtype = a.kv_dtype = cabi.BF16
    a.Q, a.K, a.V, a.O = q.data_ptr(), kc.data_ptr(), kc.data_ptr(), torch.empty_like(q).data_ptr()
    a.batch, a.tokens_q, a.heads_q, a.heads_kv, a.head_dim = 1, 1, 8, 2, 128
    a.q_stride_token = a.o_stride_token = 1024
    a.q_stride_head = a.o_stride_head = a.k_stride_row = a.v_stride_row = 128
    a.k_stride_head = a.v_stride_head = 64 * 128
    a.k_stride_page = a.v_stride_page = 2 * 64 * 128
    a.page_table, a.seqlens_k, a.max_pages, a.pages, a.page_size = table.data_ptr(), lens.data_ptr(), 64, 64, 64
    a.page_table_stride, a.scale, a.causal = 64, 0.1, 1
    need = cabi.lib().cmpx_attention_seq_workspace_size(ctypes.byref(a))
    assert need > 0
    call = lambda: cabi.lib().cmpx_attention_seq(ctypes.byref(a), None)  # noqa: E731
    assert call() == cabi.ERR_INVALID_ARG  # none
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need - 1
    assert call() == cabi.ERR_WORKSPACE
    a.workspace_bytes = need
    assert call() == cabi.OK
    a.workspace = ws.data_ptr() + 4
    assert call() == cabi.ERR_INVALID_ARG  # not on 16 bytes
    finish()


# ---------------------------------------------------------------- streams, graphs, threads
def test_streams_and_concurrent_calls(cuda):
    c = Paged([5000, 4000, 100], 64, 2, 128, BF16, "e4m3", seed=11)
    q1, q2 = queries(3, 8, 128, BF16, 1), queries(120, 8, 128, BF16, 2)
    p = qkv(600, 8, 2, 128, BF16, 3)
    cu = cu_of([599, 1])
    want = [c.run(q1), c.run(q2), cx.attention_varlen(*p, cu)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[] for _ in range(3)]
    for _ in range(5):
        for i, f in enumerate((lambda: c.run(q1), lambda: c.run(q2), lambda: cx.attention_varlen(*p, cu))):
            with torch.cuda.stream(streams[i]):
                got[i].append(f())
    finish()
    for i in range(3):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_graphs_follow_their_inputs(cuda):
    """Two captured graphs replayed at once on two streams, after lengths,
    pages and values changed in place."""
    c = Paged([5000, 300], 64, 2, 128, BF16, seed=12)
    d = Paged([2500, 4000], 64, 2, 128, BF16, seed=13)
    q1, q2 = queries(2, 8, 128, BF16, 1), queries(60, 8, 128, BF16, 2)
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, q in ((c, q1), (d, q2)):
        x.run(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(x.run(q))
        graphs.append(g)
    for step in range(3):
        c.lens.copy_(torch.tensor([4999 - 700 * step, 30 + step], dtype=torch.int32))
        d.lens.copy_(torch.tensor([60 + 900 * step, 3999 - step], dtype=torch.int32))
        q1.add_(0.25)
        q2.mul_(0.9)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        finish()
        assert torch.equal(outs[0], c.run(q1)) and torch.equal(outs[1], d.run(q2))


# ---------------------------------------------------------------- as they are used together
@pytest.mark.parametrize("kv", ["same", "e4m3"])
def test_prompt_then_chunks_then_tokens(cuda, kv):
    """A prompt through attention_varlen and into the cache, then chunks and
    single tokens over it: each step agrees with attention over all tokens so
    far (of what the cache holds)."""
    d, hq, hkv, page, dtype = 64, 8, 2, 16, F16
    steps = [[70, 33], [19, 40], [1, 1], [1, 1], [5, 0]]
    total = [sum(s[b] for s in steps) for b in range(2)]
    pages = 40
    table = torch.randperm(pages, generator=gen(1), device="cuda").int().view(2, 20)
    held = E4M3 if kv == "e4m3" else dtype
    kc, vc = (torch.zeros(pages, hkv, page, d, device="cuda").to(held) for _ in range(2))
    ks, vs = (torch.zeros(pages, hkv, page, dtype=torch.uint8, device="cuda").view(E8M0) if kv == "e4m3" else None
              for _ in range(2))
    x = [qkv(t, hq, hkv, d, dtype, 20 + b) for b, t in enumerate(total)]
    done = [0, 0]
    for n in steps:
        q, k, v = (torch.cat([x[b][i][done[b] : done[b] + n[b]] for b in range(2)]) for i in range(3))
        pos = [torch.arange(done[b], done[b] + n[b], device="cuda") for b in range(2)]
        slots = torch.cat([table[b].long()[p // page] * page + p % page for b, p in enumerate(pos)])
        cx.kv_cache_write(k, v, kc, vc, slots, ks, vs)
        first = done == [0, 0]
        done = [done[b] + n[b] for b in range(2)]
        cu, lens = cu_of(n), torch.tensor(done, dtype=torch.int32, device="cuda")
        out = cx.attention_paged(q, kc, vc, table, lens, cu_seqlens_q=cu, key_scale=ks, value_scale=vs)
        if first and kv == "same":
            prompt = cx.attention_varlen(q, k, v, cu)
        for b in range(2):
            p = torch.arange(done[b], device="cuda")
            kk, vv = cx.kv_cache_read(kc, vc, table[b].long()[p // page] * page + p % page, ks, vs, dtype=dtype)
            a = sum(n[:b])
            want, tol = attend(q[a : a + n[b]], kk, vv, 1 / math.sqrt(d), True, U[BF16], U[dtype])
            check(out[a : a + n[b]], want, tol, f"step {n}, sequence {b}")
            if first and kv == "same":
                check(prompt[a : a + n[b]], want, tol, f"prompt, sequence {b}")
    finish()


def test_random_cases(cuda):
    """Many small problems over the whole range of shapes, one seed."""
    rng = random.Random(5)
    for trial in range(60):
        dtype, d = rng.choice((F16, BF16)), rng.choice((64, 128))
        hkv = rng.choice((1, 2, 3))
        hq = hkv * rng.choice((1, 2, 3, 4, 5, 8, 16, 17, 40, 100))
        b = rng.randint(1, 5)
        n = [rng.choice((0, 1, 1, 2, 7, rng.randint(1, 90))) for _ in range(b)]
        lens = [max(0, x + rng.choice((0, 0, -1, 5, rng.randint(0, 600)))) for x in n]
        causal, page = rng.random() < 0.7, rng.choice((8, 16, 32, 64, 128, 256, 512))
        c = Paged(lens, page, hkv, d, dtype, rng.choice(("same", "e4m3")), seed=trial, nhd=rng.random() < 0.3)
        q, cu = queries(sum(n), hq, d, dtype, trial), cu_of(n)
        out = c.run(q, cu_seqlens_q=cu, causal=causal, max_seqlen_q=rng.choice((None, max(n))))
        finish()
        c.check(out, q, cu, causal, 1 / math.sqrt(d), f"trial {trial}")
        if c.ks is None and sum(n):
            k, v = torch.cat(c.keys), torch.cat(c.values)
            out = cx.attention_varlen(q, k, v, cu, cu_of(lens), causal=causal)
            finish()
            c.check(out, q, cu, causal, 1 / math.sqrt(d), f"trial {trial}, packed")


@pytest.mark.parametrize("kv", ["same", "e4m3"])
@pytest.mark.parametrize("hq,page,longest", [(300, 1024, 3), (4, 64, 1), (4, 64, 60)])
def test_sequences_that_share_their_pages(cuda, hq, page, longest, kv):
    """One row of the page table for every sequence (a row stride of 0), 150
    query heads to a kv head, pages longer than a tile."""
    c = Paged([1500], page, 2, 64, BF16, kv, seed=hq)
    lens = [1500, 0, 1, 1023, 1024, 1025, 64]
    n = [min(longest, 1 + 7 * i) for i in range(len(lens))]
    c.table = c.table[:1].expand(len(lens), -1)
    c.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.keys, c.values = [c.keys[0][:x] for x in lens], [c.values[0][:x] for x in lens]
    q, cu = queries(sum(n), hq, 64, BF16), cu_of(n)
    out = c.run(q, cu_seqlens_q=cu)
    finish()
    c.check(out, q, cu, True, 1 / 8)


@pytest.mark.parametrize("path", ["tc", "skinny", "simt"])
def test_many_sequences(cuda, path):
    """More sequences than a block looks through at once, most of them empty."""
    rng = random.Random(9)
    n = [rng.choice((0, 0, 0, 1, 2)) for _ in range(1500)]
    lens = [0 if rng.random() < 0.3 else rng.randint(0, 40) for _ in n]
    c = Paged(lens, 16, 1, 64, F16, "same", seed=3)
    q, cu = queries(sum(n), 2, 64, F16), cu_of(n)
    with forced(path):
        out = c.run(q, cu_seqlens_q=cu)
        finish()
        c.check(out, q, cu, True, 1 / 8)
        out = cx.attention_varlen(q, torch.cat(c.keys), torch.cat(c.values), cu, cu_of(lens))
        finish()
        c.check(out, q, cu, True, 1 / 8, "packed")


@pytest.mark.parametrize("kv", ["same", "e4m3"])
@pytest.mark.parametrize("n", [1, 40])
def test_context_of_nan(cuda, n, kv):
    """Every value NaN: a row that sees one is NaN, a row that sees nothing zeros."""
    lens = [n + 3000, n, 0]
    c = Paged(lens, 32, 2, 128, BF16, kv, seed=n)
    if kv == "same":
        c.vc.fill_(math.nan)
    else:
        c.vs.view(torch.uint8).fill_(255)
    q = queries(3 * n, 8, 128, BF16)
    out = c.run(q)
    finish()
    assert out[: 2 * n].isnan().all() and not out[2 * n :].any()
