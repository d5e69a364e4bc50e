"""attention_paged over e4m3 caches whose scales, pages and values are unusual,
on every kernel, against the definition in 64 bits.

Bound, besides seq_reference's: an output element is a sum of weight * code
products, and a weight held in fp16 is off by at most half a step of its own
(2^-11 relative) or, below 2^-14, by 2^-25.  The reference point of a row's
weights lies at or below its largest weight (the tcgen05 kernel's) or its
largest product of weight and scale 2^e (flash decoding's), so in units of the
result the second part is at most

    2^-25 * (max_j w_j * sum_j |v_j|  +  max_j w_j 2^e_j * sum_j |code_j|)

over the visible keys.

What lies below fp16's normal range may be taken as it is or rounded to fp16,
so elements of keys and values are off by 2^-25 at most for fp16 queries: a
score by scale * sum_d |q_d| 2^-25 (a weight by twice that, as in
seq_reference), the result by 2^-25, another 2^-25 its own rounding there."""
import contextlib
import math

import pytest
import torch

import cabi
import cmp_ext_b200 as cx
from seq_reference import U, attend, check, e8m0, quantise

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
KERNELS = ["simt", "tc", "skinny"]


@contextlib.contextmanager
def forced(path):
    cx._set_path(path)
    try:
        yield
    finally:
        cx._set_path("auto")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Cache:
    """One sequence in an e4m3 cache, pages in a random order; codes and scale
    bytes of keys and values [length, hkv, d] / [length, hkv] are the caller's."""

    def __init__(self, k, v, page=16, seed=0):
        self.k, self.v, self.page = k, v, page  # (codes in 64 bits, bytes)
        length, hkv, d = k[0].shape
        need = -(-length // page)
        order = torch.randperm(need + 2, generator=gen(seed), device="cuda")[:need]
        self.table = order.int().view(1, need)
        self.lens = torch.tensor([length], dtype=torch.int32, device="cuda")
        j = torch.arange(length, device="cuda")
        held = []
        for codes, byte in (k, v):
            c = torch.full((need + 2, hkv, page, d), math.nan, device="cuda")
            s = torch.full((need + 2, hkv, page), 255, dtype=torch.uint8, device="cuda")
            c[order[j // page], :, j % page] = codes.float()
            s[order[j // page], :, j % page] = byte
            held += [c.to(E4M3), s.view(E8M0)]
        self.kc, self.ks, self.vc, self.vs = held

    def lose(self, pages):
        """These pages of the sequence are none: their keys and values are zeros."""
        for p in pages:
            self.table[0, p] = -1 if p % 2 else 10**6
            for codes, byte in (self.k, self.v):
                codes[p * self.page : (p + 1) * self.page] = 0
                byte[p * self.page : (p + 1) * self.page] = 127

    def run(self, q, **kw):
        return cx.attention_paged(q, self.kc, self.vc, self.table, self.lens, key_scale=self.ks, value_scale=self.vs, **kw)

    def check(self, got, q, what, u_w, scale=None):
        n, hq, d = q.shape
        length, hkv = self.k[1].shape
        scale = 1 / math.sqrt(d) if scale is None else scale
        kk, vv = (read_as(c, b, q.dtype) for c, b in (self.k, self.v))
        want, tol = attend(q, kk, vv, scale, True, u_w, U[q.dtype])
        step = 2 * 2.0**-25 if q.dtype == F16 else 2.0**-134  # half of the output's smallest; the values'
        for i in range(n):
            lim = max(0, min(length, length - n + i + 1))
            if lim == 0:
                continue
            s = torch.einsum("hd,jhd->hj", q[i].double(), kk[:lim].repeat_interleave(hq // hkv, 1)) * scale
            w = torch.softmax(s, -1)
            e = torch.exp2(self.v[1][:lim].double() - 127).repeat_interleave(hq // hkv, 1).t()
            e = torch.where(self.v[1][:lim].repeat_interleave(hq // hkv, 1).t() == 255, 0.0, e)
            codes = self.v[0][:lim].double().nan_to_num().abs().sum(0).repeat_interleave(hq // hkv, 0)
            vals = vv[:lim].nan_to_num().abs().sum(0).repeat_interleave(hq // hkv, 0)
            if q.dtype == F16:
                spread = torch.einsum("hj,jhd->hd", w, vv[:lim].repeat_interleave(hq // hkv, 1).abs().nan_to_num())
                tol[i] += 2 * abs(scale) * 2.0**-25 * q[i].double().abs().sum(-1, keepdim=True) * spread
            tol[i] += step + 2.0**-25 * (w.amax(-1, keepdim=True) * vals + (w * e).amax(-1, keepdim=True) * codes)
        check(got, want, tol, what)


def read_as(codes, byte, dtype):
    """What the cache holds in the queries' type: rounded to it, held to its finite range."""
    x = codes.double() * e8m0(byte).unsqueeze(-1)
    top = torch.finfo(dtype).max
    return x.clamp(-top, top).to(dtype).double()


def normal(length, hkv, d, seed):
    """Codes and bytes of unit-normal vectors."""
    return quantise(torch.randn(length, hkv, d, generator=gen(seed), device="cuda"))


def scaled(length, hkv, d, bytes_, seed):
    """Codes of full size with these scale bytes."""
    codes, _ = quantise(torch.randn(length, hkv, d, generator=gen(seed), device="cuda"))
    return codes, bytes_.to(torch.uint8).cuda().view(length, 1).expand(length, hkv).contiguous()


def queries(n, hq, d, dtype, seed=1):
    return torch.randn(n, hq, d, generator=gen(seed), device="cuda").to(dtype)


def finish():
    torch.cuda.synchronize()
    assert cabi.device_error() == 0


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 24])
@pytest.mark.parametrize("lost", [[0], [3], [0, 1, 2, 3, 4, 5, 6], [12], range(0, 13, 2), range(13)])
def test_pages_that_are_none(cuda, lost, n, dtype, path):
    """Table entries that name no page read as zeros, wherever they lie."""
    c = Cache(normal(200, 2, 64, 1), normal(200, 2, 64, 2))
    c.lose(lost)
    q = queries(n, 4, 64, dtype)
    with forced(path):
        out = c.run(q)
    finish()
    c.check(out, q, f"lost {list(lost)}", U[dtype])
    if len(lost) == 13:
        assert not out.any()


def ramp(low, high, length):
    return torch.linspace(low + 127, high + 127, length).round()


SCALES = {
    "rising": lambda x: ramp(-127, 100, x),
    "falling": lambda x: ramp(100, -127, x),
    "one first strip of 2^-127": lambda x: torch.where(torch.arange(x) < 16, 0, 120),
    "one last key of 2^100": lambda x: torch.where(torch.arange(x) == x - 1, 227, 120),
    "one first key of 2^100": lambda x: torch.where(torch.arange(x) == 0, 227, 120),
    "in turn": lambda x: torch.tensor([7, 127, 200])[torch.arange(x) % 3],
    "random": lambda x: torch.randint(0, 228, (x,), generator=torch.Generator().manual_seed(3)),
}


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("n", [1, 24])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scales", list(SCALES))
def test_value_scales_far_apart(cuda, scales, d, n, path):
    """Every scale a byte can name, in any order along a sequence."""
    length = 333
    c = Cache(normal(length, 2, d, 3), scaled(length, 2, d, SCALES[scales](length), 4))
    q = queries(n, 8, d, BF16)
    with forced(path):
        out = c.run(q)
    finish()
    c.check(out, q, scales, U[BF16])


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("n", [1, 24])
@pytest.mark.parametrize("at", [0, 40, 199])
def test_zero_vectors_beside_tiny_values(cuda, at, n, path):
    """A vector of zeros has the scale 1, which lies far above that of values near 1e-10."""
    length = 200
    codes, byte = quantise(torch.randn(length, 2, 64, generator=gen(5), device="cuda") * 1e-10)
    codes[at], byte[at] = 0, 127
    c = Cache(normal(length, 2, 64, 6), (codes, byte))
    q = queries(n, 4, 64, BF16)
    with forced(path):
        out = c.run(q)
    finish()
    c.check(out, q, f"zeros at {at}", U[BF16])


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("n", [1, 24])
@pytest.mark.parametrize("length", [40, 1000])
def test_weights_of_fp16_queries(cuda, length, n, path):
    """Ordinary scales cost fp16 queries no more than fp16's own half step."""
    x = torch.randn(length, 2, 128, generator=gen(7), device="cuda")
    x *= 2.0 ** torch.randint(-2, 3, (length, 2, 1), generator=gen(8), device="cuda")
    c = Cache(normal(length, 2, 128, 9), quantise(x))
    q = queries(n, 8, 128, F16)
    with forced(path):
        out = c.run(q)
    finish()
    c.check(out, q, "fp16", U[F16])


BEYOND = {  # exponents of scales along a sequence, in turn
    "above": [5, 9, 12, 40, 127],
    "below": [-15, -20, -26, -33, -60, -127],
    "both": [-7, 9, -20, 100, -127, 3],
    "one above": [-7] * 40 + [9],
    "one below": [-7] * 40 + [-16],
}


def in_turn(exponents, length):
    return torch.tensor(exponents)[torch.arange(length) % len(exponents)] + 127


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("n,length", [(1, 150), (24, 150), (3, 7)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scales", list(BEYOND))
def test_values_beyond_fp16(cuda, scales, d, n, length, path):
    """What a cache holds of larger and of smaller vectors than fp16 does is
    taken as fp16 has it, as kv_cache_read gives it: on every kernel."""
    c = Cache(normal(length, 2, d, 10), scaled(length, 2, d, in_turn(BEYOND[scales], length), 11))
    q = queries(n, 8, d, F16)
    with forced(path):
        out = c.run(q)
    finish()
    c.check(out, q, scales, U[F16])


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("n,length", [(1, 150), (24, 150), (3, 7)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scales", list(BEYOND))
def test_keys_beyond_fp16(cuda, scales, d, n, length, path):
    c = Cache(scaled(length, 2, d, in_turn(BEYOND[scales], length), 12), normal(length, 2, d, 13))
    scale = 0.2 if scales in ("below", "one below") else 1e-5
    q = queries(n, 8, d, F16)
    with forced(path):
        out = c.run(q, scale=scale)
    finish()
    c.check(out, q, scales, U[F16], scale)


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_the_largest_value(cuda, dtype, path):
    """e4m3 rounds the types' largest values up to a power of two beyond them;
    read back they are the largest ones again, and a row that sees one key
    gives its value."""
    if dtype == F32 and path != "simt":
        pytest.skip("not this kernel's")
    top = torch.finfo(dtype).max
    v = torch.full((1, 2, 64), top, dtype=dtype, device="cuda")
    v[:, :, ::2] *= -1
    kc, vc = (torch.zeros(2, 2, 16, 64, device="cuda").to(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(2, 2, 16, dtype=torch.uint8, device="cuda").view(E8M0) for _ in range(2))
    cx.kv_cache_write(torch.ones_like(v), v, kc, vc, torch.tensor([19], device="cuda"), ks, vs)
    table, lens = torch.tensor([[1]], dtype=torch.int32, device="cuda"), torch.tensor([4], dtype=torch.int32, device="cuda")
    # the first three tokens' values are zeros of the smallest scale; their keys give -inf of weight
    kc[1, :, :3] = torch.full((2, 3, 64), -448.0, device="cuda").to(E4M3)
    ks.view(torch.uint8)[1, :, :3] = 127
    q = torch.full((1, 4, 64), 8.0, dtype=dtype, device="cuda")
    with forced(path):
        out = cx.attention_paged(q, kc, vc, table, lens, key_scale=ks, value_scale=vs)
    finish()
    read = cx.kv_cache_read(kc, vc, torch.tensor([19], device="cuda"), ks, vs, dtype=dtype)[1]
    assert torch.equal(read, v)
    assert torch.equal(out, v.repeat_interleave(2, 1))


SPREAD = {  # scale bytes of a sequence's values: 14 and 28 binades at random, a weighty first token of small values, ...
    "spread": lambda x: torch.randint(112, 126, (x,), generator=torch.Generator().manual_seed(1)),
    "wide": lambda x: torch.randint(100, 128, (x,), generator=torch.Generator().manual_seed(2)),
    "sink": lambda x: torch.where(torch.arange(x) == 0, 105, 120),
    "steps": lambda x: 100 + torch.arange(x) // 16 % 20,
    "zeros": lambda x: torch.where(torch.arange(x) % 64 == 5, 127, 111),
}


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 5, 24])
@pytest.mark.parametrize("scales", list(SPREAD))
def test_value_scales_that_vary(cuda, scales, n, dtype, path):
    """The reference of the weights follows the strips up and down: no bits are lost."""
    length = 900
    v = scaled(length, 2, 128, SPREAD[scales](length), 15)
    if scales == "zeros":
        v[0][torch.arange(length) % 64 == 5] = 0
    k = normal(length, 2, 128, 14)
    c = Cache(k, v)
    q = queries(n, 4, 128, dtype)
    if scales == "sink":  # queries that look at the first key
        q += read_as(k[0][:1], k[1][:1], dtype)[0].repeat_interleave(2, 0).to(dtype)
    with forced(path):
        out = c.run(q)
        for _ in range(2):
            assert torch.equal(c.run(q), out)
    finish()
    c.check(out, q, scales, U[dtype])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_strips_out_of_the_band_stay_matrix_products(cuda, dtype):
    """Measured 1.5 times as long; key by key it was five times."""

    def best(high):
        g = gen(16)
        kc, vc = (torch.randint(0, 120, (600, 8, 64, 128), generator=g, dtype=torch.uint8, device="cuda").view(E4M3)
                  for _ in range(2))
        ks = torch.full((600, 8, 64), 120, dtype=torch.uint8, device="cuda").view(E8M0)
        vs = torch.randint(112, high, (600, 8, 64), generator=g, dtype=torch.uint8, device="cuda").view(E8M0)
        table = torch.randperm(600, generator=g, device="cuda").int().view(12, 50)
        lens = torch.full((12,), 3200, dtype=torch.int32, device="cuda")
        q = queries(12, 32, 128, dtype)
        times = []
        for _ in range(7):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(5):
                cx.attention_paged(q, kc, vc, table, lens, key_scale=ks, value_scale=vs)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) / 5)
        return min(times)

    even, varied = best(114), best(126)
    print(f"{dtype}: {even * 1e3:.1f} us, scales of 14 binades {varied * 1e3:.1f}")
    assert varied <= 2.5 * even


@pytest.mark.parametrize("path", KERNELS)
@pytest.mark.parametrize("n", [1, 9])
def test_queries_with_an_infinity(cuda, n, path):
    """Scores of -inf hide a key, whatever the row's other elements are (in
    fp16, which flash decoding multiplies, 1e5 would be an infinity too)."""
    length = 60
    codes, byte = normal(length, 2, 64, 17)
    codes[:, :, 0] = torch.where(torch.arange(length) % 3 == 0, -1.0, 1.0).to(codes).view(-1, 1)  # q[0] hides two of three
    codes[:, :, 1] = 1
    c = Cache((codes, byte), normal(length, 2, 64, 18))
    q = queries(n, 4, 64, BF16)
    q[:, :2, 0] = -math.inf
    q[:, :2, 1] = 1e5
    q[:, 2:, :2] = torch.tensor([1e5, -1e5])  # no infinity: as ever
    with forced(path):
        out = c.run(q)
    finish()
    assert out[:, :2].isnan().all()  # one of three scores is +inf
    assert out[:, 2:].isfinite().all()
    c.k[0][:, :, 0] = 1
    c = Cache(c.k, c.v)
    with forced(path):
        out = c.run(q)
    finish()
    assert not out[:, :2].any()  # all are -inf: zeros
