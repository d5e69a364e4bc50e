"""Cases of the serving attention operators: attention_varlen, attention_paged, kv_cache_write and kv_cache_read.

A case is a dict of plain values.  Sequence lengths of a ragged case come from the case's own numbers
(`random.Random(case["ragged"])`), so `work` and `prepare` agree on them; values come from the seed alone.

Layouts: queries, keys and values of new tokens are [tokens, heads, D] views of one fused projection's output,
caches are [pages, kv heads, page size, D].  An 8-bit cache holds e4m3 codes with one power-of-two scale (e8m0)
for each vector of D.
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


# ---------------------------------------------------------------- cases
def listed():
    return [
        # three short prompts of a small model, one of a single token: latency
        dict(name="prompt_fp16_short", op="varlen", dtype="fp16", d=64, hq=8, hkv=8, seqs=3, q_short=1, q_long=130, ragged=3, causal=True),
        # an ordinary prefill batch, equal lengths (the benchmark's 8 x 1024)
        dict(name="prompt_bf16_8x1024", op="varlen", dtype="bf16", d=128, hq=32, hkv=8, seqs=8, q_short=1024, q_long=1024, ragged=0, causal=True),
        # packed prompts of very different, odd lengths, seven query heads to a kv head
        dict(name="prompt_bf16_ragged", op="varlen", dtype="bf16", d=128, hq=28, hkv=4, seqs=12, q_short=33, q_long=1501, ragged=5, causal=True),
        # two long prompts
        dict(name="prompt_fp16_long", op="varlen", dtype="fp16", d=128, hq=16, hkv=4, seqs=2, q_short=8000, q_long=8192, ragged=7, causal=True),
        # one user's next token over a short cache: latency
        dict(name="decode_bf16_one", op="paged", dtype="bf16", kv="same", d=128, hq=32, hkv=8, seqs=1, q_short=1, q_long=1, k_short=777, k_long=777, ragged=0, page=16, causal=True),
        # a serving batch's next tokens over long ragged contexts in an 8-bit cache
        dict(name="decode_e4m3_batch", op="paged", dtype="bf16", kv="e4m3", d=128, hq=32, hkv=8, seqs=48, q_short=1, q_long=1, k_short=1000, k_long=24000, ragged=11, page=64, causal=True),
        # the next chunk of two long prompts over what the cache holds of them
        dict(name="chunk_bf16_2x1024", op="paged", dtype="bf16", kv="same", d=128, hq=32, hkv=8, seqs=2, q_short=1024, q_long=1024, k_short=16000, k_long=16384, ragged=13, page=128, causal=True),
        # continuous batching: single tokens and chunks of several users in one call, 8-bit cache
        dict(name="mixed_e4m3_16", op="paged", dtype="fp16", kv="e4m3", d=128, hq=32, hkv=4, seqs=16, q_short=1, q_long=200, k_short=201, k_long=6000, ragged=17, page=32, causal=True),
        # one decode step's keys and values of a batch of 64: latency
        dict(name="write_e4m3_step", op="write", dtype="bf16", kv="e4m3", d=128, hkv=8, hq=32, tokens=64, page=16, pages=512),
        # a prefill batch's keys and values
        dict(name="write_e4m3_prompt", op="write", dtype="bf16", kv="e4m3", d=128, hkv=8, hq=32, tokens=16384, page=64, pages=320),
        # a short context read back from a 16-bit cache
        dict(name="read_bf16_short", op="read", dtype="bf16", kv="same", d=128, hkv=8, hq=32, tokens=1001, page=16, pages=128),
        # the contexts of a batch read back from an 8-bit cache
        dict(name="read_e4m3_long", op="read", dtype="bf16", kv="e4m3", d=128, hkv=8, hq=32, tokens=65500, page=64, pages=1100),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("varlen", "varlen", "paged", "paged", "paged", "write", "read"))
    c = dict(op=op, dtype=rng.choice(("fp16", "bf16")), d=rng.choice((64, 128, 128)), hkv=rng.choice((1, 2, 4, 8)))
    c["hq"] = c["hkv"] * rng.choice((1, 2, 3, 4, 7, 8))
    if op in ("write", "read"):
        c.update(kv=rng.choice(("same", "e4m3")), page=rng.choice((16, 32, 64, 128)), tokens=_spread(rng, 1, 32768))
        c["pages"] = c["tokens"] // c["page"] + rng.randint(1, 64)
        return c
    c.update(seqs=_spread(rng, 1, 64), ragged=rng.randrange(1 << 20), causal=rng.random() < 0.8)
    most = 700_000_000 // (c["seqs"] * c["hq"])  # query-key pairs of the padded batch, for each head
    if op == "varlen":
        c["q_long"] = _spread(rng, 1, min(8192, math.isqrt(most)))
        c["q_short"] = _spread(rng, 1, c["q_long"])
        return c
    c.update(kv=rng.choice(("same", "e4m3")), page=rng.choice((16, 32, 64, 128)))
    c["q_long"] = 1 if rng.random() < 0.4 else _spread(rng, 1, 1024)
    c["q_short"] = _spread(rng, 1, c["q_long"])
    room = min(most // c["q_long"], 6_000_000 // c["seqs"] // c["hkv"], 65536)
    c["k_long"] = _spread(rng, c["q_long"], max(c["q_long"], room))
    c["k_short"] = _spread(rng, 1, c["k_long"])
    return c


def lengths(case):
    """New tokens and keys of each sequence, as two lists."""
    rng = random.Random(case["ragged"])
    n = [_spread(rng, case["q_short"], case["q_long"]) for _ in range(case["seqs"])]
    if case["op"] == "varlen":
        return n, list(n)
    return n, [max(q, _spread(rng, case["k_short"], case["k_long"])) for q in n]


def _pairs(case):
    """Query-key pairs of one query head, and keys that any query sees."""
    pairs = 0
    for n, k in zip(*lengths(case)):
        pairs += n * (k - n) + n * (n + 1) // 2 if case["causal"] else n * k
    return pairs


def work(case):
    d, hq, hkv = case["d"], case["hq"], case["hkv"]
    if case["op"] in ("write", "read"):
        vectors = 2 * case["tokens"] * hkv
        held = d + 1 if case["kv"] == "e4m3" else 2 * d
        return {"bytes": vectors * (2 * d + held) + 8 * case["tokens"], "flops": vectors * 2 * d}
    n, k = lengths(case)
    held = (d + 1 if case.get("kv") == "e4m3" else 2 * d) * 2 * hkv
    table = sum(-(-x // case["page"]) for x in k) * 4 if case["op"] == "paged" else 0
    return {"bytes": sum(n) * hq * d * 4 + sum(k) * held + table, "flops": 4 * d * hq * _pairs(case)}


# ---------------------------------------------------------------- inputs
def _quantise(x):
    """e4m3 codes and e8m0 bytes of the vectors along x's last axis (for caches that are there before the call)."""
    a = x.float().abs().amax(-1)
    m, k = torch.frexp(a)
    e = torch.where(a == 0, 0, torch.clamp(k - 9 + (m > 0.875), min=-127))
    return torch.ldexp(x.float(), -e.unsqueeze(-1)).to(E4M3), (e + 127).to(torch.uint8).view(E8M0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, d, hq, hkv = TYPES[case["dtype"]], case["d"], case["hq"], case["hkv"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": case}
    if case["op"] in ("varlen", "paged"):
        n, k = lengths(case)
        s["n"], s["k"] = n, k
        s["cu"] = torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        tokens = sum(n)
    else:
        tokens = case["tokens"]
    qkv = normal(tokens, hq + 2 * hkv, d).to(t)  # the projection's output; the operators take views of it
    s["q"], s["key"], s["value"] = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    if case["op"] == "varlen":
        return s
    page = case["page"]
    if case["op"] == "paged":
        need = [-(-x // page) for x in s["k"]]
        pages = sum(need) + 8
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
        rows = torch.repeat_interleave(torch.arange(len(need)), torch.tensor(need))
        cols = torch.cat([torch.arange(x) for x in need])
        table[rows.cuda(), cols.cuda()] = order[: sum(need)]
        s["table"] = table
        s["lens"] = torch.tensor(s["k"], dtype=torch.int32, device="cuda")
    else:
        pages = case["pages"]
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    shape = (pages, hkv, page, d)
    if case["op"] == "write":
        held = E4M3 if case["kv"] == "e4m3" else t
        s["kc"], s["vc"] = (torch.zeros(shape, device="cuda").to(held) for _ in range(2))
        s["ks"], s["vs"] = (torch.full(shape[:3], 127, dtype=torch.uint8, device="cuda").view(E8M0) if case["kv"] == "e4m3" else None for _ in range(2))
        return s
    s["ks"] = s["vs"] = None
    if case["kv"] == "e4m3":
        (s["kc"], s["ks"]), (s["vc"], s["vs"]) = (_quantise(normal(*shape).to(t)) for _ in range(2))
    else:
        s["kc"], s["vc"] = (normal(*shape).to(t) for _ in range(2))
    return s


# ---------------------------------------------------------------- plain forms
def _scales(b, shape):
    """Powers of two of e8m0 bytes, along a new last axis (255: NaN)."""
    b = b.view(torch.uint8).to(torch.int32)
    return torch.where(b == 255, math.nan, torch.ldexp(torch.ones(shape, device=b.device), b - 127)).unsqueeze(-1)


def _attend(case, q, k, v, n, lens, scale):
    """Padded batch: q [B, N, Hq, D], k and v [B, L, Hkv, D] in 32 bits, n and lens [B]: [B, N, Hq, D]."""
    b, longest, hq, d = q.shape
    hkv, keys = k.shape[2], k.shape[1]
    q = q.view(b, longest, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(scale).view(b, hkv, hq // hkv, longest, keys)
    i, j = torch.arange(longest, device=q.device), torch.arange(keys, device=q.device)
    last = lens.view(-1, 1).expand(-1, longest)
    if case["causal"]:
        last = (lens.view(-1, 1) - n.view(-1, 1) + i + 1).clamp(min=0)
    hidden = j >= last.unsqueeze(-1)
    s.masked_fill_(hidden.view(b, 1, 1, longest, keys), -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, 0, m)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hkv, -1, keys), v.permute(0, 2, 1, 3)).view(b, hkv, hq // hkv, longest, d)
    return (o / torch.where(total == 0, 1, total)).permute(0, 3, 1, 2, 4).reshape(b, longest, hq, d)


def _plain_attention(s):
    case, q = s["case"], s["q"]
    cu = s["cu"].long()
    n = cu[1:] - cu[:-1]
    i = torch.arange(max(s["n"]), device=q.device)
    there = i < n.view(-1, 1)
    at = torch.where(there, cu[:-1].view(-1, 1) + i, 0)
    padded = q[at].float()
    if case["op"] == "varlen":
        lens, k, v = n, s["key"][at].float(), s["value"][at].float()
    else:
        lens = s["lens"].long()
        j = torch.arange(max(s["k"]), device=q.device)
        page = s["table"].long()[:, j // case["page"]].clamp(min=0)
        spot = (j % case["page"]).expand_as(page)
        k, v = s["kc"].transpose(1, 2)[page, spot].float(), s["vc"].transpose(1, 2)[page, spot].float()
        if s["ks"] is not None:
            by = k.shape[:3]
            k *= _scales(s["ks"].view(torch.uint8).transpose(1, 2)[page, spot], by)
            v *= _scales(s["vs"].view(torch.uint8).transpose(1, 2)[page, spot], by)
    o = _attend(case, padded, k, v, n, lens, 1 / math.sqrt(case["d"]))
    return o[there].to(q.dtype)


def _plain_write(s):
    page = s["kc"].shape[2]
    at = (s["slots"] // page, slice(None), s["slots"] % page)
    if s["ks"] is None:
        s["kc"][at], s["vc"][at] = s["key"], s["value"]
        return s["kc"], s["vc"]
    x = torch.stack((s["key"], s["value"])).float()
    a = x.abs().amax(-1)
    m, k = torch.frexp(a)
    e = torch.where(a == 0, 0, torch.clamp(k - 9 + (m > 0.875), min=-127))
    code = torch.ldexp(x, -e.unsqueeze(-1)).to(E4M3).view(torch.uint8)
    byte = torch.where(a.isfinite(), e + 127, 255).to(torch.uint8)
    s["kc"].view(torch.uint8)[at], s["vc"].view(torch.uint8)[at] = code[0], code[1]
    s["ks"].view(torch.uint8)[at], s["vs"].view(torch.uint8)[at] = byte[0], byte[1]
    return s["kc"], s["vc"], s["ks"].view(torch.uint8), s["vs"].view(torch.uint8)


def _plain_read(s):
    page = s["kc"].shape[2]
    at = (s["slots"] // page, slice(None), s["slots"] % page)
    if s["ks"] is None:
        return s["kc"][at], s["vc"][at]
    code = torch.stack((s["kc"].view(torch.uint8)[at], s["vc"].view(torch.uint8)[at])).view(E4M3)
    byte = torch.stack((s["ks"].view(torch.uint8)[at], s["vs"].view(torch.uint8)[at]))
    x = (code.float() * _scales(byte, byte.shape)).to(s["key"].dtype)
    return x[0], x[1]


def run(s):
    case = s["case"]
    if own:
        import cmpext3

        if case["op"] == "varlen":
            return cmpext3.attention_varlen(s["q"], s["key"], s["value"], s["cu"], causal=case["causal"])
        if case["op"] == "paged":
            return cmpext3.attention_paged(s["q"], s["kc"], s["vc"], s["table"], s["lens"], cu_seqlens_q=s["cu"], causal=case["causal"],
                                           key_scale=s["ks"], value_scale=s["vs"], max_seqlen_q=max(s["n"]))
        if case["op"] == "write":
            cmpext3.kv_cache_write(s["key"], s["value"], s["kc"], s["vc"], s["slots"], key_scale=s["ks"], value_scale=s["vs"])
            return (s["kc"], s["vc"]) if s["ks"] is None else (s["kc"], s["vc"], s["ks"].view(torch.uint8), s["vs"].view(torch.uint8))
        return cmpext3.kv_cache_read(s["kc"], s["vc"], s["slots"], key_scale=s["ks"], value_scale=s["vs"], dtype=s["key"].dtype)
    if case["op"] in ("varlen", "paged"):
        return _plain_attention(s)
    return _plain_write(s) if case["op"] == "write" else _plain_read(s)


# ---------------------------------------------------------------- in 64 bits
def _read64(cache, scale, page, spot):
    """Vectors [len(page), Hkv, D] of a cache."""
    x = cache[page, :, spot].double()
    if scale is not None:
        b = scale.view(torch.uint8)[page, :, spot].double()
        x = x * torch.where(b == 255, math.nan, torch.exp2(b - 127)).unsqueeze(-1)
    return x


def _round_e4m3(y):
    """The nearest e4m3 values of y in 64 bits, ties to even: three bits after the leading one, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read":
        page, spot = s["slots"] // case["page"], s["slots"] % case["page"]
        return _read64(s["kc"], s["ks"], page, spot), _read64(s["vc"], s["vs"], page, spot)
    if case["op"] == "write":
        page, spot = s["slots"] // case["page"], s["slots"] % case["page"]
        held, bytes_ = [], []
        for x, cache in ((s["key"], s["kc"]), (s["value"], s["vc"])):
            c, x = cache.double(), x.double()
            if s["ks"] is not None:
                a = x.abs().amax(-1)
                e = torch.where(a == 0, 0, torch.ceil(torch.log2(a / 448)).clamp(min=-127))
                e = torch.where(a > 448 * torch.exp2(e), e + 1, e)  # a logarithm that was rounded down over a border
                e = torch.where((a > 0) & (a <= 448 * torch.exp2(e - 1)), e - 1, e)
                x = _round_e4m3(x * torch.exp2(-e).unsqueeze(-1))
                b = torch.full(c.shape[:3], 127, dtype=torch.int64, device=c.device)
                b[page, :, spot] = (e + 127).long()
                bytes_.append(b)
            c[page, :, spot] = x
            held.append(c)
        return tuple(held + bytes_)
    outs, scale, first = [], 1 / math.sqrt(case["d"]), 0
    group = case["hq"] // case["hkv"]
    for b, (n, length) in enumerate(zip(s["n"], s["k"])):
        q = s["q"][first : first + n].double()
        if case["op"] == "varlen":
            k, v = s["key"][first : first + n].double(), s["value"][first : first + n].double()
        else:
            j = torch.arange(length, device="cuda")
            page, spot = s["table"][b].long()[j // case["page"]], j % case["page"]
            k, v = _read64(s["kc"], s["ks"], page, spot), _read64(s["vc"], s["vs"], page, spot)
        first += n
        sees = torch.ones(n, length, dtype=torch.bool, device="cuda")
        if case["causal"]:
            sees = sees.tril(length - n)
        o = torch.empty(n, case["hq"], case["d"], dtype=torch.float64, device="cuda")
        for h in range(case["hq"]):
            w = q[:, h] @ k[:, h // group].t() * scale
            o[:, h] = torch.softmax(w.masked_fill_(~sees, -math.inf), -1) @ v[:, h // group]
        outs.append(o)
    return torch.cat(outs)
