"""What kv_cache_write and the attention operators take for an overlap: shared
elements, not ranges that interleave.  A call that passes its checks on the CPU
ends at "expects CUDA tensors"."""
import itertools
import random

import pytest
import torch

import cmp_ext_b200 as cx

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
P, H, S, D = 3, 2, 4, 16


def write(kc, vc, ks=None, vs=None, key=None, value=None, slots=None):
    key = torch.zeros(5, kc.shape[1], kc.shape[3], dtype=torch.bfloat16) if key is None else key
    value = torch.zeros_like(key) if value is None else value
    slots = torch.zeros(5, dtype=torch.int64) if slots is None else slots
    with pytest.raises(RuntimeError) as e:
        cx.kv_cache_write(key, value, kc, vc, slots, ks, vs)
    return str(e.value).split("\n")[0]


def codes(x):
    return x.view(E4M3)


def scales(x):
    return x.view(E8M0)


def test_codes_and_scales_in_one_page():
    """[codes of a page | scales of a page], keys and values in pools of their own or page by page in one."""
    for pools in (1, 2):
        pool = torch.zeros(P, 2, H * S * (D + 1), dtype=torch.uint8)
        k, v = (pool[:, 0], pool[:, 1]) if pools == 1 else (pool[:, 0].contiguous(), pool[:, 1].contiguous())
        n = H * S * D
        parts = [(codes(x[:, :n].view(P, H, S, D)), scales(x[:, n:].view(P, H, S))) for x in (k, v)]
        assert "expects CUDA" in write(parts[0][0], parts[1][0], parts[0][1], parts[1][1])


def test_scale_beside_each_vector():
    pool = torch.zeros(P, H, S, 2, D + 1, dtype=torch.uint8)
    kc, vc = (codes(pool[..., i, :D]) for i in (0, 1))
    ks, vs = (scales(pool[..., i, D]) for i in (0, 1))
    assert "expects CUDA" in write(kc, vc, ks, vs)
    # a scale that lies on a code
    assert "value_scale must not be" in write(kc, vc, ks, scales(pool[..., 1, D - 1]))
    assert "key_scale must not be" in write(kc, vc, scales(pool[..., 1, 3]), vs)


def test_other_layouts_of_the_two_caches():
    """Keys heads first, values token first, in turn within one buffer."""
    pool = torch.zeros(P, 2, H * S * D)
    kc = pool[:, 0].view(P, H, S, D)
    vc = pool[:, 1].view(P, S, H, D).transpose(1, 2)
    key = torch.zeros(5, H, D)
    assert "expects CUDA" in write(kc, vc, key=key)
    vc = pool.view(P, -1)[:, 8 : 8 + H * S * D].view(P, S, H, D).transpose(1, 2)  # over the keys' last rows
    assert "value_cache must not be key_cache or overlap it" in write(kc, vc, key=key)


def test_inputs_between_the_pages():
    pool = torch.zeros(5, H * S * D + H * D)
    kc, key = pool[:, : H * S * D].view(5, H, S, D), pool[:, H * S * D :].view(5, H, D)
    assert "expects CUDA" in write(kc, torch.zeros_like(kc), key=key)
    assert "key_cache must not overlap an input" in write(kc, torch.zeros_like(kc), key=pool[:, : H * D].view(5, H, D))
    one = torch.zeros(1, H, D).expand(5, H, D)  # an input may repeat itself
    assert "expects CUDA" in write(kc, torch.zeros_like(kc), key=one)


def test_out_between_the_queries():
    pool = torch.zeros(6, 2, 4, 8)
    q, k = pool[:, 0], torch.zeros(6, 2, 8)
    cu = torch.tensor([0, 6], dtype=torch.int32)
    for out, what in ((pool[:, 1], "expects CUDA"), (pool[:, 0], "expects CUDA"), (pool.view(-1)[8:200].view(6, 4, 8), "expects CUDA")):
        with pytest.raises(RuntimeError, match=what):  # (the device is checked first)
            cx.attention_varlen(q, k, k, cu, out=out)


def offsets(t):
    """Byte addresses of a tensor's elements, from its start of storage."""
    es, out = t.element_size(), set()
    for at in itertools.product(*(range(n) for n in t.shape)):
        first = (t.storage_offset() + sum(i * s for i, s in zip(at, t.stride()))) * es
        out.update(range(first, first + es))
    return out


def test_random_views():
    """Views of one buffer, of the same or other layouts, against a look at every address."""
    rng = random.Random(7)
    seen = {True: 0, False: 0}
    for _ in range(400):
        buf = torch.zeros(4000, dtype=torch.uint8)

        def view(sizes, unit):
            order = list(range(len(sizes)))
            rng.shuffle(order)
            strides, reach = [0] * len(sizes), unit
            for i in order:
                strides[i] = reach + rng.choice((0, 0, 0, 1, 2, 5, 17))
                reach = strides[i] * sizes[i]
            room = sum((n - 1) * s for n, s in zip(sizes, strides)) + unit
            first = rng.randrange(0, max(1, min(4000 - room, 200)))
            return buf.as_strided(sizes + ((unit,) if unit > 1 else ()), tuple(strides) + ((1,) if unit > 1 else ()), first)

        sizes = (rng.randint(1, 3), rng.randint(1, 3), rng.randint(1, 4))
        d = rng.choice((2, 4))
        kc, vc = codes(view(sizes, d)), codes(view(sizes, d))
        ks, vs = (scales(torch.zeros(sizes, dtype=torch.uint8)) if rng.random() < 0.5 else scales(view(sizes, 1)) for _ in range(2))
        views = {"key_cache": kc, "value_cache": vc, "key_scale": ks, "value_scale": vs}
        base = buf.untyped_storage().data_ptr()
        inside = [n for n, t in views.items() if t.untyped_storage().data_ptr() == base]
        shared = any(offsets(views[a]) & offsets(views[b]) for a, b in itertools.combinations(inside, 2))
        seen[shared] += 1
        got = write(kc, vc, ks, vs, key=torch.zeros(5, sizes[1], d))
        assert ("or overlap it" in got) == shared, (got, {n: (t.shape, t.stride(), t.storage_offset()) for n, t in views.items()})
    assert min(seen.values()) > 40, seen
