"""Argument checks of attention_varlen, attention_paged, kv_cache_write and
kv_cache_read, and of their C ABI: all raised before any device work."""
import ctypes

import pytest
import torch

import cabi
import cmp_ext_b200 as cx
import cmpext3

I32 = torch.int32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def raises(msg, fn, *a, **kw):
    with pytest.raises(RuntimeError, match=msg):
        fn(*a, **kw)


def cu(*x):
    return torch.tensor(x, dtype=I32)


def test_exported_names():
    for name in ("attention_varlen", "attention_paged", "kv_cache_write", "kv_cache_read"):
        assert getattr(cmpext3, name) is getattr(cx, name)
        assert name in cmpext3.__all__ and name in cx.__all__


def test_varlen_checks():
    q, k = torch.zeros(6, 4, 8), torch.zeros(6, 2, 8)
    f = cx.attention_varlen
    raises(r"Query must be 3D \(Tokens, Heads, Dim\)", f, torch.zeros(6, 8), k, k, cu(0, 6))
    raises("Key must be 3D", f, q, torch.zeros(6, 8), k, cu(0, 6))
    raises("Value must be 3D", f, q, k, torch.zeros(6, 8), cu(0, 6))
    raises("Key shape mismatch", f, q, torch.zeros(6, 2, 9), torch.zeros(6, 2, 9), cu(0, 6))
    raises("Value shape mismatch", f, q, k, torch.zeros(6, 1, 8), cu(0, 6))
    raises("multiple of key heads", f, q, torch.zeros(6, 3, 8), torch.zeros(6, 3, 8), cu(0, 6))
    raises("multiple of key heads", f, q, torch.zeros(6, 0, 8), torch.zeros(6, 0, 8), cu(0, 6))
    raises("Dtype mismatch", f, q, k.half(), k, cu(0, 6))
    raises("Unsupported dtype for attention", f, q.double(), k.double(), k.double(), cu(0, 6))
    raises("cu_seqlens_q must be 1D", f, q, k, k, cu())
    raises("cu_seqlens_q must be int32", f, q, k, k, cu(0, 6).long())
    raises("cu_seqlens_k must have 2 elements, got 3", f, q, k, k, cu(0, 6), cu(0, 3, 6))
    raises("as many tokens as query", f, q, torch.zeros(7, 2, 8), torch.zeros(7, 2, 8), cu(0, 6))
    raises("expects CUDA tensors", f, q, k, k, cu(0, 6))
    raises("expects CUDA tensors", f, q, k, k, cu(0, 6), cu(0, 6), False, 0.5)


def paged(page=4, pages=3, heads=2, d=8, dtype=torch.float32):
    return torch.zeros(pages, heads, page, d).to(dtype), torch.zeros(pages, heads, page, d).to(dtype)


def test_paged_checks():
    f = cx.attention_paged
    q = torch.zeros(2, 4, 8)
    kc, vc = paged()
    table, lens = torch.zeros(2, 3, dtype=I32), cu(1, 2)
    raises(r"Query must be 3D", f, torch.zeros(2, 8), kc, vc, table, lens)
    raises("key_cache must be 4D", f, q, kc[0], vc, table, lens)
    raises("value_cache must have key_cache's shape", f, q, kc, vc[:2], table, lens)
    raises("key_cache head dim mismatch", f, torch.zeros(2, 4, 9), kc, vc, table, lens)
    raises("multiple of key_cache heads", f, torch.zeros(2, 3, 8), kc, vc, table, lens)
    raises("Dtype mismatch", f, q.half(), kc, vc, table, lens)
    raises("Dtype mismatch", f, q, kc, vc.half(), table, lens)
    raises("Unsupported dtype for attention", f, q.double(), kc.double(), vc.double(), table, lens)
    raises("contiguous along their last dimension", f, q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, lens)
    raises("page_table must be 2D", f, q, kc, vc, table[0], lens)
    raises("page_table must be int32", f, q, kc, vc, table.long(), lens)
    raises("seqlens_k must have 2 elements", f, q, kc, vc, table, cu(1))
    raises("cu_seqlens_q must have 3 elements", f, q, kc, vc, table, lens, cu(0, 2))
    raises("same number of query tokens", f, torch.zeros(3, 4, 8), kc, vc, table, lens)
    raises("belong to a float8_e4m3fn cache", f, q, kc, vc, table, lens, key_scale=torch.zeros(3, 2, 4).to(E8M0))
    raises("max_seqlen_q must not be negative", f, q, kc, vc, table, lens, max_seqlen_q=-1)
    raises("expects CUDA tensors", f, q, kc, vc, table, lens)
    k8, v8 = paged(dtype=E4M3)
    s = torch.zeros(3, 2, 4, dtype=torch.uint8).view(E8M0)
    raises("needs key_scale and value_scale", f, q, k8, v8, table, lens)
    raises("needs key_scale and value_scale", f, q, k8, v8, table, lens, key_scale=s)
    raises("must be float8_e8m0fnu", f, q, k8, v8, table, lens, key_scale=s.view(torch.uint8), value_scale=s)
    raises(r"must be \(Pages, Heads, Page size\)", f, q, k8, v8, table, lens, key_scale=s[:2], value_scale=s)
    raises("expects CUDA tensors", f, q, k8, v8, table, lens, key_scale=s, value_scale=s)


def test_cache_checks():
    k = torch.zeros(5, 2, 8)
    kc, vc = paged()
    slots = torch.zeros(5, dtype=torch.int64)
    w, r = cx.kv_cache_write, cx.kv_cache_read
    raises(r"Key must be 3D", w, k[0], k[0], kc, vc, slots)
    raises("Value shape mismatch", w, k, k[:4], kc, vc, slots)
    raises("Dtype mismatch", w, k, k.half(), kc, vc, slots)
    raises("Dtype mismatch", w, k.half(), k.half(), kc, vc, slots)
    raises("Unsupported dtype for kv_cache_write", w, k.double(), k.double(), kc, vc, slots)
    raises("key_cache heads mismatch", w, k[:, :1], k[:, :1], kc, vc, slots)
    raises("key_cache head dim mismatch", w, k[..., :7], k[..., :7], kc, vc, slots)
    raises("slots must be int64", w, k, k, kc, vc, slots.int())
    raises("one element for each token", w, k, k, kc, vc, slots[:4])
    raises("value_cache must not be key_cache", w, k, k, kc, kc, slots)
    raises("key_cache must not overlap itself", w, k, k, kc[:1].expand(3, 2, 4, 8), vc, slots)
    raises("expects CUDA tensors", w, k, k, kc, vc, slots)
    k8, v8 = paged(dtype=E4M3)
    s = torch.zeros(3, 2, 4, dtype=torch.uint8).view(E8M0)
    raises("value_scale must not be key_scale", w, k, k, k8, v8, slots, s, s)
    raises("needs key_scale and value_scale", w, k, k, k8, v8, slots)
    raises("slots must be 1D", r, kc, vc, slots.view(1, 5))
    raises("Dtype mismatch", r, kc, vc, slots, dtype=torch.float16)
    raises("Unsupported dtype for kv_cache_read", r, k8, v8, slots, s, s, dtype=torch.int32)
    raises("page size must be positive", r, kc[:, :, :0], vc[:, :, :0], slots)
    raises("expects CUDA tensors", r, kc, vc, slots)


def test_cache_overlaps_are_refused():
    w = cx.kv_cache_write
    k = torch.zeros(5, 2, 8)
    slots = torch.zeros(5, dtype=torch.int64)
    buf = torch.zeros(8, 2, 4, 8)
    raises("value_cache must not be key_cache or overlap it", w, k, k, buf[:6], buf[2:], slots)
    raises("value_cache must not be key_cache or overlap it", w, k, k, buf[:4], buf.view(-1)[8:8 + 256].view(4, 2, 4, 8), slots)
    raises("key_cache must not overlap an input", w, buf.view(-1)[:80].view(5, 2, 8), k, buf, torch.zeros_like(buf), slots)
    # both in one buffer, page by page or side by side: shared by nobody, so the next check is reached
    pair = torch.zeros(3, 2, 2, 4, 8)
    raises("expects CUDA tensors", w, k, k, pair[:, 0], pair[:, 1], slots)
    wide = torch.zeros(3, 2, 4, 16)
    raises("expects CUDA tensors", w, k, k, wide[..., :8], wide[..., 8:], slots)
    raises("value_cache must not be key_cache or overlap it", w, k, k, wide[..., :8], wide[..., 7:15], slots)
    raises("expects CUDA tensors", w, k, k, buf[:4], buf[4:], slots)


# ---------------------------------------------------------------- C ABI
def seq_args(**kw):
    a = cabi.AttentionSeqArgs()
    a.dtype = a.kv_dtype = cabi.F16
    a.Q, a.K, a.V, a.O = 0x100000, 0x200000, 0x300000, 0x400000  # fake, aligned; never dereferenced
    a.batch, a.tokens_q, a.heads_q, a.heads_kv, a.head_dim = 2, 8, 4, 2, 128
    a.q_stride_token = a.o_stride_token = 512
    a.q_stride_head = a.o_stride_head = 128
    a.k_stride_row = a.v_stride_row = 256
    a.k_stride_head = a.v_stride_head = 128
    a.tokens_kv = 8
    a.cu_seqlens_q = 0x500000
    a.scale, a.causal = 0.1, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def paged_args(**kw):
    base = dict(page_table=0x600000, seqlens_k=0x700000, page_table_stride=4, max_pages=4, pages=16, page_size=16,
                tokens_kv=0, k_stride_row=128, v_stride_row=128, k_stride_head=2048, v_stride_head=2048,
                k_stride_page=4096, v_stride_page=4096)
    base.update(kw)
    return seq_args(**base)


def run(a):
    return cabi.lib().cmpx_attention_seq(ctypes.byref(a), None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=9), dict(kv_dtype=cabi.BF16), dict(kv_dtype=cabi.E4M3),
                                dict(batch=-1), dict(tokens_q=-1), dict(heads_kv=3), dict(heads_kv=0), dict(Q=None),
                                dict(O=None), dict(K=None), dict(V=None), dict(path=9), dict(k_stride_row=-1),
                                dict(cu_seqlens_q=None, tokens_q=7), dict(cu_seqlens_q=None, cu_seqlens_k=0x500000),
                                dict(max_seqlen_q=-1)])
def test_seq_invalid_args(kw):
    assert run(seq_args(**kw)) == cabi.ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(seqlens_k=None), dict(page_size=0), dict(pages=-1), dict(max_pages=-1),
                                dict(kv_dtype=cabi.E4M3), dict(k_stride_page=-1), dict(page_table_stride=-1),
                                dict(kv_dtype=cabi.E4M3, k_scale=0x800000)])
def test_paged_invalid_args(kw):
    assert run(paged_args(**kw)) == cabi.ERR_INVALID_ARG


def test_seq_empty_and_too_large():
    assert cabi.lib().cmpx_attention_seq(None, None) == cabi.ERR_INVALID_ARG
    for kw in (dict(tokens_q=0), dict(heads_q=0), dict(head_dim=0)):
        assert run(seq_args(Q=None, O=None, K=None, V=None, **kw)) == cabi.OK
    assert run(seq_args(head_dim=513)) == cabi.ERR_UNSUPPORTED
    assert run(seq_args(tokens_q=2**31)) == cabi.ERR_UNSUPPORTED
    assert run(paged_args(max_pages=2**31)) == cabi.ERR_UNSUPPORTED


def select(a):
    return cabi.lib().cmpx_attention_seq_select_path(ctypes.byref(a))


def test_path_selection_is_host_logic():
    assert select(seq_args()) == cabi.PATH_SKINNY                       # 4 tokens a sequence x 2 heads
    assert select(seq_args(tokens_q=64, tokens_kv=64)) == cabi.PATH_TC   # 32 tokens
    assert select(seq_args(tokens_q=64, tokens_kv=64, max_seqlen_q=8)) == cabi.PATH_SKINNY
    assert select(seq_args(max_seqlen_q=9)) == cabi.PATH_TC
    assert select(seq_args(dtype=cabi.F32, kv_dtype=cabi.F32)) == cabi.PATH_SIMT
    assert select(seq_args(head_dim=96)) == cabi.PATH_SIMT
    assert select(seq_args(head_dim=1024)) == -1
    assert select(seq_args(K=0x200008)) == cabi.PATH_SIMT               # not on 16 bytes
    assert select(seq_args(k_stride_row=260)) == cabi.PATH_SIMT          # rows not on 16 bytes
    assert select(seq_args(tokens_kv=0)) == cabi.PATH_SIMT               # no key at all
    assert select(seq_args(scale=0.0, tokens_q=64)) == cabi.PATH_SKINNY  # the tcgen05 kernel masks with -inf
    assert select(seq_args(path=cabi.PATH_SIMT)) == cabi.PATH_SIMT
    assert select(seq_args(path=cabi.PATH_TC, head_dim=96)) == -1
    wide = dict(heads_q=400, tokens_q=2, k_stride_row=256)
    assert select(seq_args(**wide)) == cabi.PATH_SKINNY                  # 200 heads a kv head fill no 128-row tile
    for page, want in ((1, cabi.PATH_SIMT), (4, cabi.PATH_SIMT), (8, cabi.PATH_SKINNY), (24, cabi.PATH_SIMT),
                       (64, cabi.PATH_SKINNY)):
        assert select(paged_args(page_size=page)) == want, page
    e4m3 = dict(kv_dtype=cabi.E4M3, k_scale=0x800000, v_scale=0x900000, ks_stride_row=1, vs_stride_row=1,
                ks_stride_head=16, vs_stride_head=16, ks_stride_page=32, vs_stride_page=32)
    assert select(paged_args(**e4m3)) == cabi.PATH_SKINNY
    assert select(paged_args(**{**e4m3, "ks_stride_row": 2})) == cabi.PATH_SIMT
    assert select(paged_args(**{**e4m3, "page_size": 8})) == cabi.PATH_SIMT
    assert select(paged_args(**{**e4m3, "k_stride_row": 136})) == cabi.PATH_SIMT


def cache_args(**kw):
    a = cabi.KVCacheArgs()
    a.dtype = a.cache_dtype = cabi.F16
    a.key, a.value, a.key_cache, a.value_cache, a.slots = (0x100000 * i for i in range(1, 6))
    a.tokens, a.heads, a.head_dim, a.pages, a.page_size = 4, 2, 64, 8, 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_cache_invalid_args():
    for name in ("cmpx_kv_cache_write", "cmpx_kv_cache_read"):
        f = getattr(cabi.lib(), name)
        call = lambda **kw: f(ctypes.byref(cache_args(**kw)), None)  # noqa: E731
        assert f(None, None) == cabi.ERR_INVALID_ARG
        for kw in (dict(dtype=3), dict(cache_dtype=cabi.BF16), dict(tokens=-1), dict(key=None), dict(slots=None),
                   dict(key_cache=None), dict(cache_dtype=cabi.E4M3), dict(kc_stride_row=-1)):
            assert call(**kw) == cabi.ERR_INVALID_ARG, (name, kw)
        assert call(tokens=0, key=None, slots=None) == cabi.OK
        assert call(head_dim=513) == cabi.ERR_UNSUPPORTED
    assert cabi.lib().cmpx_kv_cache_write(ctypes.byref(cache_args(pages=0)), None) == cabi.OK
