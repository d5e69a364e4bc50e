// Attention over packed sequences and paged caches (cmpx_attention_seq):
// argument checks, path selection and the CUDA-core kernel.  No counterpart
// in the reference.
#include <climits>

#include "attention_math.cuh"
#include "attention_seq.h"

namespace cmpx {
namespace {

// Scalar loads of keys and values; `up` an 8-bit code's scale.
template <typename T, typename KV>
__device__ __forceinline__ float ldkv(const KV* p, float up) {
  if constexpr (sizeof(KV) == 1) return held<T>(*p, up);
  else return ldf(p);
}

// Sequence that holds token t (the last one that begins at or before it), or
// -1 for a token of none.
__device__ __forceinline__ int seq_find(const SeqProblem& p, int t) {
  if (p.cu_q == nullptr) return p.uniform_n > 0 ? t / p.uniform_n : -1;
  int lo = 0, hi = p.batch;  // first b with cu_q[b] > t lies in [lo, hi]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.cu_q + mid) <= t) lo = mid + 1; else hi = mid;
  }
  const int b = lo - 1;
  if (b < 0) return -1;
  const int2 q = seq_queries(p, b);
  return t >= q.x && t < q.x + q.y ? b : -1;
}

// One warp per (token, query head): lane d holds columns d, d + 32, ... of
// the query and the accumulator; online softmax in fp32 over the visible
// keys.  Every dtype, layout and head_dim up to kSimtMaxD; bound by the two
// dependent warp steps a key takes, not by memory.
template <typename T, typename KV, int NV>
__global__ void __launch_bounds__(128) attention_seq_simt_kernel(const SeqProblem p) {
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (long long)p.tokens_q * p.heads_q) return;
  const int t = int(row / p.heads_q), h = int(row - (long long)t * p.heads_q);
  T* orow = static_cast<T*>(p.O) + t * p.o_token + h * p.o_head;
  const int b = seq_find(p, t);
  if (b < 0) {
    if (p.zero_rest)
      for (int d = lane; d < p.d; d += 32) stf(orow + d, 0.0f);
    return;
  }
  const Seq s = seq_of(p, b);
  const int lim = seq_limit(p, s, t - s.q0);
  const int hk = h / p.group;
  const T* q = static_cast<const T*>(p.Q) + t * p.q_token + h * p.q_head;
  const KV* kb = static_cast<const KV*>(p.k.base) + hk * p.k.head;
  const KV* vb = static_cast<const KV*>(p.v.base) + hk * p.v.head;
  float qv[NV], acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int d = lane + 32 * i;
    qv[i] = d < p.d ? ldf(q + d) : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  int page = 0, off = 0, slot = 0;  // slot of the page that holds key j
  for (int j = 0; j < lim; ++j) {
    int64_t ko, vo;
    float ks = 1.0f, vs = 1.0f;
    bool there = true;
    if (p.table != nullptr) {
      if (slot == 0) page = __ldg(p.table + b * p.table_stride + off);
      there = page >= 0 && page < p.pages;
      ko = page * p.k.page + slot * p.k.row;
      vo = page * p.v.page + slot * p.v.row;
      if (sizeof(KV) == 1 && there) {
        ks = e8m0_to_float(p.k.scale[page * p.k.s_page + hk * p.k.s_head + slot * p.k.s_row]);
        vs = e8m0_to_float(p.v.scale[page * p.v.s_page + hk * p.v.s_head + slot * p.v.s_row]);
      }
      if (++slot == p.page_size) {
        slot = 0;
        ++off;
      }
    } else {
      ko = int64_t(s.k0 + j) * p.k.row;
      vo = int64_t(s.k0 + j) * p.v.row;
    }
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int d = lane + 32 * i;
      if (there && d < p.d) dot = fmaf(qv[i], ldkv<T>(kb + ko + d, ks), dot);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float x = dot * p.scale_log2;
    const float m_new = fmaxf(m, x);
    const float m_use = m_new == -INFINITY ? 0.0f : m_new;  // nothing finite so far: all weights 0
    const float alpha = exp2f(m - m_use);
    const float w = exp2f(x - m_use);
    l = l * alpha + w;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int d = lane + 32 * i;
      acc[i] *= alpha;
      if (there && d < p.d) acc[i] = fmaf(w, ldkv<T>(vb + vo + d, vs), acc[i]);
    }
    m = m_new;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int d = lane + 32 * i;
    if (d < p.d) stf(orow + d, l == 0.0f ? 0.0f : acc[i] * inv);
  }
}

template <typename T, typename KV>
cudaError_t launch_simt_typed(const SeqProblem& p, cudaStream_t s) {
  const unsigned blocks = unsigned(((long long)p.tokens_q * p.heads_q + 3) / 4);
  if (p.d <= 64) attention_seq_simt_kernel<T, KV, 2><<<blocks, 128, 0, s>>>(p);
  else if (p.d <= 128) attention_seq_simt_kernel<T, KV, 4><<<blocks, 128, 0, s>>>(p);
  else if (p.d <= 256) attention_seq_simt_kernel<T, KV, 8><<<blocks, 128, 0, s>>>(p);
  else attention_seq_simt_kernel<T, KV, 16><<<blocks, 128, 0, s>>>(p);
  return cudaGetLastError();
}

// Checks everything the host can see.  CMPX_OK with *empty set: nothing to do.
int validate_seq(const cmpx_attention_seq_args* a, bool* empty) {
  *empty = false;
  if (a == nullptr) return CMPX_ERR_INVALID_ARG;
  if (a->dtype != CMPX_F16 && a->dtype != CMPX_BF16 && a->dtype != CMPX_F32) return CMPX_ERR_INVALID_ARG;
  const bool paged = a->page_table != nullptr;
  if (a->kv_dtype != a->dtype && !(paged && a->kv_dtype == CMPX_E4M3)) return CMPX_ERR_INVALID_ARG;
  if (a->batch < 0 || a->tokens_q < 0 || a->heads_q < 0 || a->heads_kv < 0 || a->head_dim < 0 || a->tokens_kv < 0 ||
      a->max_seqlen_q < 0)
    return CMPX_ERR_INVALID_ARG;
  if (a->tokens_q == 0 || a->heads_q == 0 || a->head_dim == 0) {
    *empty = true;
    return CMPX_OK;
  }
  if (a->heads_kv == 0 || a->heads_q % a->heads_kv != 0) return CMPX_ERR_INVALID_ARG;
  if (a->Q == nullptr || a->O == nullptr) return CMPX_ERR_INVALID_ARG;
  if (a->cu_seqlens_q == nullptr && (a->batch == 0 ? a->tokens_q != 0 : a->tokens_q % a->batch != 0))
    return CMPX_ERR_INVALID_ARG;
  if (a->path != CMPX_PATH_AUTO && a->path != CMPX_PATH_TC && a->path != CMPX_PATH_SKINNY && a->path != CMPX_PATH_SIMT)
    return CMPX_ERR_INVALID_ARG;
  if (a->q_stride_token < 0 || a->q_stride_head < 0 || a->o_stride_token < 0 || a->o_stride_head < 0 ||
      a->k_stride_row < 0 || a->k_stride_head < 0 || a->v_stride_row < 0 || a->v_stride_head < 0)
    return CMPX_ERR_INVALID_ARG;
  int64_t keys;  // rows of K that sequences can name
  if (paged) {
    if (a->seqlens_k == nullptr || a->pages < 0 || a->page_size <= 0 || a->max_pages < 0 || a->page_table_stride < 0 ||
        a->k_stride_page < 0 || a->v_stride_page < 0)
      return CMPX_ERR_INVALID_ARG;
    if (a->kv_dtype == CMPX_E4M3 && a->pages > 0 &&
        (a->k_scale == nullptr || a->v_scale == nullptr || a->ks_stride_page < 0 || a->ks_stride_head < 0 ||
         a->ks_stride_row < 0 || a->vs_stride_page < 0 || a->vs_stride_head < 0 || a->vs_stride_row < 0))
      return CMPX_ERR_INVALID_ARG;
    if (a->max_pages > (INT_MAX - 1024) / a->page_size) return CMPX_ERR_UNSUPPORTED;
    keys = a->pages;
  } else {
    if (a->cu_seqlens_k != nullptr && a->cu_seqlens_q == nullptr) return CMPX_ERR_INVALID_ARG;
    keys = a->tokens_kv;
  }
  if (keys > 0 && (a->K == nullptr || a->V == nullptr)) return CMPX_ERR_INVALID_ARG;
  if (a->tokens_q > INT_MAX / 2 || a->tokens_kv > INT_MAX / 2 || a->batch >= INT_MAX / 2 || a->heads_q > 65535 ||
      a->pages > INT_MAX / 2 || a->page_size > INT_MAX / 2)
    return CMPX_ERR_UNSUPPORTED;
  return CMPX_OK;
}

SeqProblem resolve_seq(const cmpx_attention_seq_args* a) {
  SeqProblem p = {};
  p.Q = a->Q;
  p.O = a->O;
  p.q_token = a->q_stride_token;
  p.q_head = a->q_stride_head;
  p.o_token = a->o_stride_token;
  p.o_head = a->o_stride_head;
  p.k = SeqKV{a->K, a->k_stride_row, a->k_stride_head, a->k_stride_page, static_cast<const uint8_t*>(a->k_scale),
              a->ks_stride_row, a->ks_stride_head, a->ks_stride_page};
  p.v = SeqKV{a->V, a->v_stride_row, a->v_stride_head, a->v_stride_page, static_cast<const uint8_t*>(a->v_scale),
              a->vs_stride_row, a->vs_stride_head, a->vs_stride_page};
  p.cu_q = a->cu_seqlens_q;
  p.cu_k = a->cu_seqlens_k;
  p.table = a->page_table;
  p.lens_k = a->seqlens_k;
  p.table_stride = a->page_table_stride;
  p.batch = int(a->batch);
  p.uniform_n = a->cu_seqlens_q == nullptr && a->batch > 0 ? int(a->tokens_q / a->batch) : 0;
  p.tokens_q = int(a->tokens_q);
  p.tokens_kv = int(a->tokens_kv);
  p.heads_q = int(a->heads_q);
  p.heads_kv = int(a->heads_kv);
  p.group = int(a->heads_q / a->heads_kv);
  p.d = int(a->head_dim);
  if (a->page_table != nullptr) {
    p.page_size = int(a->page_size);
    p.pages = int(a->pages);
    p.max_keys = int(a->max_pages * a->page_size);
    while ((2 << p.page_lg) <= p.page_size) ++p.page_lg;
  }
  p.scale_log2 = a->scale * kLog2e;
  p.causal = a->causal != 0;
  p.zero_rest = a->zero_rest != 0;
  return p;
}

// Query rows a kv head has in a typical sequence: those of the longest one if
// the caller or the layout says so, else of the mean one.
int64_t typical_rows(const cmpx_attention_seq_args* a, const SeqProblem& p) {
  const int64_t tokens = a->cu_seqlens_q == nullptr ? p.uniform_n
                         : a->max_seqlen_q > 0      ? a->max_seqlen_q
                         : a->batch > 0             ? (a->tokens_q + a->batch - 1) / a->batch
                                                    : 0;
  return tokens > INT_MAX ? INT_MAX : tokens * p.group;
}

// The kernel that runs a checked, non-empty problem, or -1.  Few query rows a
// kv head run the flash-decoding kernel, whose units hold at most 16 of them;
// more the tcgen05 kernel.  16 sequences over 4000 keys, 32 / 8 heads of 128,
// flash decoding against tcgen05: 4 rows 53 and 76 us (e4m3 cache 39 and 89),
// 16 rows 57 and 77 (52 and 90), 24 rows, where keys are read twice, 95 and 77
// (82 and 90); 64 sequences over 1000 keys, 24 rows: 113 and 83 (121 and 98).
int seq_path(const cmpx_attention_seq_args* a, const SeqProblem& p) {
  const bool simt_ok = a->head_dim <= kSimtMaxD && (a->tokens_q * a->heads_q + 3) / 4 <= INT_MAX;
  const bool tile_ok = seq_tile_ok(p, a->dtype, a->kv_dtype);
  const bool decode_ok = seq_decode_ok(p, a->dtype, a->kv_dtype);
  if (a->path == CMPX_PATH_SIMT) return simt_ok ? CMPX_PATH_SIMT : -1;
  if (a->path == CMPX_PATH_TC) return tile_ok ? CMPX_PATH_TC : -1;
  if (a->path == CMPX_PATH_SKINNY) return decode_ok ? CMPX_PATH_SKINNY : -1;
  if (decode_ok && (typical_rows(a, p) <= 16 || !tile_ok)) return CMPX_PATH_SKINNY;
  return tile_ok ? CMPX_PATH_TC : simt_ok ? CMPX_PATH_SIMT : -1;
}

int decode_rows(const cmpx_attention_seq_args* a, const SeqProblem& p) { return typical_rows(a, p) <= 8 ? 8 : 16; }

size_t seq_workspace(const cmpx_attention_seq_args* a, const SeqProblem& p, int path, const DeviceInfo& dev) {
  return path == CMPX_PATH_TC       ? seq_tile_workspace(p, dev)
         : path == CMPX_PATH_SKINNY ? seq_decode_workspace(p, decode_rows(a, p), dev)
                                    : 0;
}

}  // namespace

bool seq_rows_ok(const void* base, int64_t stride, int64_t count, int64_t unit) {
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 &&
         (count <= 1 || (stride > 0 && stride % unit == 0 && stride < (int64_t(1) << 38)));
}

bool seq_tma_ok(const SeqProblem& p, int kv_dtype) {
  const bool paged = p.table != nullptr;
  if (paged && (p.page_size < 8 || (p.page_size & (p.page_size - 1)) != 0)) return false;
  if (paged ? (p.pages == 0 || p.max_keys == 0) : p.tokens_kv == 0) return false;  // no key at all
  const bool q8 = kv_dtype == CMPX_E4M3;
  const int64_t unit = q8 ? 16 : 8;
  for (const SeqKV* x : {&p.k, &p.v}) {
    // a page's scales are copied in 16-byte units
    if (q8 && (p.page_size < 16 || !seq_rows_ok(x->scale, x->s_head, p.heads_kv, 16) ||
               !seq_rows_ok(x->scale, x->s_page, p.pages, 16) || x->s_row != 1))
      return false;
    if (!seq_rows_ok(x->base, x->row, paged ? p.page_size : p.tokens_kv, unit) ||
        !seq_rows_ok(x->base, x->head, p.heads_kv, unit) || (paged && !seq_rows_ok(x->base, x->page, p.pages, unit)))
      return false;
  }
  return true;
}

bool seq_rows_map(CUtensorMap* m, int dtype, const void* base, const uint64_t (&dims)[4], const int64_t (&strides)[3],
                  uint32_t box0, uint32_t box1, uint32_t box3, uint32_t swizzle_bytes) {
  const uint64_t es = dtype == CMPX_E4M3 ? 1 : 2;
  uint64_t bytes[3];
  for (int i = 0; i < 3; ++i) bytes[i] = dims[i + 1] > 1 ? uint64_t(strides[i]) * es : dims[0] * es;
  return encode_tmap_4d(m, dtype, base, dims, bytes, box0, box1, box3, swizzle_bytes) == CMPX_OK;
}

bool seq_kv_maps(const SeqProblem& p, int kv_dtype, int box_rows, bool swizzled, CUtensorMap* tk, CUtensorMap* tv) {
  const bool paged = p.table != nullptr, q8 = kv_dtype == CMPX_E4M3;
  const uint64_t dims[4] = {uint64_t(p.d), uint64_t(paged ? p.page_size : p.tokens_kv), uint64_t(p.heads_kv),
                            uint64_t(paged ? p.pages : 1)};
  const uint32_t inner = q8 ? uint32_t(p.d) : 64u;
  const uint32_t swizzle = !swizzled ? 0u : q8 ? uint32_t(p.d) : 128u;
  const int64_t ks[3] = {p.k.row, p.k.head, p.k.page}, vs[3] = {p.v.row, p.v.head, p.v.page};
  return seq_rows_map(tk, kv_dtype, p.k.base, dims, ks, inner, uint32_t(box_rows), 1, swizzle) &&
         seq_rows_map(tv, kv_dtype, p.v.base, dims, vs, inner, uint32_t(box_rows), 1, swizzle);
}

cudaError_t launch_seq_simt(const SeqProblem& p, int dtype, int kv_dtype, cudaStream_t s) {
  if (kv_dtype == CMPX_E4M3)
    return dtype == CMPX_F16    ? launch_simt_typed<__half, uint8_t>(p, s)
           : dtype == CMPX_BF16 ? launch_simt_typed<__nv_bfloat16, uint8_t>(p, s)
                                : launch_simt_typed<float, uint8_t>(p, s);
  return dtype == CMPX_F16    ? launch_simt_typed<__half, __half>(p, s)
         : dtype == CMPX_BF16 ? launch_simt_typed<__nv_bfloat16, __nv_bfloat16>(p, s)
                              : launch_simt_typed<float, float>(p, s);
}

}  // namespace cmpx

using namespace cmpx;

extern "C" int cmpx_attention_seq(const cmpx_attention_seq_args* args, cmpx_stream_t stream) {
  bool empty = false;
  int st = validate_seq(args, &empty);
  if (st != CMPX_OK || empty) return st;
  const SeqProblem p = resolve_seq(args);
  const int path = seq_path(args, p);
  if (path < 0) return CMPX_ERR_UNSUPPORTED;
  DeviceInfo dev;
  int* err = nullptr;
  st = device_facts(&dev, &err);
  if (st != CMPX_OK) return st;
  const size_t need = seq_workspace(args, p, path, dev);
  if (need > 0 && (args->workspace == nullptr || reinterpret_cast<uintptr_t>(args->workspace) % 16 != 0))
    return CMPX_ERR_INVALID_ARG;
  if (args->workspace_bytes < need) return CMPX_ERR_WORKSPACE;
  const cudaError_t e =
      path == CMPX_PATH_SKINNY
          ? launch_seq_decode(p, args->dtype, args->kv_dtype, decode_rows(args, p), args->workspace, dev, err,
                              stream)
      : path == CMPX_PATH_TC ? launch_seq_tile(p, args->dtype, args->kv_dtype, args->workspace, dev, err, stream)
                           : launch_seq_simt(p, args->dtype, args->kv_dtype, stream);
  return e == cudaSuccess ? CMPX_OK : CMPX_ERR_CUDA;
}

extern "C" size_t cmpx_attention_seq_workspace_size(const cmpx_attention_seq_args* args) {
  bool empty = false;
  if (validate_seq(args, &empty) != CMPX_OK || empty) return 0;
  const SeqProblem p = resolve_seq(args);
  DeviceInfo dev;
  int* err = nullptr;
  if (device_facts(&dev, &err) != CMPX_OK) return 0;
  return seq_workspace(args, p, seq_path(args, p), dev);
}

extern "C" int cmpx_attention_seq_select_path(const cmpx_attention_seq_args* args) {
  bool empty = false;
  if (validate_seq(args, &empty) != CMPX_OK) return -1;
  return empty ? CMPX_PATH_SIMT : seq_path(args, resolve_seq(args));
}
