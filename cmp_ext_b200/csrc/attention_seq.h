// Problem description shared by the kernels behind cmpx_attention_seq
// (attention_seq.cu: checks, dispatch, CUDA-core kernel).
#pragma once
#include <cstdint>
#include <type_traits>

#include "attention_math.cuh"
#include "internal.h"

namespace cmpx {

// Keys or values: rows of one kv head, in a packed tensor or in pages.
struct SeqKV {
  const void* base;
  int64_t row, head, page;        // strides (elements)
  const uint8_t* scale;           // e8m0 bytes of an 8-bit cache, else nullptr
  int64_t s_row, s_head, s_page;  // their strides
};

struct SeqProblem {
  const void* Q;
  void* O;
  int64_t q_token, q_head, o_token, o_head;  // strides (elements)
  SeqKV k, v;
  const int* cu_q;    // nullptr: uniform_n tokens each
  const int* cu_k;    // packed form
  const int* table;   // paged form, else nullptr
  const int* lens_k;  // paged form
  int64_t table_stride;
  int batch, uniform_n, tokens_q, tokens_kv, heads_q, heads_kv, group, d;
  int page_size, pages, max_keys;  // max_keys: keys a row of the page table can name
  int page_lg;                     // log2 page_size where that is whole (the TMA kernels')
  float scale_log2;                // scale * log2 e
  int causal, zero_rest;
};

// One sequence: query tokens [q0, q0 + n), keys [k0, k0 + len) of the packed
// tensor (k0 = 0 in the paged form).
struct Seq {
  int q0, n, k0, len;
};

#ifdef __CUDACC__
// Clamped, so that lengths no caller should pass never lead outside a tensor.
__device__ __forceinline__ int2 seq_queries(const SeqProblem& p, int b) {
  if (p.cu_q == nullptr) return make_int2(b * p.uniform_n, p.uniform_n);
  const int q0 = min(max(__ldg(p.cu_q + b), 0), p.tokens_q);
  const int q1 = min(max(__ldg(p.cu_q + b + 1), q0), p.tokens_q);
  return make_int2(q0, q1 - q0);
}
__device__ __forceinline__ Seq seq_of(const SeqProblem& p, int b) {
  Seq s;
  const int2 q = seq_queries(p, b);
  s.q0 = q.x;
  s.n = q.y;
  if (p.table != nullptr) {
    s.k0 = 0;
    s.len = min(max(__ldg(p.lens_k + b), 0), p.max_keys);
  } else if (p.cu_k != nullptr) {
    s.k0 = min(max(__ldg(p.cu_k + b), 0), p.tokens_kv);
    s.len = min(max(__ldg(p.cu_k + b + 1), s.k0), p.tokens_kv) - s.k0;
  } else {
    s.k0 = min(s.q0, p.tokens_kv);
    s.len = min(s.n, p.tokens_kv - s.k0);
  }
  return s;
}
// Keys that query token i of a sequence sees: the first seq_limit() of them.
__device__ __forceinline__ int seq_limit(const SeqProblem& p, const Seq& s, int i) {
  return p.causal ? min(max(s.len - s.n + i + 1, 0), s.len) : s.len;
}
// Records a bounded wait that ran out and ends the block's other waits.
__device__ __forceinline__ void rec_err(int* err, volatile int* abort, int code) {
  *abort = 1;
  atomicCAS(err, 0, code);
}
// Whether a value of keys [from, to) of a sequence is not finite (a warp
// looks; T the values' type, or uint8_t for e4m3 codes).  A row whose result
// is not finite although its sum is has to be computed again only if such a
// value is among those it may not see: it reaches the row through 0 * NaN.
template <typename T, int D>
__device__ __forceinline__ bool seq_hidden_bad(const SeqProblem& p, int b, int k0, int hk, int from, int to) {
  const int lane = threadIdx.x & 31;
  bool bad = false;
  for (int j = from; j < to; ++j) {
    int64_t at = int64_t(k0 + j) * p.v.row;
    if (p.table != nullptr) {
      const int page = __ldg(p.table + b * p.table_stride + j / p.page_size), slot = j % p.page_size;
      if (page < 0 || page >= p.pages) continue;  // zeros
      at = page * p.v.page + slot * p.v.row;
      if (sizeof(T) == 1) bad = bad || p.v.scale[page * p.v.s_page + hk * p.v.s_head + slot * p.v.s_row] == 255;
    }
    const T* v = static_cast<const T*>(p.v.base) + at + hk * p.v.head;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      if constexpr (sizeof(T) == 1) {
        bad = bad || (v[lane + 32 * i] & 0x7f) == 0x7f;
      } else {
        const float x = float(v[lane + 32 * i]);
        bad = bad || x - x != 0.0f;
      }
    }
  }
  return __any_sync(0xffffffffu, bad);
}
// One row over keys [kbeg, kend) of a sequence from its definition: the sums
// of weights 2^(x - m) times values.  A warp computes it, lane i the columns
// i, i + 32, ...
template <typename T, int D, bool Q8>
__device__ __forceinline__ void redo_row(const SeqProblem& p, int b, int k0, int hk, const T* q, int kbeg, int kend,
                                         float m, float (&acc)[D / 32]) {
  const int lane = threadIdx.x & 31;
  constexpr int NV = D / 32;
  using KV = typename std::conditional<Q8, uint8_t, T>::type;
  auto load = [](const KV* at, float up) -> float {
    if constexpr (Q8) return held<T>(*at, up);
    else return ldf(at);
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.0f;
  for (int j = kbeg; j < kend; ++j) {
    int64_t ko = int64_t(k0 + j) * p.k.row, vo = int64_t(k0 + j) * p.v.row;
    float ks = 1.0f, vs = 1.0f;
    if (p.table != nullptr) {
      const int page = __ldg(p.table + b * p.table_stride + j / p.page_size), slot = j % p.page_size;
      if (page < 0 || page >= p.pages) continue;  // reads as zeros: nothing to add
      ko = page * p.k.page + slot * p.k.row;
      vo = page * p.v.page + slot * p.v.row;
      if (Q8) {
        ks = e8m0_to_float(p.k.scale[page * p.k.s_page + hk * p.k.s_head + slot * p.k.s_row]);
        vs = e8m0_to_float(p.v.scale[page * p.v.s_page + hk * p.v.s_head + slot * p.v.s_row]);
      }
    }
    const KV* kr = static_cast<const KV*>(p.k.base) + ko + hk * p.k.head;
    const KV* vr = static_cast<const KV*>(p.v.base) + vo + hk * p.v.head;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) dot = fmaf(ldf(q + lane + 32 * i), load(kr + lane + 32 * i, ks), dot);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float w = ex2_approx(fmaf(dot, p.scale_log2, -m));
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = fmaf(w, load(vr + lane + 32 * i, vs), acc[i]);
  }
}
// x: tokens before the first sequence; y: first token behind the last one
// (the first and last offset, clamped).
__device__ __forceinline__ int2 seq_rest(const SeqProblem& p) {
  if (p.cu_q == nullptr) return make_int2(0, p.batch * p.uniform_n);
  return make_int2(min(max(__ldg(p.cu_q), 0), p.tokens_q), min(max(__ldg(p.cu_q + p.batch), 0), p.tokens_q));
}
#endif

// Host side of the kernels.  Each returns a cudaError_t of its launches.
cudaError_t launch_seq_simt(const SeqProblem& p, int dtype, int kv_dtype, cudaStream_t s);

// Whether TMA can describe a stride of `count` rows (in units that make 16
// bytes), and the keys and values of a problem.
bool seq_rows_ok(const void* base, int64_t stride, int64_t count, int64_t unit);
bool seq_tma_ok(const SeqProblem& p, int kv_dtype);
// 4-D map of rows, innermost dimension first, boxes {box0, box1, 1, box3};
// a dimension of one element takes any stride.
bool seq_rows_map(CUtensorMap* m, int dtype, const void* base, const uint64_t (&dims)[4], const int64_t (&strides)[3],
                  uint32_t box0, uint32_t box1, uint32_t box3, uint32_t swizzle_bytes);
// Maps of keys and values, boxes of box_rows keys of a head: 16-bit rows in
// 128-byte columns; 8-bit rows whole, swizzled by their own length or not.
bool seq_kv_maps(const SeqProblem& p, int kv_dtype, int box_rows, bool swizzled, CUtensorMap* tk, CUtensorMap* tv);

// flash-decoding kernel (attention_decode.cu)
bool seq_decode_ok(const SeqProblem& p, int dtype, int kv_dtype);
size_t seq_decode_workspace(const SeqProblem& p, int rows, const DeviceInfo& dev);
// rows: 8 or 16 query rows share a pass over the keys
cudaError_t launch_seq_decode(const SeqProblem& p, int dtype, int kv_dtype, int rows, void* ws, const DeviceInfo& dev,
                              int* err, cudaStream_t s);

// tcgen05 kernel (attention_tile.cu)
bool seq_tile_ok(const SeqProblem& p, int dtype, int kv_dtype);
size_t seq_tile_workspace(const SeqProblem& p, const DeviceInfo& dev);
cudaError_t launch_seq_tile(const SeqProblem& p, int dtype, int kv_dtype, void* ws, const DeviceInfo& dev, int* err,
                            cudaStream_t s);

}  // namespace cmpx
