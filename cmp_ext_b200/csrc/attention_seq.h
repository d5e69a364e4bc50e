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
// Place of key j of a sequence's kv head hk in K and V (elements), and its
// scales of an 8-bit cache; false for a page that is none (zeros).
struct SeqKey {
  int64_t k, v;
  uint32_t k_scale, v_scale;
};
template <bool Q8>
__device__ __forceinline__ bool seq_key(const SeqProblem& p, int b, int k0, int hk, int j, SeqKey& x) {
  if (p.table == nullptr) {
    x.k = int64_t(k0 + j) * p.k.row + hk * p.k.head;
    x.v = int64_t(k0 + j) * p.v.row + hk * p.v.head;
    return true;
  }
  const int page = __ldg(p.table + b * p.table_stride + j / p.page_size), slot = j % p.page_size;
  if (page < 0 || page >= p.pages) return false;
  x.k = page * p.k.page + slot * p.k.row + hk * p.k.head;
  x.v = page * p.v.page + slot * p.v.row + hk * p.v.head;
  if constexpr (Q8) {
    x.k_scale = p.k.scale[page * p.k.s_page + hk * p.k.s_head + slot * p.k.s_row];
    x.v_scale = p.v.scale[page * p.v.s_page + hk * p.v.s_head + slot * p.v.s_row];
  }
  return true;
}
// The last of keys [from, to) of a sequence whose value is not finite, or -1
// (a warp looks, a lane a key).  A row whose result is not finite although its
// sum is has to be computed again only if such a value is among those it may
// not see: it reaches the row through 0 * NaN.  Rows of 16 bytes, as the
// tensor-core kernels take them.
template <typename T, int D, bool Q8>
__device__ __forceinline__ int seq_last_bad(const SeqProblem& p, int b, int k0, int hk, int from, int to) {
  int last = -1;
  for (int j = from + int(threadIdx.x & 31); j < to; j += 32) {
    SeqKey x;
    if (!seq_key<Q8>(p, b, k0, hk, j, x)) continue;
    const uint4* row = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.v.base) + x.v * (Q8 ? 1 : 2));
    bool bad = Q8 && x.v_scale == 255;
#pragma unroll 2
    for (int i = 0; i < D * (Q8 ? 1 : 2) / 16; ++i) {
      const uint4 u = __ldg(row + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (Q8) {
          bad = bad || __vcmpeq4(w[k] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
        } else {
          constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
          bad = bad || (w[k] & E) == E || (w[k] >> 16 & E) == E;
        }
      }
    }
    if (bad) last = j;
  }
  return __reduce_max_sync(0xffffffffu, last);
}
// R rows of a kv head from their definition, row r over keys [kbeg, lim[r]) of
// a sequence: the sums of weights 2^(x - m[r]) times values.  A warp computes
// them, lane i the columns i, i + 32, ... of the sums.  32 keys at a time, a
// lane a key's scores and then all lanes a key's value: key by key and row by
// row, with a sum over the lanes for each score, a key took a microsecond (40 x
// 40 new tokens over 16384 keys with a NaN beside them 260 ms, this way 60, and
// 0.8 without one), and a million of them the time that other warps wait for.
template <typename T, int D, bool Q8, int R>
__device__ __forceinline__ void redo_rows(const SeqProblem& p, int b, int k0, int hk, const T* const (&q)[R], int kbeg,
                                          const int (&lim)[R], const float (&m)[R], float (&acc)[R][D / 32]) {
  const int lane = threadIdx.x & 31;
  constexpr int NV = D / 32, CHUNK = 8;  // of columns
  int kend = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    kend = max(kend, lim[r]);
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[r][i] = 0.0f;
  }
#pragma unroll 1
  for (int base = kbeg; base < kend; base += 32) {
    SeqKey x = {};  // (of a page that is none, or behind the last key: the first row, not used)
    const bool there = base + lane < kend && seq_key<Q8>(p, b, k0, hk, base + lane, x);
    if (!there) x = SeqKey{};
    float w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = 0.0f;
    const float up = Q8 ? e8m0_to_float(x.k_scale) : 1.0f;
#pragma unroll(R == 1 ? 1 : 2)
    for (int c = 0; c < D; c += CHUNK) {
      float k[CHUNK];
      if constexpr (Q8) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.k.base) + x.k + c));
#pragma unroll
        for (int i = 0; i < CHUNK; i += 2) {
          const uint32_t two = dequant2((i < 4 ? u.x : u.y) >> 8 * (i & 3) & 0xffffu, up, (T*)nullptr);
          k[i] = ldf(reinterpret_cast<const T*>(&two));
          k[i + 1] = ldf(reinterpret_cast<const T*>(&two) + 1);
        }
      } else {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.k.base) + x.k + c));
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) k[i] = ldf(reinterpret_cast<const T*>(&u) + i);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(q[r] + c));
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) w[r] = fmaf(ldf(reinterpret_cast<const T*>(&u) + i), k[i], w[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = ex2_approx(fmaf(w[r], p.scale_log2, -m[r]));
    const float vs = Q8 ? e8m0_to_float(x.v_scale) : 1.0f;
    const unsigned present = __ballot_sync(0xffffffffu, there);
#pragma unroll(R == 1 ? 4 : 2)
    for (int t = 0; t < 32; ++t) {
      const float st = Q8 ? __shfl_sync(0xffffffffu, vs, t) : 1.0f;
      const int64_t at = __shfl_sync(0xffffffffu, (long long)x.v, t);
      const bool on = present >> t & 1;
      float v[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if constexpr (Q8) v[i] = held<T>(static_cast<const uint8_t*>(p.v.base)[at + lane + 32 * i], st);
        else v[i] = ldf(static_cast<const T*>(p.v.base) + at + lane + 32 * i);
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float wt = __shfl_sync(0xffffffffu, w[r], t);
        if (on && base + t < lim[r])
#pragma unroll
          for (int i = 0; i < NV; ++i) acc[r][i] = fmaf(wt, v[i], acc[r][i]);
      }
    }
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
