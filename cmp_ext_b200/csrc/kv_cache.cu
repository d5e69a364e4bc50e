// Paged key / value cache: new tokens written (quantised to e4m3 with one
// power-of-two scale a vector, or copied) and tokens read back.  No
// counterpart in the reference.
//
// The scale is 2^e with e the smallest integer that brings the vector's
// largest magnitude to at most e4m3's 448.  x * 2^-e and code * 2^e are exact
// in fp32, so e4m3's rounding is the only one; a power of two costs no
// precision against max / 448, since e4m3 keeps four significant bits at any
// magnitude down to 2^-6 and the scale only moves which magnitudes those are.
#include <cuda_fp8.h>

#include <climits>
#include <cstring>
#include <type_traits>

#include "attention_math.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace cmpx {
namespace {

// One of the two tensors (keys or values) of a call.
struct Side {
  void* x;          // [tokens][heads][d]
  void* cache;      // [pages][heads][page_size][d]
  uint8_t* scale;   // [pages][heads][page_size]
  int64_t x_token, x_head, c_page, c_head, c_row, s_page, s_head, s_row;
};
struct CacheCall {
  Side side[2];
  const int64_t* slots;
  int64_t slot_end;  // pages * page_size
  uint32_t vectors;  // tokens * heads (32 bits: a 64-bit division for each lane took longer than its memory traffic)
  int heads, d, page_size;
};

// N consecutive values of a vector, moved as one access of their whole size
// (copied as a struct of bytes they would be loaded one by one).
template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};
template <int BYTES>
struct Raw;
template <> struct Raw<1> { using type = uint8_t; };
template <> struct Raw<2> { using type = uint16_t; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  const auto r = *reinterpret_cast<const typename Raw<sizeof(Pack<T, N>)>::type*>(p);
  Pack<T, N> x;
  memcpy(&x, &r, sizeof(x));
  return x;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& x) {
  typename Raw<sizeof(x)>::type r;
  memcpy(&r, &x, sizeof(x));
  *reinterpret_cast<decltype(r)*>(p) = r;
}

// e4m3 scale byte of a vector whose largest magnitude is a: the exponent of
// the smallest power of two 2^e with a <= 448 * 2^e = 1.75 * 2^(e + 8).  Both
// come from a's own bits: a = m * 2^k gives e = k - 8, plus one if m > 1.75.
__device__ __forceinline__ uint32_t scale_byte(float a) {
  const uint32_t bits = __float_as_uint(a);
  if (bits == 0) return 127;            // all zeros: scale 1
  if (bits >= 0x7f800000u) return 255;  // infinity or NaN
  const int b = int(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return uint32_t(max(b, 0));           // below 2^-127 the smallest scale serves
}
// max that keeps a NaN (fmaxf would drop it)
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Largest magnitude of a pack, NaN if one is.
template <typename T, int N>
__device__ __forceinline__ float top_of(const Pack<T, N>& x) {
  if constexpr (sizeof(T) == 2 && N >= 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 top = __habs2(*reinterpret_cast<const T2*>(&x.v[0]));
#pragma unroll
    for (int k = 2; k < N; k += 2) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const T2*>(&x.v[k])));
    return max_nan(ldf(reinterpret_cast<const T*>(&top)), ldf(reinterpret_cast<const T*>(&top) + 1));
  } else {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) top = max_nan(top, fabsf(ldf(&x.v[k])));
    return top;
  }
}

struct Place {
  int64_t page;
  int row;
  bool there;
};
__device__ __forceinline__ Place place_of(const CacheCall& c, int64_t slot) {
  Place r;
  r.there = slot >= 0 && slot < c.slot_end;
  if (c.slot_end <= INT_MAX) {  // the usual case: a 32-bit division
    const uint32_t s = r.there ? uint32_t(slot) : 0u;
    r.page = s / uint32_t(c.page_size);
    r.row = int(s - uint32_t(r.page) * uint32_t(c.page_size));
  } else {
    const int64_t s = r.there ? slot : 0;
    r.page = s / c.page_size;
    r.row = int(s - r.page * c.page_size);
  }
  return r;
}

// A group of 2^lg lanes owns one vector of keys and the same token's vector
// of values; a lane holds NC chunks of VEC consecutive values of each, so the
// largest magnitude takes lg shuffles and the vector is read once, before the
// slot that says where it goes is needed.
//
// Bound by memory once the instructions are few: 64-bit divisions, one chunk
// a lane and conversions value by value made 16384 tokens of 8 heads of 128
// (bf16 to e4m3) take 36 us, with 32-bit ones, two chunks a lane and pairs
// 23 us (4.4 TB/s); several vectors a lane lose more threads than they hide
// latency (25 us with two, 59 with four).
template <typename T, bool Q8, int VEC, int NC>
__global__ void __launch_bounds__(256) kv_write_kernel(const CacheCall c, int lg) {
  using C = typename std::conditional<Q8, __nv_fp8_storage_t, T>::type;
  pdl_trigger();
  pdl_wait();
  const uint32_t vec = blockIdx.x * (256u >> lg) + (threadIdx.x >> lg);
  const int lane = threadIdx.x & ((1 << lg) - 1);
  if (vec >= c.vectors) return;  // whole groups leave together
  const uint32_t token = vec / uint32_t(c.heads);
  const int head = int(vec - token * uint32_t(c.heads));
  const int64_t slot = __ldg(c.slots + token);
  Pack<T, VEC> x[2][NC];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const T* src = static_cast<const T*>(c.side[s].x) + token * c.side[s].x_token + head * c.side[s].x_head;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int d = (lane + (i << lg)) * VEC;
      if (d < c.d) x[s][i] = load_pack<T, VEC>(src + d);
    }
  }
  const Place at = place_of(c, slot);
  if (!at.there) return;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    C* dst = static_cast<C*>(c.side[s].cache) + at.page * c.side[s].c_page + head * c.side[s].c_head +
             at.row * c.side[s].c_row;
    if constexpr (Q8) {
      float a = 0.0f;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if ((lane + (i << lg)) * VEC < c.d) a = max_nan(a, top_of(x[s][i]));
      // the lanes of a group leave the kernel together, so they are the mask
      const unsigned mask = lg == 5 ? 0xffffffffu : ((1u << (1 << lg)) - 1u) << (threadIdx.x & 31 & ~((1 << lg) - 1));
      for (int o = 1 << lg >> 1; o > 0; o >>= 1) a = max_nan(a, __shfl_xor_sync(mask, a, o));
      const uint32_t b = scale_byte(a);
      const float down = b == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - b) << 23);  // 2^-e
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int d = (lane + (i << lg)) * VEC;
        if (d >= c.d) continue;
        Pack<C, VEC> q;
        if constexpr (VEC == 1) {
          q.v[0] = __nv_cvt_float_to_fp8(ldf(&x[s][i].v[0]) * down, __NV_SATFINITE, __NV_E4M3);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; k += 2) {
            const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(
                make_float2(ldf(&x[s][i].v[k]) * down, ldf(&x[s][i].v[k + 1]) * down), __NV_SATFINITE, __NV_E4M3);
            q.v[k] = uint8_t(two);
            q.v[k + 1] = uint8_t(two >> 8);
          }
        }
        store_pack(dst + d, q);
      }
      if (lane == 0)
        c.side[s].scale[at.page * c.side[s].s_page + head * c.side[s].s_head + at.row * c.side[s].s_row] = uint8_t(b);
    } else {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int d = (lane + (i << lg)) * VEC;
        if (d < c.d) store_pack(dst + d, x[s][i]);
      }
    }
  }
}

// Stores x rounded to T; what lies beyond T's largest value becomes that
// value (the largest magnitudes can round up to the next power of two in
// e4m3).  A NaN stays one.
template <typename T>
__device__ __forceinline__ void st_sat(T* p, float x) {
  constexpr float top = std::is_same<T, __half>::value ? 65504.0f
                        : std::is_same<T, __nv_bfloat16>::value ? 3.3895313892515355e38f : 3.4028234663852886e38f;
  stf(p, x > top ? top : x < -top ? -top : x);
}

// The other way, with the same layout of threads.  The slot's latency and the
// codes' cannot overlap within a thread: 65500 tokens of 8 heads of 128 (e4m3
// to bf16, scattered slots) take 87-94 us (4.3-4.7 TB/s), 131 us before the same
// changes.
template <typename T, bool Q8, int VEC, int NC>
__global__ void __launch_bounds__(256) kv_read_kernel(const CacheCall c, int lg) {
  using C = typename std::conditional<Q8, __nv_fp8_storage_t, T>::type;
  pdl_trigger();
  pdl_wait();
  const uint32_t vec = blockIdx.x * (256u >> lg) + (threadIdx.x >> lg);
  const int lane = threadIdx.x & ((1 << lg) - 1);
  if (vec >= c.vectors) return;
  const uint32_t token = vec / uint32_t(c.heads);
  const int head = int(vec - token * uint32_t(c.heads));
  const Place at = place_of(c, __ldg(c.slots + token));
  Pack<C, VEC> x[2][NC];
  uint8_t scale[2] = {0, 0};
  if (at.there) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const C* src = static_cast<const C*>(c.side[s].cache) + at.page * c.side[s].c_page + head * c.side[s].c_head +
                     at.row * c.side[s].c_row;
      if (Q8) scale[s] = c.side[s].scale[at.page * c.side[s].s_page + head * c.side[s].s_head + at.row * c.side[s].s_row];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int d = (lane + (i << lg)) * VEC;
        if (d < c.d) x[s][i] = load_pack<C, VEC>(src + d);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    T* dst = static_cast<T*>(c.side[s].x) + token * c.side[s].x_token + head * c.side[s].x_head;
    const float up = e8m0_to_float(scale[s]);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int d = (lane + (i << lg)) * VEC;
      if (d >= c.d) continue;
      Pack<T, VEC> y;
      if (!at.there) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) stf(&y.v[k], 0.0f);
      } else if constexpr (!Q8) {
        y = x[s][i];
      } else if constexpr (sizeof(T) == 2 && VEC >= 2) {
#pragma unroll
        for (int k = 0; k < VEC; k += 2) {
          const uint32_t two = dequant2(uint32_t(x[s][i].v[k]) | uint32_t(x[s][i].v[k + 1]) << 8, up, (T*)nullptr);
          memcpy(&y.v[k], &two, 4);
        }
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          st_sat(&y.v[k], __half2float(__half(__nv_cvt_fp8_to_halfraw(x[s][i].v[k], __NV_E4M3))) * up);
      }
      store_pack(dst + d, y);
    }
  }
}

template <typename T, bool Q8, int VEC, int NC>
cudaError_t launch_rows(const CacheCall& c, int lg, bool write, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(((int64_t(c.vectors) << lg) + 255) / 256));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  apply_pdl(cfg, attr, 0);
  return cudaLaunchKernelEx(&cfg, write ? kv_write_kernel<T, Q8, VEC, NC> : kv_read_kernel<T, Q8, VEC, NC>, c, lg);
}

// wide: 16-byte accesses of T (VEC = 16 / sizeof(T)), two a lane where the
// vector has them (a lane's address arithmetic costs as much as its data);
// otherwise single values.
template <typename T, bool Q8>
cudaError_t launch_typed(const CacheCall& c, bool wide, bool write, cudaStream_t s) {
  constexpr int W = 16 / int(sizeof(T));
  int lg = 0;
  if (!wide) {
    while (lg < 5 && (1 << lg) < c.d) ++lg;
    return launch_rows<T, Q8, 1, kSimtMaxD / 32>(c, lg, write, s);
  }
  while (lg < 5 && (2 * W << lg) < c.d) ++lg;
  if (c.d <= (2 * W << lg)) return launch_rows<T, Q8, W, 2>(c, lg, write, s);
  return launch_rows<T, Q8, W, kSimtMaxD / (32 * W)>(c, lg, write, s);
}

int run_cache(const cmpx_kv_cache_args* a, bool write, cudaStream_t s) {
  if (a == nullptr) return CMPX_ERR_INVALID_ARG;
  if (a->dtype != CMPX_F16 && a->dtype != CMPX_BF16 && a->dtype != CMPX_F32) return CMPX_ERR_INVALID_ARG;
  if (a->cache_dtype != a->dtype && a->cache_dtype != CMPX_E4M3) return CMPX_ERR_INVALID_ARG;
  if (a->tokens < 0 || a->heads < 0 || a->head_dim < 0 || a->pages < 0 || a->page_size < 0) return CMPX_ERR_INVALID_ARG;
  const int64_t strides[] = {a->key_stride_token, a->key_stride_head, a->value_stride_token, a->value_stride_head,
                             a->kc_stride_page, a->kc_stride_head, a->kc_stride_row, a->vc_stride_page,
                             a->vc_stride_head, a->vc_stride_row, a->ks_stride_page, a->ks_stride_head,
                             a->ks_stride_row, a->vs_stride_page, a->vs_stride_head, a->vs_stride_row};
  for (int64_t x : strides)
    if (x < 0) return CMPX_ERR_INVALID_ARG;
  if (a->tokens == 0 || a->heads == 0 || a->head_dim == 0) return CMPX_OK;
  if (a->key == nullptr || a->value == nullptr || a->slots == nullptr) return CMPX_ERR_INVALID_ARG;
  const bool q8 = a->cache_dtype == CMPX_E4M3;
  const bool empty_cache = a->pages == 0 || a->page_size == 0;
  if (!empty_cache && (a->key_cache == nullptr || a->value_cache == nullptr)) return CMPX_ERR_INVALID_ARG;
  if (!empty_cache && q8 && (a->key_scale == nullptr || a->value_scale == nullptr)) return CMPX_ERR_INVALID_ARG;
  if (a->head_dim > kSimtMaxD) return CMPX_ERR_UNSUPPORTED;
  if (a->page_size > INT_MAX || a->heads > INT_MAX || a->tokens > INT_MAX ||
      a->tokens * a->heads > INT_MAX)
    return CMPX_ERR_UNSUPPORTED;
  if (!empty_cache && a->pages > INT64_MAX / a->page_size) return CMPX_ERR_UNSUPPORTED;
  if (empty_cache && write) return CMPX_OK;  // every slot is outside
  DeviceInfo dev;
  int* err = nullptr;
  const int st = device_facts(&dev, &err);
  if (st != CMPX_OK) return st;

  CacheCall c = {};
  c.side[0] = Side{a->key, a->key_cache, static_cast<uint8_t*>(a->key_scale), a->key_stride_token, a->key_stride_head,
                   a->kc_stride_page, a->kc_stride_head, a->kc_stride_row, a->ks_stride_page, a->ks_stride_head,
                   a->ks_stride_row};
  c.side[1] = Side{a->value, a->value_cache, static_cast<uint8_t*>(a->value_scale), a->value_stride_token,
                   a->value_stride_head, a->vc_stride_page, a->vc_stride_head, a->vc_stride_row, a->vs_stride_page,
                   a->vs_stride_head, a->vs_stride_row};
  c.slots = a->slots;
  c.slot_end = empty_cache ? 0 : a->pages * a->page_size;
  c.vectors = uint32_t(a->tokens * a->heads);
  c.heads = int(a->heads);
  c.d = int(a->head_dim);
  c.page_size = empty_cache ? 1 : int(a->page_size);
  // wide accesses: every vector starts on 16 bytes in key / value and on the
  // bytes of as many codes in the cache
  const int64_t es = elem_bytes(a->dtype), w = 16 / es, cb = (q8 ? 1 : es) * w;
  bool wide = c.d % w == 0;
  for (const Side& x : c.side) {
    wide = wide && reinterpret_cast<uintptr_t>(x.x) % 16 == 0 && x.x_token % w == 0 && x.x_head % w == 0;
    wide = wide && (empty_cache || reinterpret_cast<uintptr_t>(x.cache) % cb == 0) && x.c_page % w == 0 &&
           x.c_head % w == 0 && x.c_row % w == 0;
  }
  cudaError_t e;
  if (a->dtype == CMPX_F16)
    e = q8 ? launch_typed<__half, true>(c, wide, write, s) : launch_typed<__half, false>(c, wide, write, s);
  else if (a->dtype == CMPX_BF16)
    e = q8 ? launch_typed<__nv_bfloat16, true>(c, wide, write, s) : launch_typed<__nv_bfloat16, false>(c, wide, write, s);
  else
    e = q8 ? launch_typed<float, true>(c, wide, write, s) : launch_typed<float, false>(c, wide, write, s);
  return e == cudaSuccess ? CMPX_OK : CMPX_ERR_CUDA;
}

}  // namespace
}  // namespace cmpx

extern "C" int cmpx_kv_cache_write(const cmpx_kv_cache_args* args, cmpx_stream_t stream) {
  return cmpx::run_cache(args, true, stream);
}

extern "C" int cmpx_kv_cache_read(const cmpx_kv_cache_args* args, cmpx_stream_t stream) {
  return cmpx::run_cache(args, false, stream);
}
