// Arithmetic shared by the attention kernels: the base-2 exponential, paired
// fp32 instructions, packing to 16 bits and scalar loads / stores.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>
#include <type_traits>

namespace cmpx {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSimtMaxD = 512;  // largest head dimension of the CUDA-core kernels

// 2^x with the hardware's approximate base-2 exponential (ex2.approx,
// relative error ~2^-22; results below 2^-126 flush to zero, which a softmax
// weight that small does not need).  2^-inf = 0.
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Blackwell's paired fp32 arithmetic: two lanes in one 64-bit register, one
// instruction, each lane rounded exactly as the scalar fmaf / + (.rn), so a
// softmax written with them gives the same bits as the scalar one with about
// half the issue slots.  max3f is the three-input maximum (exact).
__device__ __forceinline__ uint64_t f2pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2unpack(uint64_t r) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ float ldf(const T* p);
template <>
__device__ __forceinline__ float ldf<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float ldf<__half>(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float ldf<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
// 2^(b - 127) for an e8m0 byte (NaN for 255).
__device__ __forceinline__ float e8m0_to_float(uint32_t b) {
  return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7fffffffu : b << 23);
}
// b - 127, its exponent (NaN for 255).
__device__ __forceinline__ float e8m0_exponent(uint32_t b) {
  return b == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float(0x4b000000u | b) - 8388735.0f;  // (2^23 + b) - ...
}
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void stf(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// What an 8-bit cache holds is the same to every kernel: code * 2^e rounded to
// the queries' type T, beyond its largest value that value.
// Two e4m3 codes times a scale, in T, saturating.
__device__ __forceinline__ uint32_t dequant2(uint32_t codes, float up, __half*) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y * up), "f"(f.x * up));
  return r;
}
__device__ __forceinline__ uint32_t dequant2(uint32_t codes, float up, __nv_bfloat16*) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes), __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  uint32_t r;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y * up), "f"(f.x * up));
  return r;
}
// One code, as a float (T = float: nothing to round to but fp32).
template <typename T>
__device__ __forceinline__ float held(uint32_t code, float up) {
  if constexpr (sizeof(T) == 4) {
    const float x = __half2float(__half(__nv_cvt_fp8_to_halfraw(__nv_fp8_storage_t(code), __NV_E4M3))) * up;
    return x > 3.4028234663852886e38f ? 3.4028234663852886e38f : x < -3.4028234663852886e38f ? -3.4028234663852886e38f : x;
  } else {
    const uint16_t one = uint16_t(dequant2(code, up, (T*)nullptr) & 0xffffu);
    return ldf(reinterpret_cast<const T*>(&one));
  }
}

// Four e4m3 codes as two fp16 pairs (exact): codes 0 and 1, codes 2 and 3.
__device__ __forceinline__ void e4m3_to_half(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
__device__ __forceinline__ uint32_t half2_to_bf16(uint32_t h2) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
  return pack2(f.x, f.y, (__nv_bfloat16*)nullptr);
}

// Whether the scale byte is one that scale4 takes: 2^e such that no code times
// it leaves T's finite range, and 2^e itself is a normal T.
__device__ __forceinline__ bool scale4_takes(uint32_t byte, __half*) { return byte >= 113 && byte <= 134; }
__device__ __forceinline__ bool scale4_takes(uint32_t byte, __nv_bfloat16*) { return byte >= 1 && byte <= 245; }
// Four e4m3 codes times 2^(byte - 127) in T, as two pairs; rounded like
// dequant2, with packed multiplications instead of fp32 ones.
__device__ __forceinline__ void scale4(uint32_t codes, uint32_t byte, uint32_t& lo, uint32_t& hi, __half*) {
  const uint32_t bits = (byte - 112) << 10, two = bits | bits << 16;
  uint32_t a, b;
  e4m3_to_half(codes, a, b);
  const __half2 s = *reinterpret_cast<const __half2*>(&two);
  const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&a), s), y = __hmul2(*reinterpret_cast<const __half2*>(&b), s);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ void scale4(uint32_t codes, uint32_t byte, uint32_t& lo, uint32_t& hi, __nv_bfloat16*) {
  const uint32_t two = byte << 7 | byte << 23;
  uint32_t a, b;
  e4m3_to_half(codes, a, b);
  a = half2_to_bf16(a);
  b = half2_to_bf16(b);
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&two);
  const __nv_bfloat162 x = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), s),
                       y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&b), s);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}


// For kernels that multiply codes and keep the scale 2^e outside:
// held(code, up) * down is the code whose product with 2^e T holds.
struct CodeScale {
  float up, down;  // 2^e, 2^-e
};
__device__ __forceinline__ CodeScale code_scale(uint32_t byte) {
  if (byte == 255) return CodeScale{1.0f, 1.0f};  // (the NaN stays outside)
  return CodeScale{e8m0_to_float(byte), e8m0_to_float(254u - byte)};
}

}  // namespace cmpx
