// Element types of a logits row (fp32, bf16, fp16) as the kernels read them: 16-byte vectors, their
// largest element, and exact up-casts to fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace pb {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int ES = 4, EPV = 4;
  static constexpr uint32_t NEG_INF_WORD = 0xFF800000u;  // a 32-bit word of -inf elements
  __device__ static float ld(const float* p) { return __ldg(p); }
  // NaN-propagating max of the elements of two words, lane by lane (a word holds 1 or 2 elements)
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(r);
  }
  // the largest element of a word, as fp32 (NaN if it holds one)
  __device__ static float word_max(uint32_t w) { return __uint_as_float(w); }
  // element q (runtime index < EPV) of a vector, as fp32
  __device__ static float elem(uint4 v, int q) {
    const uint32_t w = (q & 2) ? ((q & 1) ? v.w : v.z) : ((q & 1) ? v.y : v.x);
    return __uint_as_float(w);
  }
  __device__ static void unpack(uint4 v, float* x) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int ES = 2, EPV = 8;
  static constexpr uint32_t NEG_INF_WORD = 0xFF80FF80u;
  __device__ static float ld(const __nv_bfloat16* p) {
    return __uint_as_float(((uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p))) << 16);
  }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static float word_max(uint32_t w) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(w << 16)), "f"(__uint_as_float(w & 0xFFFF0000u)));
    return r;
  }
  __device__ static float elem(uint4 v, int q) {
    const uint32_t w = (q & 4) ? ((q & 2) ? v.w : v.z) : ((q & 2) ? v.y : v.x);
    return __uint_as_float((q & 1) ? (w & 0xFFFF0000u) : (w << 16));
  }
  __device__ static void unpack(uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Elem<__half> {
  static constexpr int ES = 2, EPV = 8;
  static constexpr uint32_t NEG_INF_WORD = 0xFC00FC00u;
  __device__ static float ld(const __half* p) { return __half2float(__ldg(p)); }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static float word_max(uint32_t w) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;"
        : "=f"(r)
        : "f"(__half2float(__ushort_as_half((unsigned short)(w & 0xFFFF)))),
          "f"(__half2float(__ushort_as_half((unsigned short)(w >> 16)))));
    return r;
  }
  __device__ static float elem(uint4 v, int q) {
    const uint32_t w = (q & 4) ? ((q & 2) ? v.w : v.z) : ((q & 2) ? v.y : v.x);
    return __half2float(__ushort_as_half((unsigned short)((q & 1) ? (w >> 16) : (w & 0xFFFF))));
  }
  __device__ static void unpack(uint4 v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __half2float(__ushort_as_half((unsigned short)(w[i] & 0xFFFF)));
      x[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16)));
    }
  }
};

}  // namespace pb
