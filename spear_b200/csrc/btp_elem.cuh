// Storage types of the token-major operators (scan, convolution, norm): conversion to and from float, and loads and
// stores of runs of consecutive elements that fall back to single elements where a row is not aligned or ends.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace btp_elem {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// N consecutive elements as whole 16-byte (or smaller) words.
template <class T, int N>
struct alignas((N & (N - 1)) != 0 ? sizeof(T) : sizeof(T) * N >= 16 ? 16 : sizeof(T) * N) Pack {
  T v[N];
};

// out[0..N) = p[0..N) as floats; elements from `count` on are 0 and are not read.  `aligned`: p is a multiple of the
// pack's size (16 bytes at most) and all N elements may be read.
template <class T, int N>
__device__ __forceinline__ void load_run(float (&out)[N], const T* p, bool aligned, int count) {
  if (aligned) {
    const Pack<T, N> w = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_f(w.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = i < count ? to_f(p[i]) : 0.f;
  }
}

template <class T, int N>
__device__ __forceinline__ void store_run(T* p, const float (&in)[N], bool aligned, int count) {
  if (aligned) {
    Pack<T, N> w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.v[i] = from_f<T>(in[i]);
    *reinterpret_cast<Pack<T, N>*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < count) p[i] = from_f<T>(in[i]);
  }
}

// A parameter vector that is stored in the activations' type or in float.
template <class T, int N>
__device__ __forceinline__ void load_param(float (&out)[N], const void* base, long long at, bool is_f32, bool aligned, int count) {
  if (is_f32)
    load_run<float, N>(out, static_cast<const float*>(base) + at, aligned, count);
  else
    load_run<T, N>(out, static_cast<const T*>(base) + at, aligned, count);
}

// 2^v, 1/v on the special-function unit (2 and 1 units in the last place).
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
// 1 / (1 + e^-v); the exponent's rounding makes it |v| 2^-24 off relative for very negative v, a few 2^-24 elsewhere.
__device__ __forceinline__ float sigmoid(float v) { return rcp(1.f + ex2(-v * kLog2e)); }

// log(1 + e^v) to a few units in the last place, without overflow:  max(v, 0) + log(1 + w) with w = e^-|v| <= 1, and
// log(1 + w) = 2 atanh(s), s = w / (2 + w) <= 1/3, by the series s + s^3/3 + s^5/5 + ... up to s^15 (the rest is below 2^-28).
__device__ __forceinline__ float softplus(float v) {
  const float w = ex2(-fabsf(v) * kLog2e);
  const float s = w * rcp(2.f + w), q = s * s;
  float p = 2.f / 15.f;
  p = fmaf(p, q, 2.f / 13.f);
  p = fmaf(p, q, 2.f / 11.f);
  p = fmaf(p, q, 2.f / 9.f);
  p = fmaf(p, q, 2.f / 7.f);
  p = fmaf(p, q, 2.f / 5.f);
  p = fmaf(p, q, 2.f / 3.f);
  p = fmaf(p, q, 2.f);
  return (v < 0.f ? 0.f : v) + p * s;  // not fmaxf: NaN stays
}

// Two floats side by side in one 64-bit register pair: one instruction does the arithmetic of both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(float& lo, float& hi, f32x2 v) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ float lo2(f32x2 v) {
  float a, b;
  unpack2(a, b, v);
  return a;
}
__device__ __forceinline__ float hi2(f32x2 v) {
  float a, b;
  unpack2(a, b, v);
  return b;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 ex2_2(f32x2 v) { return pack2(ex2(lo2(v)), ex2(hi2(v))); }

// Tokens of sequence b that are there: `lengths` may be null (all L), its values are held to 0 ... L.
__device__ __forceinline__ int tokens_of(const int* lengths, long long b, int L) {
  if (!lengths) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : (n < L ? n : L);
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace btp_elem
