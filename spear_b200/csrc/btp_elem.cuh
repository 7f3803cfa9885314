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

__device__ __forceinline__ f32x2 both(float v) { return pack2(v, v); }

// e^-a for a >= 0: the product a log2(e) is rounded, and log2(e) is too; what that leaves of the exponent (up to a 2^-24, the largest
// error otherwise) comes back as a factor.  From 128 on the result is 0; a NaN stays.
constexpr float kEx2Low = 5e-8f;  // by which ex2.approx is low on average away from 0, relative
constexpr float kLog2eLow = 1.92596299e-8f, kLn2 = 0.6931471805599453f;  // log2(e) - kLog2e, log(2)
__device__ __forceinline__ float at_most_128(float a) {
  asm("min.NaN.f32 %0, %0, 0f43000000;" : "+f"(a));
  return a;
}
__device__ __forceinline__ float exp_minus(float a) {
  a = at_most_128(a);
  const float t = a * -kLog2e, w = ex2(t);
  return fmaf(w, fmaf(fmaf(a, kLog2eLow, fmaf(a, kLog2e, t)), -kLn2, kEx2Low), w);
}
__device__ __forceinline__ f32x2 exp_minus2(float a0, float a1) { return pack2(exp_minus(a0), exp_minus(a1)); }

// log(1 + e^v) = max(v, 0) + log(1 + w) with w = e^-|v| in (0, 1]: no overflow, and relative accuracy where it is small, since
// log(1 + w) = w P(w).  P: degree 10, fitted to log(1 + w) / w on [0, 1] by least squares with weights that even out the relative error;
// with these coefficients it is off by 1.8e-8, and by at most 1e-7 as evaluated.  (Degree 8 with a plain e^-|v| was off by
// up to 9e-7 at v = -12, in one direction on average, which doubled the error of the rates' gradient.)
#define BTP_LOG1P_COEFFICIENTS \
  {1.f, -0.499999821f, 0.333325595f, -0.249872714f, 0.198907465f, -0.161056876f, 0.124184281f, -0.0824416354f, 0.0414781272f, \
   -0.0134074828f, 0.00203023176f}
__device__ __forceinline__ float softplus(float v) {
  constexpr float kLog1p[11] = BTP_LOG1P_COEFFICIENTS;
  const float w = exp_minus(fabsf(v));
  float p = kLog1p[10];
#pragma unroll
  for (int i = 9; i >= 0; --i) p = fmaf(p, w, kLog1p[i]);
  return fmaf(p, w, fmaxf(v, 0.f));  // a NaN stays: w is NaN
}
__device__ __forceinline__ f32x2 softplus2(f32x2 v) {
  constexpr float kLog1p[11] = BTP_LOG1P_COEFFICIENTS;
  float a, b;
  unpack2(a, b, v);
  const f32x2 w = exp_minus2(fabsf(a), fabsf(b));
  f32x2 p = both(kLog1p[10]);
#pragma unroll
  for (int i = 9; i >= 0; --i) p = fma2(p, w, both(kLog1p[i]));
  return fma2(p, w, pack2(fmaxf(a, 0.f), fmaxf(b, 0.f)));
}
// Its slope 1 / (1 + e^-v), accurate where that is small.
__device__ __forceinline__ f32x2 softplus_slope2(f32x2 v) {
  const float a = lo2(v), b = hi2(v);
  const f32x2 w = exp_minus2(fabsf(a), fabsf(b)), q = add2(w, both(1.f));
  return mul2(pack2(a < 0.f ? lo2(w) : 1.f, b < 0.f ? hi2(w) : 1.f), pack2(rcp(lo2(q)), rcp(hi2(q))));
}
__device__ __forceinline__ f32x2 sigmoid2(f32x2 v) {
  const f32x2 e = add2(ex2_2(mul2(v, both(-kLog2e))), both(1.f));
  return pack2(rcp(lo2(e)), rcp(hi2(e)));
}

// Two neighbouring elements of an array whose element 0 is aligned to the pair, as floats, and back.
__device__ __forceinline__ f32x2 load_pair(const float* p) { return *reinterpret_cast<const f32x2*>(p); }
__device__ __forceinline__ f32x2 load_pair(const __nv_bfloat16* p) {
  const unsigned w = *reinterpret_cast<const unsigned*>(p);
  return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ f32x2 load_pair(const __half* p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
  return pack2(f.x, f.y);
}
__device__ __forceinline__ f32x2 word_pair(unsigned w, __nv_bfloat16) { return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ f32x2 word_pair(unsigned w, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pack2(f.x, f.y);
}
// Four consecutive elements, aligned to all of them, as pairs of floats.
__device__ __forceinline__ void load_quad(f32x2 (&out)[2], const float* p) {
  const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(p);
  out[0] = w.x, out[1] = w.y;
}
template <class T>
__device__ __forceinline__ void load_quad(f32x2 (&out)[2], const T* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  out[0] = word_pair(w.x, T{}), out[1] = word_pair(w.y, T{});
}

// 2 PAIRS consecutive elements as pairs; `aligned`: one word of all of them may be read, else element by element, `count` of them.
template <int PAIRS, class T>
__device__ __forceinline__ void load_channels(f32x2 (&out)[PAIRS], const T* p, bool aligned, int count) {
  if (aligned) {
    if constexpr (PAIRS == 2)
      load_quad(out, p);
    else
      out[0] = load_pair(p);
  } else {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) out[i] = pack2(2 * i < count ? to_f(p[2 * i]) : 0.f, 2 * i + 1 < count ? to_f(p[2 * i + 1]) : 0.f);
  }
}
template <int PAIRS, class T>
__device__ __forceinline__ void store_channels(T* p, const f32x2 (&in)[PAIRS], bool aligned, int count) {
  float f[2 * PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) unpack2(f[2 * i], f[2 * i + 1], in[i]);
  store_run<T, 2 * PAIRS>(p, f, aligned, count);
}
template <class T>
__device__ __forceinline__ void store_pair(T* p, f32x2 v, bool aligned, int count) {
  float f[2];
  unpack2(f[0], f[1], v);
  store_run<T, 2>(p, f, aligned, count);
}

// Asynchronous copies into shared memory.
__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy8(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ROWS rows of COLS elements (row pitch `pitch`, `cols` of them there) into dst[ROWS][COLS], by the threads of a group of
// GROUP threads.  Rows from `rows` on and columns from `cols` on are not touched.
template <class T, int ROWS, int COLS, int GROUP>
__device__ __forceinline__ void fetch(T (*dst)[COLS], const T* src, long long pitch, int rows, int cols, bool aligned, int tid) {
  constexpr int kBytes = COLS * static_cast<int>(sizeof(T)) < 16 ? 8 : 16, E = kBytes / static_cast<int>(sizeof(T)), CPR = COLS / E;
  static_assert(COLS % E == 0 && CPR >= 1, "a row is whole copies");
  if (aligned) {
#pragma unroll
    for (int i0 = 0; i0 < ROWS * CPR; i0 += GROUP) {
      const int i = i0 + tid, r = i / CPR, c = (i - r * CPR) * E;
      if ((ROWS * CPR % GROUP == 0 || i < ROWS * CPR) && r < rows && c < cols) {
        if (kBytes == 16)
          copy16(&dst[r][c], src + r * pitch + c);
        else
          copy8(&dst[r][c], src + r * pitch + c);
      }
    }
  } else {
#pragma unroll 4
    for (int i0 = 0; i0 < ROWS * COLS; i0 += GROUP) {
      const int i = i0 + tid, r = i / COLS, c = i - r * COLS;
      if (i < ROWS * COLS && r < rows && c < cols) {
        if (sizeof(T) == 4)
          copy4(&dst[r][c], src + r * pitch + c);
        else
          dst[r][c] = src[r * pitch + c];
      }
    }
  }
}

// Tokens of sequence b that are there: `lengths` may be null (all L), its values are held to 0 ... L.
__device__ __forceinline__ int tokens_of(const int* lengths, long long b, int L) {
  if (!lengths) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : (n < L ? n : L);
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

}  // namespace btp_elem
