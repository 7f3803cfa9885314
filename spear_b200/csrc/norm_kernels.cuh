// Root-mean-square norm with the residual's addition (sm_100a).
//
//   h = x + residual          r = 1 / sqrt(mean(h^2) + eps)          y = h r weight
//
// forward: one pass; a row stays in registers between the sum of its squares and its output (up to 8192 columns some instances spill
// 40 to 220 bytes of it, float or with a float residual; the backward of more than 8192 columns spills 850 to 920).  y leaves in x's type or as
// e4m3 with scale = max|y| / 448 over the row or over 128 columns (scale 1 where that is 0 or no number).  The norm
// is taken of the unrounded sum; h is rounded once, to the residual's type, as it is stored.
// backward: with xhat = h r and g = weight dy,  dh = r (g - xhat mean(g xhat)) + dh_out;  dweight = sum over rows of dy xhat,
// summed per thread over the rows of a persistent CTA, then over the CTAs by a second kernel in a fixed order.
//
// Both are bound by memory: forward moves x, residual, y, h once; backward h, dy, dh_out in and the gradients out.  A CTA takes rows in
// turn and fetches the next one, as it lies in memory, while it works on one.
// Measured with a cold L2 (copy rate of this device type: 6.57 TB/s): 16384 x 2048 bfloat16 with a float residual forward 67 us
// (6.0 TB/s), backward 93 us (5.8 TB/s); 16384 x 4096 in 8 bits with block scales 93 us (5.1 TB/s; 128 us with a CTA per row and nothing
// ahead).  That form is nearer to the issue rate than to memory (ncu: 68 % of the SM's throughput); it has one barrier per row, for the
// sum.  4096 rows of 16384 columns: forward 0.76 to 0.87 of the copy rate, in 8 bits 0.4 to 0.65; backward 210 to 310 us (0.3 to
// 0.65), for its spills.
// A group of `TPR` threads owns a row, thread i of it the runs of 8 columns i, i + TPR, ...: 16-byte accesses at 16 bits,
// and the 128 columns that share a scale always lie in 16 neighbouring lanes.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "btp_elem.cuh"

namespace btp_norm {

using namespace btp_elem;

constexpr int kRun = 8;        // consecutive columns per thread and step
constexpr int kBlockCols = 128;  // columns that share a scale in the blockwise 8-bit form
constexpr float kF8Max = 448.f;
constexpr int kMaxRowThreads = 512;
constexpr int kMaxDim = kMaxRowThreads * kRun * 4;

enum Out { kSame = 0, kRow8 = 1, kBlock8 = 2 };
enum Res { kNone = 0, kResSame = 1, kResF32 = 2 };

struct FwdParams {
  const void* x;
  const void* residual;
  const void* weight;  // nullptr: ones
  void* y;             // T or e4m3, dense rows
  void* h;             // residual's type, dense rows
  float* rstd;         // [rows] or nullptr
  float* scale;        // [rows] or [rows, ceil(dim / 128)]
  long long rows, ld_x, ld_r;
  int dim;
  float eps;
  bool weight_f32;
  bool al_x, al_r, al_w, al_out;  // every run of 8 that lies in the row is 16-byte accessible (8 for e4m3 output)
};

struct BwdParams {
  const void* h;       // residual's type (x's where there is none), row pitch ld_h
  const void* weight;
  const void* dy;      // T, dense rows
  const void* dh;      // residual's type, dense rows, or nullptr
  const float* rstd;
  void* dx;            // T, or nullptr
  void* dres;          // residual's type where that differs from T, else nullptr
  float* partial;      // [grid * rows per CTA][dim], or nullptr
  long long rows, ld_h;
  int dim;
  bool weight_f32;
  bool al_h, al_w, al_dense;
};

template <int TPR_WARP>
__device__ __forceinline__ float row_sum(float v, float* slot, int warp, int warps) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (TPR_WARP) return v;
  if ((threadIdx.x & 31) == 0) slot[warp] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < warps; ++i) v += slot[i];
  return v;
}
// Largest magnitude as its bit pattern: the order of the patterns is the order of the magnitudes, with NaN on top.
template <int TPR_WARP>
__device__ __forceinline__ unsigned row_max(unsigned v, unsigned* slot, int warp, int warps) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (TPR_WARP) return v;
  if ((threadIdx.x & 31) == 0) slot[warp] = v;
  __syncthreads();
  v = 0u;
  for (int i = 0; i < warps; ++i) v = max(v, slot[i]);
  return v;
}
// Scale of values whose largest magnitude has the bits `top`; 1 where that is 0 (or too small for a reciprocal) or NaN.
__device__ __forceinline__ float scale_of(unsigned top) {
  const float s = __uint_as_float(top) / kF8Max;
  return s > 1e-37f ? s : 1.f;
}

// A run of 8 columns as pairs; see load_run.
constexpr int kPairs = kRun / 2;
template <class T>
__device__ __forceinline__ void load_row(f32x2 (&v)[kPairs], const T* p, bool aligned, int left) {
  if (aligned && left >= kRun) {
    if constexpr (sizeof(T) == 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      v[0] = word_pair(w.x, T{}), v[1] = word_pair(w.y, T{}), v[2] = word_pair(w.z, T{}), v[3] = word_pair(w.w, T{});
    } else {
      const ulonglong2 a = reinterpret_cast<const ulonglong2*>(p)[0], b = reinterpret_cast<const ulonglong2*>(p)[1];
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
  } else {
    float f[kRun];
    load_run<T, kRun>(f, p, false, left);
#pragma unroll
    for (int k = 0; k < kPairs; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
  }
}
// The same run as it lies in memory: a row that is fetched while the one before is worked on costs half the registers that way.
template <class T>
struct RawRow {
  uint4 w[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ void load_raw(RawRow<T>& r, const T* p, bool aligned, int left) {
  if (aligned && left >= kRun) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    Pack<T, kRun> v;
#pragma unroll
    for (int k = 0; k < kRun; ++k) v.v[k] = k < left ? p[k] : from_f<T>(0.f);
    r = *reinterpret_cast<const RawRow<T>*>(&v);
  }
}
template <class T>
__device__ __forceinline__ void unpack_raw(f32x2 (&v)[kPairs], const RawRow<T>& r) {
  if constexpr (sizeof(T) == 2) {
    v[0] = word_pair(r.w[0].x, T{}), v[1] = word_pair(r.w[0].y, T{}), v[2] = word_pair(r.w[0].z, T{}), v[3] = word_pair(r.w[0].w, T{});
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[2 * i] = pack2(__uint_as_float(r.w[i].x), __uint_as_float(r.w[i].y));
      v[2 * i + 1] = pack2(__uint_as_float(r.w[i].z), __uint_as_float(r.w[i].w));
    }
  }
}
template <class T>
__device__ __forceinline__ void store_row(T* p, const f32x2 (&v)[kPairs], bool aligned, int left) {
  float f[kRun];
#pragma unroll
  for (int k = 0; k < kPairs; ++k) unpack2(f[2 * k], f[2 * k + 1], v[k]);
  store_run<T, kRun>(p, f, aligned && left >= kRun, left);
}
template <class T>
__device__ __forceinline__ void load_weight(f32x2 (&w)[kPairs], const void* base, int c, bool is_f32, bool aligned, int left) {
  if (!base) {
#pragma unroll
    for (int k = 0; k < kPairs; ++k) w[k] = both(1.f);
  } else if (is_f32) {
    load_row(w, static_cast<const float*>(base) + c, aligned, left);
  } else {
    load_row(w, static_cast<const T*>(base) + c, aligned, left);
  }
}

// CTAs of 512 threads that share an SM.  Two take 64 registers per thread; a row of four runs that is float or comes with a residual, and
// the one fetched ahead, need up to 128 and spilled up to 984 bytes: 4096 x 16384 bfloat16 with a float residual 237 us against 142,
// float 158 against 95, float with a residual 327 against 213; bfloat16 alone takes 52 with two and 56 with one.
template <class T, int RES, int VPT>
constexpr int kCtas = VPT == 4 && (RES != kNone || sizeof(T) == 4) ? 1 : 2;

// WARP_ROW: a row per warp (4 in a CTA of 128 threads); otherwise a row per CTA.
template <class T, int RES, int OUT, int VPT, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 128 : kMaxRowThreads, kCtas<T, RES, VPT>) rms_norm_forward_kernel(const FwdParams p) {
  using R = typename std::conditional<RES == kResF32, float, T>::type;
  __shared__ float s_sum[2][32];
  __shared__ unsigned s_max[2][32];
  const int tpr = WARP_ROW ? 32 : static_cast<int>(blockDim.x);
  const int tid = WARP_ROW ? (threadIdx.x & 31) : static_cast<int>(threadIdx.x);
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long first = WARP_ROW ? static_cast<long long>(blockIdx.x) * 4 + warp : static_cast<long long>(blockIdx.x);
  const long long step = WARP_ROW ? static_cast<long long>(gridDim.x) * 4 : static_cast<long long>(gridDim.x);
  grid_dependency_wait();
  RawRow<T> nx[VPT];
  RawRow<R> nr[VPT];
  const auto fetch_row = [&](long long row) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun;
      load_raw(nx[i], static_cast<const T*>(p.x) + row * p.ld_x + c, p.al_x, p.dim - c);
      if constexpr (RES != kNone) load_raw(nr[i], static_cast<const R*>(p.residual) + row * p.ld_r + c, p.al_r, p.dim - c);
    }
  };
  if (first < p.rows) fetch_row(first);
  int turn = 0;
  for (long long row = first; row < p.rows; row += step, turn ^= 1) {  // whole warps: nothing waits across warps when WARP_ROW
    f32x2 v[VPT][kPairs], rv[VPT][kPairs];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      unpack_raw(v[i], nx[i]);
      if constexpr (RES != kNone) unpack_raw(rv[i], nr[i]);
    }
    if (row + step < p.rows) fetch_row(row + step);
    f32x2 ss2 = 0ull;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        if (RES != kNone) v[i][k] = add2(v[i][k], rv[i][k]);
        ss2 = fma2(v[i][k], v[i][k], ss2);
      }
      if (RES != kNone) store_row(static_cast<R*>(p.h) + row * p.dim + c, v[i], p.al_out, p.dim - c);
    }
    const float ss = row_sum<WARP_ROW>(lo2(ss2) + hi2(ss2), s_sum[turn], warp, warps);
    const float rstd = rsqrtf(ss / static_cast<float>(p.dim) + p.eps);
    if (p.rstd && tid == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun;
      f32x2 w[kPairs];
      load_weight<T>(w, p.weight, c, p.weight_f32, p.al_w, p.dim - c);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) v[i][k] = mul2(mul2(v[i][k], both(rstd)), w[k]);
    }
    if constexpr (OUT == kSame) {
      T* y = static_cast<T*>(p.y) + row * p.dim;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = (tid + i * tpr) * kRun;
        store_row(y + c, v[i], p.al_out, p.dim - c);
      }
      continue;
    }
    unsigned top[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      top[i] = 0u;
      const int left = p.dim - (tid + i * tpr) * kRun;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {  // columns behind the row's end must not count: 0 * rstd may be NaN
        if (2 * k < left) top[i] = max(top[i], __float_as_uint(lo2(v[i][k])) & 0x7fffffffu);
        if (2 * k + 1 < left) top[i] = max(top[i], __float_as_uint(hi2(v[i][k])) & 0x7fffffffu);
      }
    }
    if (OUT == kRow8) {
      unsigned all = 0u;
#pragma unroll
      for (int i = 0; i < VPT; ++i) all = max(all, top[i]);
      all = row_max<WARP_ROW>(all, s_max[turn], warp, warps);
#pragma unroll
      for (int i = 0; i < VPT; ++i) top[i] = all;
      if (tid == 0) p.scale[row] = scale_of(all);
    } else {
      const int blocks = (p.dim + kBlockCols - 1) / kBlockCols;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
#pragma unroll
        for (int o = 8; o; o >>= 1) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
        const int blk = (tid + i * tpr) / (kBlockCols / kRun);
        if ((tid & 15) == 0 && blk < blocks) p.scale[row * blocks + blk] = scale_of(top[i]);
      }
    }
    unsigned char* q = static_cast<unsigned char*>(p.y) + row * p.dim;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun, left = p.dim - c;
      // y / scale as a product with the reciprocal and one step of Markstein's correction by the remainder: the product alone lands on the
      // other side of a rounding border now and then.  An infinite scale takes no correction (inf * 0).  Measured against true divisions: 90 us and 112.
      const float scale = scale_of(top[i]);
      const f32x2 inv = both(__frcp_rn(scale)), neg = both(isinf(scale) ? 0.f : -scale);
      union {
        __nv_fp8x2_storage_t h2[kPairs];
        uint2 w;
        unsigned char b[kRun];
      } o;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        float a, b;
        const f32x2 r = mul2(v[i][k], inv);
        unpack2(a, b, fma2(fma2(neg, r, v[i][k]), inv, r));
        o.h2[k] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
      }
      if (p.al_out && left >= kRun) {
        *reinterpret_cast<uint2*>(q + c) = o.w;
      } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k)
          if (k < left) q[c + k] = o.b[k];
      }
    }
  }
}

template <class T, int RES, int VPT, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 128 : kMaxRowThreads) rms_norm_backward_kernel(const BwdParams p) {
  using R = typename std::conditional<RES == kResF32, float, T>::type;
  __shared__ float s_sum[2][32];
  const int tpr = WARP_ROW ? 32 : static_cast<int>(blockDim.x);
  const int tid = WARP_ROW ? (threadIdx.x & 31) : static_cast<int>(threadIdx.x);
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long first = WARP_ROW ? static_cast<long long>(blockIdx.x) * 4 + warp : static_cast<long long>(blockIdx.x);
  const long long step = WARP_ROW ? static_cast<long long>(gridDim.x) * 4 : static_cast<long long>(gridDim.x);
  grid_dependency_wait();
  f32x2 w[VPT][kPairs], dw[VPT][kPairs];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * tpr) * kRun;
    load_weight<T>(w[i], p.weight, c, p.weight_f32, p.al_w, p.dim - c);
#pragma unroll
    for (int k = 0; k < kPairs; ++k) dw[i][k] = 0ull;
  }
  int turn = 0;
  for (long long row = first; row < p.rows; row += step, turn ^= 1) {
    const f32x2 r = both(p.rstd[row]);
    const R* h = static_cast<const R*>(p.h) + row * p.ld_h;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dim;
    f32x2 xh[VPT][kPairs], g[VPT][kPairs], e[VPT][kPairs], dot2 = 0ull;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun;
      load_row(xh[i], h + c, p.al_h, p.dim - c);
      load_row(g[i], dy + c, p.al_dense, p.dim - c);
      if (p.dh) load_row(e[i], static_cast<const R*>(p.dh) + row * p.dim + c, p.al_dense, p.dim - c);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        xh[i][k] = mul2(xh[i][k], r);
        dw[i][k] = fma2(g[i][k], xh[i][k], dw[i][k]);
        g[i][k] = mul2(g[i][k], w[i][k]);
        dot2 = fma2(g[i][k], xh[i][k], dot2);
      }
    const float dot = row_sum<WARP_ROW>(lo2(dot2) + hi2(dot2), s_sum[turn], warp, warps) / static_cast<float>(p.dim);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const f32x2 t = fma2(xh[i][k], both(-dot), g[i][k]);
        g[i][k] = p.dh ? fma2(r, t, e[i][k]) : mul2(r, t);
      }
      if (p.dx) store_row(static_cast<T*>(p.dx) + row * p.dim + c, g[i], p.al_dense, p.dim - c);
      if (p.dres) store_row(static_cast<R*>(p.dres) + row * p.dim + c, g[i], p.al_dense, p.dim - c);
    }
  }
  if (p.partial) {
    float* to = p.partial + first * p.dim;  // every row of the buffer is written, also by groups that had no row
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun;
      store_row(to + c, dw[i], p.al_dense, p.dim - c);
    }
  }
}

}  // namespace btp_norm
