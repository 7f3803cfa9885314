// Root-mean-square norm with the residual's addition (sm_100a).
//
//   h = x + residual          r = 1 / sqrt(mean(h^2) + eps)          y = h r weight
//
// forward: one pass; a row stays in registers between the sum of its squares and its output.  y leaves in x's type or as
// e4m3 with scale = max|y| / 448 over the row or over 128 columns (scale 1 where that is 0 or no number).  The norm
// is taken of the unrounded sum; h is rounded once, to the residual's type, as it is stored.
// backward: with xhat = h r and g = weight dy,  dh = r (g - xhat mean(g xhat)) + dh_out;  dweight = sum over rows of dy xhat,
// summed per thread over the rows of a persistent CTA, then over the CTAs by a second kernel in a fixed order.
//
// Both are bound by memory: forward moves x, residual, y, h once; backward h, dy, dh_out in and the gradients out.
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
__device__ __forceinline__ float scale_of(unsigned top) {
  const float s = __uint_as_float(top) / kF8Max;
  return s > 0.f ? s : 1.f;
}

// WARP_ROW: a row per warp (4 in a CTA of 128 threads); otherwise a row per CTA.
template <class T, int RES, int OUT, int VPT, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 128 : kMaxRowThreads) rms_norm_forward_kernel(const FwdParams p) {
  using R = typename std::conditional<RES == kResF32, float, T>::type;
  __shared__ float s_sum[32];
  __shared__ unsigned s_max[32];
  const int tpr = WARP_ROW ? 32 : static_cast<int>(blockDim.x);
  const int tid = WARP_ROW ? (threadIdx.x & 31) : static_cast<int>(threadIdx.x);
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long row = WARP_ROW ? static_cast<long long>(blockIdx.x) * 4 + warp : static_cast<long long>(blockIdx.x);
  grid_dependency_wait();
  if (row >= p.rows) return;  // whole warps: nothing below waits across warps when WARP_ROW
  float v[VPT][kRun];
  const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * tpr) * kRun, left = p.dim - c;
    load_run<T, kRun>(v[i], x + c, p.al_x && left >= kRun, left);
  }
  if (RES != kNone) {
    const R* r = static_cast<const R*>(p.residual) + row * p.ld_r;
    R* h = static_cast<R*>(p.h) + row * p.dim;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun, left = p.dim - c;
      float rv[kRun];
      load_run<R, kRun>(rv, r + c, p.al_r && left >= kRun, left);
#pragma unroll
      for (int k = 0; k < kRun; ++k) v[i][k] += rv[k];
      store_run<R, kRun>(h + c, v[i], p.al_out && left >= kRun, left);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int k = 0; k < kRun; ++k) ss = fmaf(v[i][k], v[i][k], ss);
  ss = row_sum<WARP_ROW>(ss, s_sum, warp, warps);
  const float rstd = rsqrtf(ss / static_cast<float>(p.dim) + p.eps);
  if (p.rstd && tid == 0) p.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * tpr) * kRun, left = p.dim - c;
    float w[kRun];
    if (p.weight) load_param<T, kRun>(w, p.weight, c, p.weight_f32, p.al_w && left >= kRun, left);
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      v[i][k] *= rstd;
      if (p.weight) v[i][k] *= w[k];
    }
  }
  if (OUT == kSame) {
    T* y = static_cast<T*>(p.y) + row * p.dim;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun, left = p.dim - c;
      store_run<T, kRun>(y + c, v[i], p.al_out && left >= kRun, left);
    }
    return;
  }
  unsigned top[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    top[i] = 0u;
    const int left = p.dim - (tid + i * tpr) * kRun;
#pragma unroll
    for (int k = 0; k < kRun; ++k)  // columns behind the row's end must not count: 0 * rstd may be NaN
      if (k < left) top[i] = max(top[i], __float_as_uint(v[i][k]) & 0x7fffffffu);
  }
  if (OUT == kRow8) {
    unsigned all = 0u;
#pragma unroll
    for (int i = 0; i < VPT; ++i) all = max(all, top[i]);
    all = row_max<WARP_ROW>(all, s_max, warp, warps);
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
  __nv_fp8_e4m3* q = static_cast<__nv_fp8_e4m3*>(p.y) + row * p.dim;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * tpr) * kRun, left = p.dim - c;
    const float s = scale_of(top[i]);
    union {
      __nv_fp8x2_storage_t h2[kRun / 2];
      uint2 w;
      unsigned char b[kRun];
    } o;
#pragma unroll
    for (int k = 0; k < kRun; k += 2)  // a true quotient: the rounding border is that of the definition
      o.h2[k / 2] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(v[i][k], s), __fdiv_rn(v[i][k + 1], s)), __NV_SATFINITE, __NV_E4M3);
    if (p.al_out && left >= kRun) {
      *reinterpret_cast<uint2*>(q + c) = o.w;
    } else {
#pragma unroll
      for (int k = 0; k < kRun; ++k)
        if (k < left) reinterpret_cast<unsigned char*>(q)[c + k] = o.b[k];
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
  float w[VPT][kRun], dw[VPT][kRun];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (tid + i * tpr) * kRun, left = p.dim - c;
    if (p.weight) load_param<T, kRun>(w[i], p.weight, c, p.weight_f32, p.al_w && left >= kRun, left);
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      if (!p.weight) w[i][k] = 1.f;
      dw[i][k] = 0.f;
    }
  }
  int turn = 0;
  for (long long row = first; row < p.rows; row += step, turn ^= 1) {
    const float r = p.rstd[row];
    const R* h = static_cast<const R*>(p.h) + row * p.ld_h;
    const T* dy = static_cast<const T*>(p.dy) + row * p.dim;
    float xh[VPT][kRun], g[VPT][kRun], dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun, left = p.dim - c;
      load_run<R, kRun>(xh[i], h + c, p.al_h && left >= kRun, left);
      load_run<T, kRun>(g[i], dy + c, p.al_dense && left >= kRun, left);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        xh[i][k] *= r;
        dw[i][k] = fmaf(g[i][k], xh[i][k], dw[i][k]);
        g[i][k] *= w[i][k];
        dot = fmaf(g[i][k], xh[i][k], dot);
      }
    dot = row_sum<WARP_ROW>(dot, s_sum[turn], warp, warps) / static_cast<float>(p.dim);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun, left = p.dim - c;
      float out[kRun];
#pragma unroll
      for (int k = 0; k < kRun; ++k) out[k] = r * (g[i][k] - xh[i][k] * dot);
      if (p.dh) {
        float e[kRun];
        load_run<R, kRun>(e, static_cast<const R*>(p.dh) + row * p.dim + c, p.al_dense && left >= kRun, left);
#pragma unroll
        for (int k = 0; k < kRun; ++k) out[k] += e[k];
      }
      if (p.dx) store_run<T, kRun>(static_cast<T*>(p.dx) + row * p.dim + c, out, p.al_dense && left >= kRun, left);
      if (p.dres) store_run<R, kRun>(static_cast<R*>(p.dres) + row * p.dim + c, out, p.al_dense && left >= kRun, left);
    }
  }
  if (p.partial) {
    float* to = p.partial + first * p.dim;  // every row of the buffer is written, also by groups that had no row
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (tid + i * tpr) * kRun, left = p.dim - c;
      store_run<float, kRun>(to + c, dw[i], p.al_dense && left >= kRun, left);
    }
  }
}

}  // namespace btp_norm
