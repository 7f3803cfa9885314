// Short causal convolution over tokens, one filter of W taps per channel, token-major (sm_100a).
//
//   pre[b,t,d] = bias[d] + sum_w weight[d,w] xx[b, t - (W-1) + w, d]        y = pre, or pre * sigmoid(pre)
//
// xx is x with the W-1 inputs of the initial state (or zeros) in front.  Tokens from lengths[b] on are not read; y and dx are 0
// there.  The state that is handed on is the last W-1 entries of xx before lengths[b].
// backward: e = dy * act'(pre), recomputed from x;  dx[t] = sum_w weight[w] e[t + (W-1) - w];  dweight[w] = sum e[t] xx[t-(W-1)+w].
//
// Bound by memory: x in and y out once (backward: x, dy, dx).  A thread walks down `run` tokens of a few neighbouring channels
// and keeps the window in registers, so x is read once but for W-1 tokens per run, which its neighbour has just read.
// The weight's gradient is summed per thread, over the 8 runs of a CTA in shared memory, and over CTAs by a second kernel in a
// fixed order: the same call gives the same bits.
#pragma once

#include "btp_elem.cuh"

namespace btp_conv {

using namespace btp_elem;

struct ConvParams {
  const void* x;
  const void* weight;   // [dim, W]
  const void* bias;     // [dim] or nullptr
  const void* initial;  // [B, W-1, dim] or nullptr (zeros)
  const int* lengths;   // [B] or nullptr
  void* y;              // [B, L, dim]
  void* state;          // [B, W-1, dim] or nullptr
  const void* dy;       // backward: [B, L, dim]
  const void* dstate;   // [B, W-1, dim] or nullptr
  void* dx;             // [B, L, dim]
  void* dinitial;       // [B, W-1, dim] or nullptr
  float* partial;       // [parts, W+1, dim]
  long long sx_b, sx_t;
  int B, L, dim, run, runs;
  bool silu, weight_f32;
};

constexpr int kRunsPerCta = 8;

// One vector of V channels of row `t` of xx (t may be negative: the initial state).
template <class T, int V, int W>
__device__ __forceinline__ void load_xx(float (&out)[V], const ConvParams& p, const T* x, long long b, int t, int d) {
  if (t >= 0) {
    load_run<T, V>(out, x + t * p.sx_t, true, V);
  } else if (p.initial) {
    load_run<T, V>(out, static_cast<const T*>(p.initial) + (b * (W - 1) + t + (W - 1)) * p.dim + d, true, V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.f;
  }
}

template <class T, int V, int W>
__device__ __forceinline__ void load_filter(float (&w)[W][V], float (&bias)[V], const ConvParams& p, int d) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float tap[W];
    load_param<T, W>(tap, p.weight, static_cast<long long>(d + i) * W, p.weight_f32, false, W);
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][i] = tap[k];
  }
  if (p.bias) {
    load_param<T, V>(bias, p.bias, d, p.weight_f32, false, V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = 0.f;
  }
}

// V channels per thread: one 16-byte word where every row allows it, else 1.
template <class T, int V, int W>
__global__ void __launch_bounds__(256) conv_forward_kernel(const ConvParams p) {
  grid_dependency_wait();
  const int dv = p.dim / V;
  const long long idx = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long rest = idx / dv;
  const int d = static_cast<int>(idx - rest * dv) * V;
  const long long b = rest / p.runs;
  if (b >= p.B) return;
  const int r = static_cast<int>(rest - b * p.runs);
  const int n = tokens_of(p.lengths, b, p.L);
  const T* x = static_cast<const T*>(p.x) + b * p.sx_b + d;
  T* y = static_cast<T*>(p.y) + b * p.L * p.dim + d;
  const int t0 = r * p.run, t1 = min(p.L, t0 + p.run), live = min(n, t1);
  if (t0 < live) {
    float w[W][V], bias[V], win[W][V];
    load_filter<T, V, W>(w, bias, p, d);
#pragma unroll
    for (int k = 1; k < W; ++k) load_xx<T, V, W>(win[k], p, x, b, t0 - W + k, d);
    constexpr int U = 4;
    for (int t = t0; t < live; t += U) {
      float in[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t + u < live) load_run<T, V>(in[u], x + (t + u) * p.sx_t, true, V);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t + u >= live) break;
        float out[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
          for (int k = 0; k + 1 < W; ++k) win[k][i] = win[k + 1][i];
          win[W - 1][i] = in[u][i];
          float a = bias[i];
#pragma unroll
          for (int k = 0; k < W; ++k) a = fmaf(w[k][i], win[k][i], a);
          out[i] = p.silu ? a * sigmoid(a) : a;
        }
        store_run<T, V>(y + static_cast<long long>(t + u) * p.dim, out, true, V);
      }
    }
  }
  const float zero[V] = {};
  for (int t = max(t0, live); t < t1; ++t) store_run<T, V>(y + static_cast<long long>(t) * p.dim, zero, true, V);
  if (p.state && r == p.runs - 1) {
    T* s = static_cast<T*>(p.state) + b * (W - 1) * p.dim + d;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      float v[V];
      load_xx<T, V, W>(v, p, x, b, n - (W - 1) + k, d);
      store_run<T, V>(s + static_cast<long long>(k) * p.dim, v, true, V);
    }
  }
}

// CTA: 32 lanes of V channels x 8 runs.  grid: (channel blocks) x (groups of 8 runs) x B, flattened.
template <class T, int V, int W>
__global__ void __launch_bounds__(256) conv_backward_kernel(const ConvParams p) {
  __shared__ float red[kRunsPerCta][W + 1][32 * V];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cb = (p.dim + 32 * V - 1) / (32 * V), groups = (p.runs + kRunsPerCta - 1) / kRunsPerCta;
  const int c = blockIdx.x % cb;
  const long long part = blockIdx.x / cb, b = part / groups;
  const int r = static_cast<int>(part - b * groups) * kRunsPerCta + warp;
  const int d = (c * 32 + lane) * V;
  float dw[W][V] = {}, db[V] = {};
  if (d < p.dim && r < p.runs) {  // dim is a multiple of V
    const int n = tokens_of(p.lengths, b, p.L);
    const T* x = static_cast<const T*>(p.x) + b * p.sx_b + d;
    const T* dy = static_cast<const T*>(p.dy) + b * p.L * p.dim + d;
    T* dx = static_cast<T*>(p.dx) + b * p.L * p.dim + d;
    const T* ds = p.dstate ? static_cast<const T*>(p.dstate) + b * (W - 1) * p.dim + d : nullptr;
    T* di = p.dinitial && r == 0 ? static_cast<T*>(p.dinitial) + b * (W - 1) * p.dim + d : nullptr;
    const int t0 = r * p.run, t1 = min(p.L, t0 + p.run);
    float w[W][V], bias[V], win[W][V], e[W][V];
    load_filter<T, V, W>(w, bias, p, d);
#pragma unroll
    for (int k = 0; k < W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) e[k][i] = 0.f;
#pragma unroll
    for (int k = 1; k < W; ++k) load_xx<T, V, W>(win[k], p, x, b, t0 - W + k, d);
    const int last = t1 + W - 1;
    constexpr int U = 4;
    for (int t = t0; t < last; t += U) {
      float in[U][V], up[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t + u < last && t + u < n) {
          load_run<T, V>(in[u], x + (t + u) * p.sx_t, true, V);
          load_run<T, V>(up[u], dy + static_cast<long long>(t + u) * p.dim, true, V);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int tt = t + u;
        if (tt >= last) break;
        const bool live = tt < n;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
          for (int k = 0; k + 1 < W; ++k) win[k][i] = win[k + 1][i];
#pragma unroll
          for (int k = W - 1; k > 0; --k) e[k][i] = e[k - 1][i];  // e[k] = e at tt - k
          e[0][i] = 0.f;
          if (live) {
            win[W - 1][i] = in[u][i];
            float g = up[u][i];
            if (p.silu) {
              float a = bias[i];
#pragma unroll
              for (int k = 0; k < W; ++k) a = fmaf(w[k][i], win[k][i], a);
              const float s = sigmoid(a);
              g *= s * fmaf(a, 1.f - s, 1.f);
            }
            e[0][i] = g;
            if (tt < t1) {
              db[i] += g;
#pragma unroll
              for (int k = 0; k < W; ++k) dw[k][i] = fmaf(g, win[k][i], dw[k][i]);
            }
          }
        }
        const int at = tt - (W - 1);  // its gradient is complete now
        if (at < t0 && !(di && at < 0)) continue;
        float out[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          out[i] = 0.f;
          if (at < n) {
#pragma unroll
            for (int k = 0; k < W; ++k) out[i] = fmaf(w[k][i], e[k][i], out[i]);
          }
        }
        if (ds && at < n && at >= n - (W - 1)) {
          float s[V];
          load_run<T, V>(s, ds + static_cast<long long>(at - n + (W - 1)) * p.dim, true, V);
#pragma unroll
          for (int i = 0; i < V; ++i) out[i] += s[i];
        }
        if (at >= 0)
          store_run<T, V>(dx + static_cast<long long>(at) * p.dim, out, true, V);
        else
          store_run<T, V>(di + static_cast<long long>(at + (W - 1)) * p.dim, out, true, V);
      }
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < W; ++k) red[warp][k][lane * V + i] = dw[k][i];
    red[warp][W][lane * V + i] = db[i];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < (W + 1) * 32 * V; j += 256) {
    const int k = j / (32 * V), col = j - k * (32 * V), dd = c * 32 * V + col;
    if (dd >= p.dim) continue;
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < kRunsPerCta; ++i) a += red[i][k][col];
    p.partial[(part * (W + 1) + k) * p.dim + dd] = a;
  }
}

// dweight[d, k], dbias[d] from partial[parts][W+1][dim].  CTA: 32 columns x 8 strands.
template <class T>
__global__ void __launch_bounds__(256) conv_weight_sum_kernel(const float* part, void* dweight, void* dbias, long long parts, int dim,
                                                              int width, bool out_f32) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const long long cols = static_cast<long long>(width + 1) * dim;
  const long long j = static_cast<long long>(blockIdx.x) * 32 + lane;
  grid_dependency_wait();
  float a = 0.f;
  if (j < cols)
#pragma unroll 4
    for (long long i = strand; i < parts; i += 8) a += part[i * cols + j];
  s[strand][lane] = a;
  __syncthreads();
  if (strand || j >= cols) return;
  a = s[0][lane];
#pragma unroll
  for (int i = 1; i < 8; ++i) a += s[i][lane];
  const int k = static_cast<int>(j / dim), d = static_cast<int>(j - static_cast<long long>(k) * dim);
  void* to = k < width ? dweight : dbias;
  if (!to) return;
  const long long at = k < width ? static_cast<long long>(d) * width + k : d;
  if (out_f32)
    static_cast<float*>(to)[at] = a;
  else
    static_cast<T*>(to)[at] = from_f<T>(a);
}

struct ConvStepParams {
  const void* x;      // [B, dim], row pitch ld_x
  const void* state;  // [B, W-1, dim]
  const void* weight;
  const void* bias;
  void* y;            // [B, dim]
  void* state_out;    // [B, W-1, dim]; may be `state`
  long long ld_x;
  int B, dim;
  bool silu, weight_f32;
};

// A thread reads all it needs of its channels' state before it writes any, so the update may be in place.
template <class T, int V, int W>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvStepParams p) {
  grid_dependency_wait();
  const int dv = p.dim / V;
  const long long idx = static_cast<long long>(blockIdx.x) * 128 + threadIdx.x;
  const long long b = idx / dv;
  if (b >= p.B) return;
  const int d = static_cast<int>(idx - b * dv) * V;
  float win[W][V], w[W][V], bias[V], out[V];
  const T* s = static_cast<const T*>(p.state) + b * (W - 1) * p.dim + d;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) load_run<T, V>(win[k], s + static_cast<long long>(k) * p.dim, true, V);
  load_run<T, V>(win[W - 1], static_cast<const T*>(p.x) + b * p.ld_x + d, true, V);
  ConvParams f{};
  f.weight = p.weight; f.bias = p.bias; f.weight_f32 = p.weight_f32;
  load_filter<T, V, W>(w, bias, f, d);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float a = bias[i];
#pragma unroll
    for (int k = 0; k < W; ++k) a = fmaf(w[k][i], win[k][i], a);
    out[i] = p.silu ? a * sigmoid(a) : a;
  }
  store_run<T, V>(static_cast<T*>(p.y) + b * p.dim + d, out, true, V);
  T* so = static_cast<T*>(p.state_out) + b * (W - 1) * p.dim + d;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) store_run<T, V>(so + static_cast<long long>(k) * p.dim, win[k + 1], true, V);
}

}  // namespace btp_conv
