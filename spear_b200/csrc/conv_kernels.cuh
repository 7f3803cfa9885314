// Short causal convolution over tokens, one filter of W taps per channel, token-major (sm_100a).
//
//   pre[b,t,d] = bias[d] + sum_w weight[d,w] xx[b, t - (W-1) + w, d]        y = pre, or pre * sigmoid(pre)
//
// xx is x with the W-1 inputs of the initial state (or zeros) in front.  Tokens from lengths[b] on are not read; y and dx are 0
// there.  The state that is handed on is the last W-1 entries of xx before lengths[b].
// backward: e = dy * act'(pre), recomputed from x;  dx[t] = sum_w weight[w] e[t + (W-1) - w];  dweight[w] = sum e[t] xx[t-(W-1)+w].
//
// Bound by memory: x in and y out once (backward: x, dy, dx).  A CTA walks down the tokens of 128 channels with a ring of tiles that
// asynchronous copies fill two ahead (32 tokens: enough bytes in flight, which registers cannot hold); a thread keeps the
// window of its channel pair in registers, so x is read once but for W-1 tokens per run.
// The weight's gradient is summed per thread over its run, then over the runs by a second kernel in a fixed order: the same call
// gives the same bits.
// Measured at 8 x 2048 tokens x 2048 channels, bfloat16, W = 4, silu: forward 32 us (4.2 TB/s), backward 57 us (3.5 TB/s), which is not
// the memory's limit: a lane moves one channel pair, 4 bytes, per load and store, and ncu shows no unit above half of its rate (a warp waits
// 11 and 7 cycles per instruction, 24 and 13 warps per SM).  One thread per channel run with its loads in registers took 89 and 228 us.  Tiles of 8 tokens, rings of 4 or 6, 128 threads: within 10 %, none better.
#pragma once

#include <type_traits>

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
  bool copies, copies_dy;  // rows of x and dy allow 16-byte copies
  bool aligned;  // a thread's channels are one word in every row
  bool whole_w;  // and so are their taps
};

constexpr int kThreads = 64;               // of a CTA: two channels each
constexpr int kCols = 2 * kThreads;        // channels of a CTA
constexpr int kTile = 16;                  // tokens per tile
constexpr int kStages = 3;                 // tiles in the ring

// 2 PAIRS channels of row `t` of xx (t may be negative: the initial state).
template <class T, int PAIRS, int W>
__device__ __forceinline__ void load_xx(f32x2 (&out)[PAIRS], const ConvParams& p, const T* x, long long b, int t, int d) {
  if (t >= 0) {
    load_channels<PAIRS>(out, x + t * p.sx_t, p.aligned, p.dim - d);
  } else if (p.initial) {
    load_channels<PAIRS>(out, static_cast<const T*>(p.initial) + (b * (W - 1) + t + (W - 1)) * p.dim + d, p.aligned, p.dim - d);
  } else {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) out[i] = 0ull;
  }
}

// Taps and bias of 2 PAIRS channels; the taps of neighbouring channels are contiguous and read as whole words.
template <class T, int PAIRS, int W>
__device__ __forceinline__ void load_filter(f32x2 (&w)[W][PAIRS], f32x2 (&bias)[PAIRS], const void* weight, const void* bias_at, bool f32, bool whole,
                                            int d, int dim) {
  constexpr int V = 2 * PAIRS;
  float tap[V * W], c[V] = {};
  const int count = min(V, dim - d);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    float part[V];
    load_param<T, V>(part, weight, static_cast<long long>(d) * W + i * V, f32, whole && count == V, count * W - i * V);
#pragma unroll
    for (int k = 0; k < V; ++k) tap[i * V + k] = part[k];
  }
  if (bias_at) load_param<T, V>(c, bias_at, d, f32, false, count);
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][i] = pack2(tap[2 * i * W + k], tap[(2 * i + 1) * W + k]);
    bias[i] = pack2(c[2 * i], c[2 * i + 1]);
  }
}

template <class T, int TENSORS>
struct ConvTile {
  T v[kStages][TENSORS][kTile][kCols];
};

// CTA: 128 channels x `run` tokens of one sequence; grid: channel blocks x runs x B, flattened.
template <class T, int W>
__global__ void __launch_bounds__(kThreads) conv_forward_kernel(const ConvParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<ConvTile<T, 1>*>(smem_raw);
  grid_dependency_wait();
  const int tid = threadIdx.x, cblocks = (p.dim + kCols - 1) / kCols;
  const int cw = static_cast<int>(blockIdx.x % cblocks) * kCols, d = cw + 2 * tid, left = p.dim - d, cols = min(kCols, p.dim - cw);
  const int rest = blockIdx.x / cblocks, r = rest % p.runs;
  const long long b = rest / p.runs;
  const int n = tokens_of(p.lengths, b, p.L);
  const T* x = static_cast<const T*>(p.x) + b * p.sx_b + cw;
  T* y = static_cast<T*>(p.y) + b * p.L * p.dim + d;
  const int t0 = r * p.run, t1 = min(p.L, t0 + p.run), live = min(n, t1);
  const int tiles = live > t0 ? (live - t0 + kTile - 1) / kTile : 0;
  const auto load = [&](int i) {
    const int t = t0 + i * kTile;
    if (i < tiles) fetch<T, kTile, kCols, kThreads>(sm.v[i % kStages][0], x + t * p.sx_t, p.sx_t, min(kTile, live - t), cols, p.copies, tid);
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i);
  if (tiles) {
    f32x2 w[W][1], bias[1], win[W];
    load_filter<T, 1, W>(w, bias, p.weight, p.bias, p.weight_f32, p.whole_w, d, p.dim);
#pragma unroll
    for (int k = 1; k < W; ++k) {
      f32x2 v[1] = {0ull};
      if (left > 0) load_xx<T, 1, W>(v, p, x + 2 * tid, b, t0 - W + k, d);
      win[k] = v[0];
    }
    win[0] = 0ull;
    // one walk with silu and one without: the test stays out of the token loop
    const auto walk = [&](auto act) {
      for (int i = 0; i < tiles; ++i) {
        copy_wait<kStages - 2>();
        __syncthreads();  // the tile has arrived everywhere, and the one before is read to the end: its place is free
        load(i + kStages - 1);
        const int t = t0 + i * kTile, nt = min(kTile, live - t);
        if (left <= 0) continue;
        const T* row = &sm.v[i % kStages][0][0][2 * tid];
        T* to = y + static_cast<long long>(t) * p.dim;
        const auto token = [&](int j) {
#pragma unroll
          for (int k = 0; k + 1 < W; ++k) win[k] = win[k + 1];
          win[W - 1] = load_pair(row + j * kCols);
          f32x2 out[1] = {bias[0]};
#pragma unroll
          for (int k = 0; k < W; ++k) out[0] = fma2(w[k][0], win[k], out[0]);
          if constexpr (decltype(act)::value) out[0] = mul2(out[0], sigmoid2(out[0]));
          store_channels<1>(to + static_cast<long long>(j) * p.dim, out, p.aligned, left);
        };
        if (nt == kTile) {
#pragma unroll
          for (int j = 0; j < kTile; ++j) token(j);
        } else {
          for (int j = 0; j < nt; ++j) token(j);
        }
      }
    };
    if (p.silu)
      walk(std::true_type{});
    else
      walk(std::false_type{});
  }
  copy_wait<0>();
  if (left <= 0) return;
  const f32x2 zero[1] = {};
  for (int t = max(t0, live); t < t1; ++t) store_channels<1>(y + static_cast<long long>(t) * p.dim, zero, p.aligned, left);
  if (p.state && r == p.runs - 1) {
    T* s = static_cast<T*>(p.state) + b * (W - 1) * p.dim + d;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      f32x2 v[1];
      load_xx<T, 1, W>(v, p, x + 2 * tid, b, n - (W - 1) + k, d);
      store_channels<1>(s + static_cast<long long>(k) * p.dim, v, p.aligned, left);
    }
  }
}

// The same walk over x and dy, W - 1 tokens further than the run: the gradient of a token takes the e of the W - 1 behind it.
template <class T, int W>
__global__ void __launch_bounds__(kThreads) conv_backward_kernel(const ConvParams p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  auto& sm = *reinterpret_cast<ConvTile<T, 2>*>(smem_raw);
  grid_dependency_wait();
  const int tid = threadIdx.x, cblocks = (p.dim + kCols - 1) / kCols;
  const int cw = static_cast<int>(blockIdx.x % cblocks) * kCols, d = cw + 2 * tid, left = p.dim - d, cols = min(kCols, p.dim - cw);
  const int part = blockIdx.x / cblocks, r = part % p.runs;
  const long long b = part / p.runs;
  const int n = tokens_of(p.lengths, b, p.L);
  const T* x = static_cast<const T*>(p.x) + b * p.sx_b + cw;
  const T* dy = static_cast<const T*>(p.dy) + b * p.L * p.dim + cw;
  T* dx = static_cast<T*>(p.dx) + b * p.L * p.dim + d;
  const T* ds = p.dstate ? static_cast<const T*>(p.dstate) + b * (W - 1) * p.dim + d : nullptr;
  T* di = p.dinitial && r == 0 ? static_cast<T*>(p.dinitial) + b * (W - 1) * p.dim + d : nullptr;
  const int t0 = r * p.run, t1 = min(p.L, t0 + p.run), last = t1 + W - 1, live = min(n, last);
  const int tiles = (last - t0 + kTile - 1) / kTile;  // rows from `live` on are not copied and count as zeros
  const auto load = [&](int i) {
    const int t = t0 + i * kTile;
    if (i < tiles && t < live) {
      const int rows = min(kTile, live - t);
      fetch<T, kTile, kCols, kThreads>(sm.v[i % kStages][0], x + t * p.sx_t, p.sx_t, rows, cols, p.copies, tid);
      fetch<T, kTile, kCols, kThreads>(sm.v[i % kStages][1], dy + static_cast<long long>(t) * p.dim, p.dim, rows, cols, p.copies_dy, tid);
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load(i);
  f32x2 w[W][1], bias[1], win[W], e[W] = {}, dw[W] = {}, db = 0ull;
  load_filter<T, 1, W>(w, bias, p.weight, p.bias, p.weight_f32, p.whole_w, d, p.dim);
#pragma unroll
  for (int k = 1; k < W; ++k) {
    f32x2 v[1] = {0ull};
    if (left > 0 && t0 - W + k < n) load_xx<T, 1, W>(v, p, x + 2 * tid, b, t0 - W + k, d);
    win[k] = v[0];
  }
  win[0] = 0ull;
  const auto walk = [&](auto act) {
    for (int i = 0; i < tiles; ++i) {
      copy_wait<kStages - 2>();
      __syncthreads();
      load(i + kStages - 1);
      if (left <= 0) continue;
      const int t = t0 + i * kTile;
      const T* rx = &sm.v[i % kStages][0][0][2 * tid];
      const T* ry = &sm.v[i % kStages][1][0][2 * tid];
      // e of token t + j, and the gradient of the token W - 1 before it, which is complete then
      const auto token = [&](int j, auto inner) {
        constexpr bool kInner = decltype(inner)::value;  // all of the tile's tokens are there, as are their predecessors in the run
        const int tt = t + j, at = tt - (W - 1);
#pragma unroll
        for (int k = 0; k + 1 < W; ++k) win[k] = win[k + 1];
#pragma unroll
        for (int k = W - 1; k > 0; --k) e[k] = e[k - 1];  // e[k] = e at tt - k
        const bool there = kInner || tt < n;
        win[W - 1] = there ? load_pair(rx + j * kCols) : 0ull;
        f32x2 g = there ? load_pair(ry + j * kCols) : 0ull;
        if constexpr (decltype(act)::value) {
          f32x2 a = bias[0];
#pragma unroll
          for (int k = 0; k < W; ++k) a = fma2(w[k][0], win[k], a);
          const f32x2 s = sigmoid2(a);
          g = mul2(g, mul2(s, fma2(a, fma2(s, both(-1.f), both(1.f)), both(1.f))));
          if (!there) g = 0ull;
        }
        e[0] = g;
        if (kInner || tt < t1) {
          db = add2(db, g);
#pragma unroll
          for (int k = 0; k < W; ++k) dw[k] = fma2(g, win[k], dw[k]);
        }
        if (!kInner && at < t0 && !(di && at < 0)) return;
        f32x2 out[1] = {0ull};
        if (kInner || at < n) {
#pragma unroll
          for (int k = 0; k < W; ++k) out[0] = fma2(w[k][0], e[k], out[0]);
          if (!kInner && ds && at >= n - (W - 1)) {
            f32x2 s[1];
            load_channels<1>(s, ds + static_cast<long long>(at - n + (W - 1)) * p.dim, p.aligned, left);
            out[0] = add2(out[0], s[0]);
          }
        }
        store_channels<1>(kInner || at >= 0 ? dx + static_cast<long long>(at) * p.dim : di + static_cast<long long>(at + (W - 1)) * p.dim, out, p.aligned, left);
      };
      if (i && t + kTile <= min(t1, n)) {  // (a token that the final state's gradient reaches is complete behind token n only)
#pragma unroll
        for (int j = 0; j < kTile; ++j) token(j, std::true_type{});
      } else {
        for (int j = 0; j < min(kTile, last - t); ++j) token(j, std::false_type{});
      }
    }
  };
  if (p.silu)
    walk(std::true_type{});
  else
    walk(std::false_type{});
  copy_wait<0>();
  if (!p.partial || left <= 0) return;
#pragma unroll
  for (int k = 0; k <= W; ++k) {
    const f32x2 v[1] = {k < W ? dw[k < W ? k : 0] : db};
    store_channels<1>(p.partial + (static_cast<long long>(part) * (W + 1) + k) * p.dim + d, v, p.dim % 2 == 0, left);
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
  bool silu, weight_f32, aligned, whole_w;
};

// A thread reads all it needs of its channels' state before it writes any, so the update may be in place.
template <class T, int W>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvStepParams p) {
  constexpr int P = 2;
  grid_dependency_wait();
  const int dv = (p.dim + 2 * P - 1) / (2 * P);
  const long long idx = static_cast<long long>(blockIdx.x) * 128 + threadIdx.x;
  const long long b = idx / dv;
  if (b >= p.B) return;
  const int d = static_cast<int>(idx - b * dv) * (2 * P), left = p.dim - d;
  f32x2 win[W][P], w[W][P], bias[P], out[P];
  const T* s = static_cast<const T*>(p.state) + b * (W - 1) * p.dim + d;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) load_channels<P>(win[k], s + static_cast<long long>(k) * p.dim, p.aligned, left);
  load_channels<P>(win[W - 1], static_cast<const T*>(p.x) + b * p.ld_x + d, p.aligned, left);
  load_filter<T, P, W>(w, bias, p.weight, p.bias, p.weight_f32, p.whole_w, d, p.dim);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    out[i] = bias[i];
#pragma unroll
    for (int k = 0; k < W; ++k) out[i] = fma2(w[k][i], win[k][i], out[i]);
    if (p.silu) out[i] = mul2(out[i], sigmoid2(out[i]));
  }
  store_channels<P>(static_cast<T*>(p.y) + b * p.dim + d, out, p.aligned, left);
  T* so = static_cast<T*>(p.state_out) + b * (W - 1) * p.dim + d;
#pragma unroll
  for (int k = 0; k < W - 1; ++k) store_channels<P>(so + static_cast<long long>(k) * p.dim, win[k + 1], p.aligned, left);
}

}  // namespace btp_conv
