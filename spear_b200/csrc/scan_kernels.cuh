// Selective state space scan, token-major (sm_100a): forward over prompts and one token.
//
//   Delta_t[d] = softplus(delta_t[d] + bias[d])  (or the plain sum)          u_t = Delta_t x_t
//   h_t[d,n]   = exp(Delta_t[d] A[d,n]) h_{t-1}[d,n] + u_t[d] B_t[n]
//   y_t[d]     = sum_n C_t[n] h_t[d,n] + D[d] x_t[d],  times z_t sigmoid(z_t) where there is a gate
//
// Layout.  A warp walks down the tokens of 64 / SG channels; a lane holds 2 neighbouring channels x 4 states of h, SG = N / 4 lanes
// share the channels.  Pairs of states go through two-wide (f32x2) arithmetic.  Raw rows arrive by asynchronous copies one tile
// of 16 tokens ahead; every lane turns its share of a group of 4 tokens into step sizes and inputs and hands them to the other
// lanes of its channels by warp exchanges, which also bring the partial sums of y back to it for D x, gate and store.  Nothing but
// the raw rows goes through shared memory.
// Measured against lanes of 4 channels x 4 states with step sizes and y staged in shared memory (8 x 2048 tokens x 2048
// channels x 16 states): 298 us against 520; 2 channels x 8 states 372 (half the warps), 2 x 2 states 343 (more exchanges).  Of today's
// 300 us 4 are for step sizes of full accuracy.
//
// Bound: one exponential per (token, channel, state) on the special-function unit, 16 per clock and SM: 119 us for those 5.4e8.  At
// that shape a scheduler has two warps and issues half of the time; with the tokens split 16 times (many warps) the same kernel
// takes 212 us, two thirds of the special-function unit's rate.  Taking a share of the exponentials by a polynomial on the multiply-add
// pipe was slower (the instructions it adds count more).
//
// Few channels or sequences: the tokens are split over `splits` chunks.  A first kernel runs each chunk from state zero and
// keeps its last state and its sum of step sizes (the product of its decays is exp(A times that sum), see over_chunk); the second
// combines the chunks before its own in order and runs its chunk from there.  That doubles the exponentials, so the rule in
// scan_sm100.cu splits only where warps are missing.
#pragma once

#include <type_traits>

#include "btp_elem.cuh"

namespace btp_scan {

using namespace btp_elem;

constexpr int kTile = 16;        // tokens per tile
constexpr int kCheckpoint = 16;  // tokens between the states that the forward keeps for the backward

// exp(Delta A) with the rate to the base 2.  ex2.approx is low by 2e-8 on average for results between 0.7 and 1 (measured), and a state that
// remembers 1000 tokens is multiplied by 1000 such factors: 2^-25 in the exponent takes that out, at no cost.  A step of 0 still
// keeps the state as it is: ex2.approx of 2^-25 is 1.
constexpr float kDecayBias = 0x1p-25f;
__device__ __forceinline__ f32x2 decay2(f32x2 delta, f32x2 A2) { return ex2_2(fma2(delta, A2, both(kDecayBias))); }

struct ScanParams {
  const void* x;
  const void* delta;
  const void* B;
  const void* C;
  const void* z;          // nullptr: no gate
  const float* A;         // [dim, N]
  const float* D;         // [dim] or nullptr
  const float* bias;      // [dim] or nullptr
  const float* initial;   // [B, dim, N] or nullptr
  const int* lengths;     // [B] or nullptr
  void* y;                // [B, L, dim]
  float* state;           // [B, dim, N] or nullptr
  float* checkpoints;     // [B, ceil(L / 16), dim, N] or nullptr: the state before each 16th token
  float* carry;           // [splits - 1][B][dim][N] last states, then [splits - 1][B][dim] sums of step sizes
  long long x_b, x_t, d_b, d_t, z_b, z_t, B_b, B_t, C_b, C_t;
  int batch, L, dim, N;
  int splits, chunk;      // chunk: tokens per split, a multiple of 32
  bool softplus;
  bool al_x, al_d, al_z, al_B, al_C;  // 16-byte copies are possible
};

// A tile of the backward's carries: lanes of 4 channels x 4 states, step sizes and inputs in float, C given twice.
template <class T, int SG>
struct Tile {
  static constexpr int kStates = 4 * SG;
  static constexpr int kChannels = 128 / SG;
  T x[2][kTile][kChannels];
  T d[2][kTile][kChannels];
  T z[2][kTile][kChannels];
  T C[2][kTile][kStates];
  float delta[kTile][kChannels];
  float u[kTile][kChannels];
  float C2[kTile][kStates * 2];
};

// Sums four values over the SG lanes of a state group.  SG >= 4: lane s ends with value s & 3; SG == 2: lane s with values
// 2s and 2s + 1.  v[0], v[1] are the pairs (0, 1) and (2, 3).
template <int SG>
__device__ __forceinline__ void reduce_states(float (&out)[2], f32x2 v0, f32x2 v1, int s) {
  if (SG == 2) {
    const f32x2 keep = (s & 1) ? v1 : v0, give = (s & 1) ? v0 : v1;
    const f32x2 sum = add2(keep, __shfl_xor_sync(0xffffffffu, give, 1));
    unpack2(out[0], out[1], sum);
    return;
  }
  const f32x2 keep = (s & 2) ? v1 : v0, give = (s & 2) ? v0 : v1;
  const f32x2 sum = add2(keep, __shfl_xor_sync(0xffffffffu, give, 2));
  float a, b;
  unpack2(a, b, sum);
  const float k = (s & 1) ? b : a, o = (s & 1) ? a : b;
  float r = k + __shfl_xor_sync(0xffffffffu, o, 1);
  if (SG >= 8) r += __shfl_xor_sync(0xffffffffu, r, 4);
  if (SG >= 16) r += __shfl_xor_sync(0xffffffffu, r, 8);
  out[0] = r;
  out[1] = 0.f;
}

// Four consecutive states of one channel of a [.., N] row; states from N on are 0.  STREAM: read (written) once, first to leave the cache.
template <bool STREAM = false>
__device__ __forceinline__ void load_states(float (&v)[4], const float* row, int n0, int N) {
  if ((N & 3) == 0) {
    if (n0 < N) {
      const float4* at = reinterpret_cast<const float4*>(row + n0);
      const float4 q = STREAM ? __ldcs(at) : *at;
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      v[0] = v[1] = v[2] = v[3] = 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = n0 + k < N ? row[n0 + k] : 0.f;
  }
}
template <bool STREAM = false>
__device__ __forceinline__ void store_states(float* row, const float (&v)[4], int n0, int N) {
  if ((N & 3) == 0) {
    if (n0 < N) {
      const float4 q = make_float4(v[0], v[1], v[2], v[3]);
      if (STREAM)
        __stcs(reinterpret_cast<float4*>(row + n0), q);
      else
        *reinterpret_cast<float4*>(row + n0) = q;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n0 + k < N) row[n0 + k] = v[k];
  }
}

// The lane's 4 channels x 4 states, pairs of channels: r[p][n] holds channels 2p and 2p + 1.
struct LaneState {
  f32x2 r[2][4];
};
__device__ __forceinline__ void load_lane(LaneState& h, const float* base, int c0, int dim, int n0, int N, float scale) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    float a[4] = {}, b[4] = {};
    if (c0 + 2 * p < dim) load_states(a, base + static_cast<long long>(c0 + 2 * p) * N, n0, N);
    if (c0 + 2 * p + 1 < dim) load_states(b, base + static_cast<long long>(c0 + 2 * p + 1) * N, n0, N);
#pragma unroll
    for (int n = 0; n < 4; ++n) h.r[p][n] = pack2(a[n] * scale, b[n] * scale);
  }
}
__device__ __forceinline__ void store_lane(float* base, const LaneState& h, int c0, int dim, int n0, int N) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    float a[4], b[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) unpack2(a[n], b[n], h.r[p][n]);
    if (c0 + 2 * p < dim) store_states(base + static_cast<long long>(c0 + 2 * p) * N, a, n0, N);
    if (c0 + 2 * p + 1 < dim) store_states(base + static_cast<long long>(c0 + 2 * p + 1) * N, b, n0, N);
  }
}
// Rates to the base 2, held above -inf so that a step of size 0 keeps the state.
__device__ __forceinline__ void load_rates(LaneState& A2, const float* A, int c0, int dim, int n0, int N) {
  load_lane(A2, A, c0, dim, n0, N, kLog2e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a, b;
    unpack2(a, b, A2.r[i >> 2][i & 3]);
    A2.r[i >> 2][i & 3] = pack2(a < -3e38f ? -3e38f : a, b < -3e38f ? -3e38f : b);
  }
}
// h = 2^(2 half) h + last: the effect of a whole chunk, 2 half being the rate to the base 2 times the sum of its step sizes.  The factor
// may leave the range of a float where the token by token product does not, so h takes it in two equal parts; and 0 stays 0
// however much the chunk would make a state grow, so the parts are held below infinity.
__device__ __forceinline__ f32x2 over_chunk(f32x2 h, f32x2 half, f32x2 last) {
  const f32x2 a = pack2(ex2(fminf(lo2(half), 127.99f)), ex2(fminf(hi2(half), 127.99f)));
  return fma2(mul2(a, h), a, last);
}
__device__ __forceinline__ void apply_chunk(LaneState& h, const LaneState& A2, const LaneState& last, f32x2 t0, f32x2 t1) {  // t0, t1: half of the sums
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    h.r[0][n] = over_chunk(h.r[0][n], mul2(A2.r[0][n], t0), last.r[0][n]);
    h.r[1][n] = over_chunk(h.r[1][n], mul2(A2.r[1][n], t1), last.r[1][n]);
  }
}
__device__ __forceinline__ void load_totals(f32x2& t0, f32x2& t1, const float* row, int c0, int dim) {
  float t[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = c0 + k < dim ? 0.5f * row[c0 + k] : 0.f;
  t0 = pack2(t[0], t[1]);
  t1 = pack2(t[2], t[3]);
}
// Lanes that stand for states from N on keep 0 there, whatever the inputs hold.
__device__ __forceinline__ void clear_padding(LaneState& h, int n0, int N) {
#pragma unroll
  for (int n = 0; n < 4; ++n)
    if (n0 + n >= N) h.r[0][n] = h.r[1][n] = 0ull;
}

__device__ __forceinline__ f32x2 channel_pair(const float* v, int c, int dim) {
  return pack2(v && c < dim ? v[c] : 0.f, v && c + 1 < dim ? v[c + 1] : 0.f);
}

// ---------------------------------------------------------------------------------------------------- forward
// A lane holds 2 neighbouring channels x 4 states as pairs of states; SG lanes share the channel pair.  The lane with the odd
// index in its group takes the odd channel as its first: "own" and "other" below, so that nothing is selected by parity.
// Of a group of 4 tokens each lane prepares kOwn tokens of its own channel (step size, input, in the end gate and output), straight
// from the copied rows; the group's lanes pass step sizes and inputs to one another, and sums of y back, by exchanges in the warp.
template <class T, int SG>
struct FwdTile {
  static constexpr int kStates = 4 * SG;
  static constexpr int kChannels = 64 / SG;
  T x[2][kTile][kChannels];
  T d[2][kTile][kChannels];
  T z[2][kTile][kChannels];
  T B[2][kTile][kStates];
  T C[2][kTile][kStates];
};

// Four consecutive states of the channels c0, c1 as pairs of states; a channel or state that is not there is 0.
struct PairState {
  f32x2 r[2][2];
};
__device__ __forceinline__ void load_pair_state(PairState& h, const float* base, int c0, int c1, int dim, int n0, int N) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int ch = c ? c1 : c0;
    float v[4] = {};
    if (ch < dim) load_states(v, base + static_cast<long long>(ch) * N, n0, N);
    h.r[c][0] = pack2(v[0], v[1]);
    h.r[c][1] = pack2(v[2], v[3]);
  }
}
__device__ __forceinline__ void store_pair_state(float* base, const PairState& h, int c0, int c1, int dim, int n0, int N) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int ch = c ? c1 : c0;
    float v[4];
    unpack2(v[0], v[1], h.r[c][0]);
    unpack2(v[2], v[3], h.r[c][1]);
    if (ch < dim) store_states(base + static_cast<long long>(ch) * N, v, n0, N);
  }
}
// Lanes that stand for states from N on keep 0 there, whatever the inputs hold.
__device__ __forceinline__ void clear_pair_padding(PairState& h, int n0, int N) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (n0 + 2 * k >= N)
        h.r[c][k] = 0ull;
      else if (n0 + 2 * k + 1 >= N)
        h.r[c][k] = pack2(lo2(h.r[c][k]), 0.f);
    }
}

// One warp per (channels, chunk, sequence).  CARRY: only the chunk's last state and sum of step sizes, from state zero.
template <class T, int SG, bool CARRY>
__global__ void __launch_bounds__(32) scan_forward_kernel(const ScanParams p) {
  using S = FwdTile<T, SG>;
  constexpr int WC = S::kChannels, NP = S::kStates;
  constexpr int kOwn = SG >= 8 ? 1 : 8 / SG;  // tokens of a group of 4 that a lane prepares
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  grid_dependency_wait();
  const int lane = threadIdx.x, g = lane / SG, s = lane % SG;
  const int cblocks = (p.dim + WC - 1) / WC;
  const int splits = CARRY ? p.splits - 1 : p.splits;
  const int cb = blockIdx.x % cblocks;
  const int rest = blockIdx.x / cblocks;
  const int q = rest % splits;
  const long long b = rest / splits;
  const int cw = cb * WC, odd = s & 1;
  const int l0 = 2 * g + odd, l1 = 2 * g + 1 - odd;  // own and other channel within the warp's
  const int c0 = cw + l0, c1 = cw + l1, n0 = 4 * s;
  const int n_tok = tokens_of(p.lengths, b, p.L);
  const int first = q * p.chunk, end = min(p.L, first + p.chunk), live = min(end, n_tok);
  const int cols = min(WC, p.dim - cw);
  const bool full = p.N == NP;

  PairState A2, h;
  load_pair_state(A2, p.A, c0, c1, p.dim, n0, p.N);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // rates to the base 2, held above -inf so that a step of size 0 keeps the state
      float a, e;
      unpack2(a, e, mul2(A2.r[c][k], both(kLog2e)));
      A2.r[c][k] = pack2(a < -3e38f ? -3e38f : a, e < -3e38f ? -3e38f : e);
      h.r[c][k] = 0ull;
    }
  if (!CARRY && p.initial) load_pair_state(h, p.initial + b * p.dim * p.N, c0, c1, p.dim, n0, p.N);
  const long long per_chunk = static_cast<long long>(p.batch) * p.dim;
  float* totals = p.carry + (p.splits - 1) * per_chunk * p.N;
  if (!CARRY) {
    for (int k = 0; k < q; ++k) {  // the chunks before, in order: h = exp(A total) h + last
      PairState last;
      load_pair_state(last, p.carry + (k * per_chunk + b * p.dim) * p.N, c0, c1, p.dim, n0, p.N);
      const float* row = totals + k * per_chunk + b * p.dim;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int ch = c ? c1 : c0;
        const f32x2 half = both(ch < p.dim ? 0.5f * row[ch] : 0.f);
#pragma unroll
        for (int i = 0; i < 2; ++i) h.r[c][i] = over_chunk(h.r[c][i], mul2(A2.r[c][i], half), last.r[c][i]);
      }
    }
  }
  const float bias = p.bias && c0 < p.dim ? p.bias[c0] : 0.f, skip = p.D && c0 < p.dim ? p.D[c0] : 0.f;
  for (int i = lane; i < 2 * kTile * (WC - cols); i += 32) {  // channels that are not there: never copied, read as zeros
    const int at = i / (WC - cols) * WC + cols + i % (WC - cols);
    (&sm.x[0][0][0])[at] = (&sm.d[0][0][0])[at] = (&sm.z[0][0][0])[at] = from_f<T>(0.f);
  }
  for (int i = lane; i < 2 * kTile * (NP - p.N); i += 32) {  // nor states
    const int at = i / (NP - p.N) * NP + p.N + i % (NP - p.N);
    (&sm.B[0][0][0])[at] = (&sm.C[0][0][0])[at] = from_f<T>(0.f);
  }
  const T* x = static_cast<const T*>(p.x) + b * p.x_b + cw;
  const T* dl = static_cast<const T*>(p.delta) + b * p.d_b + cw;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.z_b + cw : nullptr;
  const T* Bm = static_cast<const T*>(p.B) + b * p.B_b;
  const T* Cm = static_cast<const T*>(p.C) + b * p.C_b;
  T* y = static_cast<T*>(p.y) + (b * p.L) * p.dim + cw;
  const auto load_tile = [&](int st, int t0) {
    const int rows = min(kTile, live - t0);
    fetch<T, kTile, WC, 32>(sm.x[st], x + t0 * p.x_t, p.x_t, rows, cols, p.al_x, lane);
    fetch<T, kTile, WC, 32>(sm.d[st], dl + t0 * p.d_t, p.d_t, rows, cols, p.al_d, lane);
    fetch<T, kTile, NP, 32>(sm.B[st], Bm + t0 * p.B_t, p.B_t, rows, p.N, p.al_B, lane);
    if (!CARRY) {
      fetch<T, kTile, NP, 32>(sm.C[st], Cm + t0 * p.C_t, p.C_t, rows, p.N, p.al_C, lane);
      if (z) fetch<T, kTile, WC, 32>(sm.z[st], z + t0 * p.z_t, p.z_t, rows, cols, p.al_z, lane);
    }
  };
  float total = 0.f;
  const int mine = (s >> 1) * kOwn & 3;                          // first token of each group that this lane prepares
  const int own_src = g * SG + odd, oth_src = g * SG + 1 - odd;  // lanes that prepare token 0 of the own and the other channel
  // The walk over the chunk, once for the usual cases (all states there, softplus, a gate or none) and once with everything tested: a
  // branch per token would keep the tokens of a group from overlapping.
  const auto walk = [&](auto usual, auto gated) {
    constexpr bool kFull = decltype(usual)::value;
    const bool softplus_on = kFull || p.softplus, gate_on = kFull ? decltype(gated)::value : z != nullptr;
    if (first < live) load_tile(0, first);
    copy_commit();
    int st = 0;
    for (int t0 = first; t0 < live; t0 += kTile, st ^= 1) {
      if (t0 + kTile < live) load_tile(st ^ 1, t0 + kTile);
      copy_commit();
      copy_wait<1>();
      __syncwarp();
      const int nt = min(kTile, live - t0);
      if (!CARRY && p.checkpoints && t0 % kCheckpoint == 0) {
        const long long at = b * ((p.L + kCheckpoint - 1) / kCheckpoint) + t0 / kCheckpoint;
        store_pair_state(p.checkpoints + at * p.dim * p.N, h, c0, c1, p.dim, n0, p.N);
      }
      if (nt < kTile) {  // rows behind the last token: zeros leave the state as it is
        for (int i = lane; i < (kTile - nt) * NP; i += 32) (&sm.B[st][nt][0])[i] = (&sm.C[st][nt][0])[i] = from_f<T>(0.f);
        __syncwarp();
      }
      float de[kOwn], xx[kOwn], uu[kOwn];  // step sizes, x and inputs of this lane's tokens of a group
      const auto prepare = [&](int t) {
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
          de[k] = to_f(sm.d[st][t + mine + k][l0]) + bias;
          xx[k] = to_f(sm.x[st][t + mine + k][l0]);
        }
        if (softplus_on) {
          if constexpr (kOwn == 1) {
            de[0] = softplus(de[0]);
          } else {
#pragma unroll
            for (int k = 0; k < kOwn; k += 2) unpack2(de[k], de[k + 1], softplus2(pack2(de[k], de[k + 1])));
          }
        }
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
          uu[k] = de[k] * xx[k];
          if (t + mine + k >= nt) de[k] = uu[k] = 0.f;
          total += de[k];
        }
      };
      const auto group = [&](int t) {
        prepare(t);
        float yo[4], yt[4];  // sums of the own and the other channel
        float dc[4][2], uc[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (SG == 2) {
            dc[j][0] = de[j % kOwn], uc[j][0] = uu[j % kOwn];
            dc[j][1] = __shfl_xor_sync(0xffffffffu, dc[j][0], 1);
            uc[j][1] = __shfl_xor_sync(0xffffffffu, uc[j][0], 1);
          } else {
            const int up = 2 * (j / kOwn);
            dc[j][0] = __shfl_sync(0xffffffffu, de[j % kOwn], own_src + up);
            dc[j][1] = __shfl_sync(0xffffffffu, de[j % kOwn], oth_src + up);
            uc[j][0] = __shfl_sync(0xffffffffu, uu[j % kOwn], own_src + up);
            uc[j][1] = __shfl_sync(0xffffffffu, uu[j % kOwn], oth_src + up);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x2 bn[2], cn[2];
          load_quad(bn, &sm.B[st][t + j][n0]);
          if (!CARRY) load_quad(cn, &sm.C[st][t + j][n0]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const f32x2 d2 = both(dc[j][c]), u2 = both(uc[j][c]);
#pragma unroll
            for (int k = 0; k < 2; ++k) h.r[c][k] = fma2(decay2(d2, A2.r[c][k]), h.r[c][k], mul2(u2, bn[k]));
          }
          if (!kFull) clear_pair_padding(h, n0, p.N);
          if (!CARRY) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const f32x2 v = fma2(cn[1], h.r[c][1], mul2(cn[0], h.r[c][0]));
              (c ? yt : yo)[j] = lo2(v) + hi2(v);
            }
          }
        }
        if (CARRY) return;
        // sums over the group's lanes: each ends with the tokens and the channel that it has prepared
        float out[kOwn];
#pragma unroll
        for (int j = 0; j < 4; ++j) yo[j] += __shfl_xor_sync(0xffffffffu, yt[j], 1);
        if constexpr (SG == 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) out[j] = yo[j];
        } else {
          const bool up = s & (SG == 4 ? 2 : 4);
          float a[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) a[j] = (up ? yo[2 + j] : yo[j]) + __shfl_xor_sync(0xffffffffu, up ? yo[j] : yo[2 + j], SG == 4 ? 2 : 4);
          if constexpr (SG == 4) {
            out[0] = a[0], out[1] = a[1];
          } else {
            const bool hi = s & 2;
            out[0] = (hi ? a[1] : a[0]) + __shfl_xor_sync(0xffffffffu, hi ? a[0] : a[1], 2);
            if (SG == 16) out[0] += __shfl_xor_sync(0xffffffffu, out[0], 8);
          }
        }
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
          const int r = t + mine + k;
          float v = fmaf(skip, xx[k], out[k]);
          if (gate_on) {
            const float zz = to_f(sm.z[st][r][l0]);
            v *= zz * sigmoid(zz);
          }
          if (r < nt && c0 < p.dim && (SG < 16 || s < 8)) y[static_cast<long long>(t0 + r) * p.dim + l0] = from_f<T>(v);
        }
      };
      if (nt == kTile) {  // in one piece: a group's first loads and last exchanges overlap with its neighbours' arithmetic
#pragma unroll
        for (int t = 0; t < kTile; t += 4) group(t);
      } else {
        for (int t = 0; t < nt; t += 4) group(t);
      }
      __syncwarp();
    }
  };
  if (full && p.softplus) {
    if (!CARRY && z)
      walk(std::true_type{}, std::true_type{});
    else
      walk(std::true_type{}, std::false_type{});
  } else {
    walk(std::false_type{}, std::false_type{});
  }
  copy_wait<0>();
  if (CARRY) {
    store_pair_state(p.carry + (q * per_chunk + b * p.dim) * p.N, h, c0, c1, p.dim, n0, p.N);
    // this lane's tokens; the others of the channel lie in the other lanes of the same parity
    if (SG >= 4) total += __shfl_xor_sync(0xffffffffu, total, 2);
    if (SG >= 8) total += __shfl_xor_sync(0xffffffffu, total, 4);
    if (s < 2 && c0 < p.dim) totals[q * per_chunk + b * p.dim + c0] = total;
    return;
  }
  for (int t = max(first, live); t < end; ++t)
    for (int c = lane; c < cols; c += 32) y[static_cast<long long>(t) * p.dim + c] = from_f<T>(0.f);
  if (p.state && q == p.splits - 1) store_pair_state(p.state + b * p.dim * p.N, h, c0, c1, p.dim, n0, p.N);
}

// ---------------------------------------------------------------------------------------------------- one token
struct ScanStepParams {
  const void* x;      // [B, dim], row pitches ld_*
  const void* delta;
  const void* B;      // [B, N]
  const void* C;
  const void* z;      // or nullptr
  const float* A;
  const float* D;
  const float* bias;
  const float* state;  // [B, dim, N]
  float* state_out;    // may be `state`
  void* y;             // [B, dim]
  long long ld_x, ld_d, ld_z, ld_B, ld_C;
  int batch, dim, N;
  bool softplus;
  bool al_B, al_C;     // four states of B and C are one word
  int ctas;            // CTAs over the channels
};

constexpr int kStepBatch = 4;  // sequences per thread

// SG lanes share a channel, 4 states each, for four sequences at a time: four states' loads are under way together, A is read once, and
// each lane prepares (step size, input, later gate and output) its share of the four and hands it to the others, as the prompt's
// kernel does with four tokens.  Bound by the states' traffic, 8 bytes per state.
// Measured at 256 sequences x 4096 channels x 16 states: 37 us (3.8 TB/s; 39 without the
// streaming hints); with every lane preparing for itself 54 us (four times the instructions).
template <class T, int SG>
__global__ void __launch_bounds__(128, 7) scan_step_kernel(const ScanStepParams p) {
  constexpr int kOwn = SG >= 4 ? 1 : 4 / SG;
  grid_dependency_wait();
  const int in = static_cast<int>(blockIdx.x % p.ctas) * 128 + threadIdx.x;
  if ((in & ~31) / SG >= p.dim) return;  // a warp without a channel: it must not even read, another may be writing in place
  const int lane = threadIdx.x & 31, d = in / SG, s = in % SG, n0 = 4 * s;
  const bool ok = d < p.dim;
  const int dd = ok ? d : p.dim - 1;  // lanes without a channel follow the last one: the exchanges below need whole warps
  const int b0 = static_cast<int>(blockIdx.x / p.ctas) * kStepBatch, nb = min(kStepBatch, p.batch - b0);
  float h[kStepBatch][4], A[4];
  f32x2 Bn[kStepBatch][2], Cn[kStepBatch][2];
#pragma unroll
  for (int i = 0; i < kStepBatch; ++i) {
    const long long b = b0 + (i < nb ? i : 0);
    load_states<true>(h[i], p.state + (b * p.dim + dd) * p.N, n0, p.N);
    load_channels<2>(Bn[i], static_cast<const T*>(p.B) + b * p.ld_B + n0, p.al_B && n0 < p.N, p.N - n0);
    load_channels<2>(Cn[i], static_cast<const T*>(p.C) + b * p.ld_C + n0, p.al_C && n0 < p.N, p.N - n0);
  }
  const int mine = SG >= 4 ? (s & 3) : s * kOwn;  // first sequence of the four that this lane prepares
  float x[kOwn], v[kOwn], z[kOwn];
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    const long long b = b0 + (mine + k < nb ? mine + k : 0);
    x[k] = to_f(static_cast<const T*>(p.x)[b * p.ld_x + dd]);
    v[k] = to_f(static_cast<const T*>(p.delta)[b * p.ld_d + dd]);
    z[k] = p.z ? to_f(static_cast<const T*>(p.z)[b * p.ld_z + dd]) : 0.f;
  }
  load_states(A, p.A + static_cast<long long>(dd) * p.N, n0, p.N);
  const float bias = p.bias ? p.bias[dd] : 0.f, skip = p.D ? p.D[dd] : 0.f;
  f32x2 A2[2];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    A[k] *= kLog2e;
    A[k] = A[k] < -3e38f ? -3e38f : A[k];  // held above -inf as in the prompt's kernel; NaN stays
  }
  A2[0] = pack2(A[0], A[1]), A2[1] = pack2(A[2], A[3]);
  float u[kOwn];
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    v[k] += bias;
    if (p.softplus) v[k] = softplus(v[k]);
    u[k] = v[k] * x[k];
  }
  float y[kStepBatch];
#pragma unroll
  for (int i = 0; i < kStepBatch; ++i) {
    const int from = lane - s + i / kOwn;
    const f32x2 d2 = both(__shfl_sync(0xffffffffu, v[i % kOwn], from)), u2 = both(__shfl_sync(0xffffffffu, u[i % kOwn], from));
    f32x2 g[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      g[k] = fma2(decay2(d2, A2[k]), pack2(h[i][2 * k], h[i][2 * k + 1]), mul2(u2, Bn[i][k]));
      if (n0 + 2 * k >= p.N) g[k] = 0ull;  // states that are not there
      if (n0 + 2 * k + 1 >= p.N) g[k] = pack2(lo2(g[k]), 0.f);
      unpack2(h[i][2 * k], h[i][2 * k + 1], g[k]);
    }
    const f32x2 sum = fma2(Cn[i][1], g[1], mul2(Cn[i][0], g[0]));
    y[i] = lo2(sum) + hi2(sum);
  }
  if (ok) {
#pragma unroll
    for (int i = 0; i < kStepBatch; ++i)
      if (i < nb) {
        store_states<true>(p.state_out + (static_cast<long long>(b0 + i) * p.dim + d) * p.N, h[i], n0, p.N);
      }
  }
  // sums over the channel's lanes: each ends with the sequences that it has prepared
  float out[kOwn];
  if constexpr (SG == 2) {
    const bool up = s & 1;
#pragma unroll
    for (int k = 0; k < 2; ++k) out[k] = (up ? y[2 + k] : y[k]) + __shfl_xor_sync(0xffffffffu, up ? y[k] : y[2 + k], 1);
  } else {
    const bool hi = s & 2, odd = s & 1;
    float a[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) a[k] = (hi ? y[2 + k] : y[k]) + __shfl_xor_sync(0xffffffffu, hi ? y[k] : y[2 + k], 2);
    out[0] = (odd ? a[1] : a[0]) + __shfl_xor_sync(0xffffffffu, odd ? a[0] : a[1], 1);
#pragma unroll
    for (int o = 4; o < SG; o *= 2) out[0] += __shfl_xor_sync(0xffffffffu, out[0], o);
  }
#pragma unroll
  for (int k = 0; k < kOwn; ++k) {
    float r = fmaf(skip, x[k], out[k]);
    if (p.z) r *= z[k] * sigmoid(z[k]);
    if (ok && mine + k < nb && (SG < 8 || s < 4)) static_cast<T*>(p.y)[static_cast<long long>(b0 + mine + k) * p.dim + d] = from_f<T>(r);
  }
}

}  // namespace btp_scan
