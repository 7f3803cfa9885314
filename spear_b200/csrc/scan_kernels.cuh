// Selective state space scan, token-major (sm_100a): forward over prompts and one token.
//
//   Delta_t[d] = softplus(delta_t[d] + bias[d])  (or the plain sum)          u_t = Delta_t x_t
//   h_t[d,n]   = exp(Delta_t[d] A[d,n]) h_{t-1}[d,n] + u_t[d] B_t[n]
//   y_t[d]     = sum_n C_t[n] h_t[d,n] + D[d] x_t[d],  times z_t sigmoid(z_t) where there is a gate
//
// Layout.  A warp walks down the tokens of 128 / SG channels: lane = (channel group g, state group s), SG state groups;
// a lane holds 4 channels x 4 states of h as pairs of neighbouring channels, so that products and sums are two-wide
// (f32x2) with the step sizes as they lie in memory and with B and C given twice.  y is summed over a lane's 4 states in
// registers and over the SG lanes by exchanging halves: 3 exchanges for 4 channels and 4 lanes.
// Tiles of 16 tokens arrive by asynchronous copies one tile ahead; a first pass over the tile turns the raw values into
// step sizes, inputs u and doubled B, C in float; a last pass adds D x, applies the gate and stores.
//
// Bound: one exponential per (token, channel, state) on the special-function unit, 16 per clock and SM.
//
// Few channels or sequences: the tokens are split over `splits` chunks.  A first kernel runs each chunk from state zero and
// keeps its last state and its sum of step sizes (the product of its decays is exp(A times that sum), one exponential); the second
// combines the chunks before its own in order and runs its chunk from there.  That doubles the exponentials, so the rule in
// scan_sm100.cu splits only where warps are missing.
#pragma once

#include <type_traits>

#include "btp_elem.cuh"

namespace btp_scan {

using namespace btp_elem;

constexpr int kTile = 16;        // tokens per tile
constexpr int kCheckpoint = 16;  // tokens between the states that the forward keeps for the backward

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
  bool al_x, al_d, al_z, al_B, al_C, al_y;  // 16-byte copies (y: pairs) are possible
};

template <class T, int SG>
struct Tile {
  static constexpr int kStates = 4 * SG;
  static constexpr int kChannels = 128 / SG;
  T x[2][kTile][kChannels];
  T d[2][kTile][kChannels];
  T z[2][kTile][kChannels];
  T B[2][kTile][kStates];
  T C[2][kTile][kStates];
  float delta[kTile][kChannels];
  float u[kTile][kChannels];
  float B2[kTile][kStates * 2];
  float C2[kTile][kStates * 2];
};

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

// Four consecutive states of one channel of a [.., N] row; states from N on are 0.
__device__ __forceinline__ void load_states(float (&v)[4], const float* row, int n0, int N) {
  if ((N & 3) == 0) {
    if (n0 < N) {
      const float4 q = *reinterpret_cast<const float4*>(row + n0);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      v[0] = v[1] = v[2] = v[3] = 0.f;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = n0 + k < N ? row[n0 + k] : 0.f;
  }
}
__device__ __forceinline__ void store_states(float* row, const float (&v)[4], int n0, int N) {
  if ((N & 3) == 0) {
    if (n0 < N) *reinterpret_cast<float4*>(row + n0) = make_float4(v[0], v[1], v[2], v[3]);
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
// h = exp(A total) h + last: the effect of a whole chunk with step sizes that sum up to `total`.
__device__ __forceinline__ void apply_chunk(LaneState& h, const LaneState& A2, const LaneState& last, f32x2 t0, f32x2 t1) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    h.r[0][n] = fma2(ex2_2(mul2(A2.r[0][n], t0)), h.r[0][n], last.r[0][n]);
    h.r[1][n] = fma2(ex2_2(mul2(A2.r[1][n], t1)), h.r[1][n], last.r[1][n]);
  }
}
__device__ __forceinline__ void load_totals(f32x2& t0, f32x2& t1, const float* row, int c0, int dim) {
  float t[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) t[k] = c0 + k < dim ? row[c0 + k] : 0.f;
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
// A lane holds 2 neighbouring channels x KN states as pairs of states; SG lanes share the channel pair.  The lane with the odd
// index in its group takes the odd channel as its first: "own" and "other" below, so that nothing is selected by parity.
// Of a group of 4 tokens each lane prepares kOwn tokens of its own channel (step size, input, in the end gate and output), straight
// from the copied rows; the group's lanes pass step sizes and inputs to one another, and sums of y back, by exchanges in the warp.
template <class T, int KN, int SG>
struct FwdTile {
  static constexpr int kStates = KN * SG;
  static constexpr int kChannels = 64 / SG;
  T x[2][kTile][kChannels];
  T d[2][kTile][kChannels];
  T z[2][kTile][kChannels];
  T B[2][kTile][kStates];
  T C[2][kTile][kStates];
  float Bf[kTile][kStates];
  float Cf[kTile][kStates];
};

// KN consecutive states of the channels c0, c1 as pairs; a channel or state that is not there is 0.
template <int KN>
struct PairState {
  f32x2 r[2][KN / 2];
};
template <int KN>
__device__ __forceinline__ void load_pair_state(PairState<KN>& h, const float* base, int c0, int c1, int dim, int n0, int N) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int ch = c ? c1 : c0;
#pragma unroll
    for (int q = 0; q < KN / 4; ++q) {
      float v[4] = {};
      if (ch < dim) load_states(v, base + static_cast<long long>(ch) * N, n0 + 4 * q, N);
      h.r[c][2 * q] = pack2(v[0], v[1]);
      h.r[c][2 * q + 1] = pack2(v[2], v[3]);
    }
  }
}
template <int KN>
__device__ __forceinline__ void store_pair_state(float* base, const PairState<KN>& h, int c0, int c1, int dim, int n0, int N) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int ch = c ? c1 : c0;
#pragma unroll
    for (int q = 0; q < KN / 4; ++q) {
      float v[4];
      unpack2(v[0], v[1], h.r[c][2 * q]);
      unpack2(v[2], v[3], h.r[c][2 * q + 1]);
      if (ch < dim) store_states(base + static_cast<long long>(ch) * N, v, n0 + 4 * q, N);
    }
  }
}
template <int KN>
__device__ __forceinline__ void clear_pair_padding(PairState<KN>& h, int n0, int N) {
#pragma unroll
  for (int k = 0; k < KN / 2; ++k) {
    const int n = n0 + 2 * k;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (n >= N)
        h.r[c][k] = 0ull;
      else if (n + 1 >= N)
        h.r[c][k] = pack2(lo2(h.r[c][k]), 0.f);
    }
  }
}

// One warp per (channels, chunk, sequence).  CARRY: only the chunk's last state and sum of step sizes, from state zero.
template <class T, int KN, int SG, bool CARRY>
__global__ void __launch_bounds__(32) scan_forward_kernel(const ScanParams p) {
  using S = FwdTile<T, KN, SG>;
  constexpr int WC = S::kChannels, NP = S::kStates;
  constexpr int kOwn = SG >= 8 ? 1 : (SG == 1 ? 4 : 8 / SG);  // tokens of a group of 4 that a lane prepares
  constexpr int kMine = SG == 1 ? 2 : 1;                      // channels that it prepares them for
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
  const int c0 = cw + l0, c1 = cw + l1, n0 = KN * s;
  const int n_tok = tokens_of(p.lengths, b, p.L);
  const int first = q * p.chunk, end = min(p.L, first + p.chunk), live = min(end, n_tok);
  const int cols = min(WC, p.dim - cw);
  const bool full = p.N == NP;

  PairState<KN> A2, h;
  load_pair_state(A2, p.A, c0, c1, p.dim, n0, p.N);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int k = 0; k < KN / 2; ++k) {  // rates to the base 2, held above -inf so that a step of size 0 keeps the state
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
      PairState<KN> last;
      load_pair_state(last, p.carry + (k * per_chunk + b * p.dim) * p.N, c0, c1, p.dim, n0, p.N);
      const float* row = totals + k * per_chunk + b * p.dim;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int ch = c ? c1 : c0;
        const f32x2 total = both(ch < p.dim ? row[ch] : 0.f);
#pragma unroll
        for (int i = 0; i < KN / 2; ++i) h.r[c][i] = fma2(ex2_2(mul2(A2.r[c][i], total)), h.r[c][i], last.r[c][i]);
      }
    }
  }
  float bias[kMine], skip[kMine];
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    const int ch = m ? c1 : c0;
    bias[m] = p.bias && ch < p.dim ? p.bias[ch] : 0.f;
    skip[m] = p.D && ch < p.dim ? p.D[ch] : 0.f;
  }
  for (int i = lane; i < 2 * kTile * (WC - cols); i += 32) {  // channels that are not there: never copied, read as zeros
    const int at = i / (WC - cols) * WC + cols + i % (WC - cols);
    (&sm.x[0][0][0])[at] = (&sm.d[0][0][0])[at] = (&sm.z[0][0][0])[at] = from_f<T>(0.f);
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
  float total[kMine] = {};
  const int mine = SG == 1 ? 0 : (s >> 1) * kOwn & 3;       // first token of each group that this lane prepares
  const int own_src = g * SG + odd, oth_src = g * SG + 1 - odd;  // lanes that prepare token 0 of the own and the other channel
  // The walk over the chunk, once for the usual case (all states there, softplus, gate or not known) and once with everything tested:
  // a branch per token would keep the tokens of a group from overlapping.
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
    // B and C to float; rows behind the last token and states that are not there become zeros
#pragma unroll
    for (int i0 = 0; i0 < kTile * NP / 2; i0 += 32) {
      const int i = i0 + lane, r = i / (NP / 2), n = i % (NP / 2) * 2;
      const bool ok0 = r < nt && n < p.N, ok1 = r < nt && n + 1 < p.N;
      float v0, v1;
      unpack2(v0, v1, load_pair(&sm.B[st][r][n]));
      *reinterpret_cast<float2*>(&sm.Bf[r][n]) = make_float2(ok0 ? v0 : 0.f, ok1 ? v1 : 0.f);
      if (!CARRY) {
        unpack2(v0, v1, load_pair(&sm.C[st][r][n]));
        *reinterpret_cast<float2*>(&sm.Cf[r][n]) = make_float2(ok0 ? v0 : 0.f, ok1 ? v1 : 0.f);
      }
    }
    __syncwarp();
    for (int t = 0; t < nt; t += 4) {
      float de[kMine][kOwn], xx[kMine][kOwn], uu[kMine][kOwn];
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        const int col = m ? l1 : l0;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
          de[m][k] = to_f(sm.d[st][t + mine + k][col]) + bias[m];
          xx[m][k] = to_f(sm.x[st][t + mine + k][col]);
        }
        if (softplus_on) {
          if (kOwn == 1) {
            de[m][0] = softplus(de[m][0]);
          } else {
#pragma unroll
            for (int k = 0; k < kOwn; k += 2) unpack2(de[m][k], de[m][k + 1], softplus2(pack2(de[m][k], de[m][k + 1])));
          }
        }
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
          uu[m][k] = de[m][k] * xx[m][k];
          if (nt < kTile && t + mine + k >= nt) de[m][k] = uu[m][k] = 0.f;  // they leave the state as it is
          total[m] += de[m][k];
        }
      }
      float yo[4], yt[4];  // sums of the own and the other channel
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float dc[2], uc[2];
        if (SG == 1) {
          dc[0] = de[0][j], dc[1] = de[kMine - 1][j], uc[0] = uu[0][j], uc[1] = uu[kMine - 1][j];
        } else if (SG == 2) {
          dc[0] = de[0][j % kOwn], uc[0] = uu[0][j % kOwn];
          dc[1] = __shfl_xor_sync(0xffffffffu, dc[0], 1);
          uc[1] = __shfl_xor_sync(0xffffffffu, uc[0], 1);
        } else {
          const int up = 2 * (j / kOwn);
          dc[0] = __shfl_sync(0xffffffffu, de[0][j % kOwn], own_src + up);
          dc[1] = __shfl_sync(0xffffffffu, de[0][j % kOwn], oth_src + up);
          uc[0] = __shfl_sync(0xffffffffu, uu[0][j % kOwn], own_src + up);
          uc[1] = __shfl_sync(0xffffffffu, uu[0][j % kOwn], oth_src + up);
        }
        f32x2 bn[KN / 2], cn[KN / 2];
#pragma unroll
        for (int k = 0; k < KN / 4; ++k) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.Bf[t + j][n0 + 4 * k]);
          bn[2 * k] = v.x, bn[2 * k + 1] = v.y;
          if (!CARRY) {
            const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(&sm.Cf[t + j][n0 + 4 * k]);
            cn[2 * k] = w.x, cn[2 * k + 1] = w.y;
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const f32x2 d2 = both(dc[c]), u2 = both(uc[c]);
#pragma unroll
          for (int k = 0; k < KN / 2; ++k) h.r[c][k] = fma2(ex2_2(mul2(d2, A2.r[c][k])), h.r[c][k], mul2(u2, bn[k]));
        }
        if (!kFull) clear_pair_padding(h, n0, p.N);
        if (!CARRY) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            f32x2 v = mul2(cn[0], h.r[c][0]);
#pragma unroll
            for (int k = 1; k < KN / 2; ++k) v = fma2(cn[k], h.r[c][k], v);
            (c ? yt : yo)[j] = lo2(v) + hi2(v);
          }
        }
      }
      if (CARRY) continue;
      // sums over the group's lanes: each ends with the tokens and the channel that it has prepared
      float out[kMine][kOwn];
      if (SG == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          out[kMine - 1][j % kOwn] = yt[j];
          out[0][j % kOwn] = yo[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) yo[j] += __shfl_xor_sync(0xffffffffu, yt[j], 1);
        if (SG == 2) {
#pragma unroll
          for (int j = 0; j < 4; ++j) out[0][j % kOwn] = yo[j];
        } else {
          const bool up = s & (SG == 4 ? 2 : 4);
          float a[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) a[j] = (up ? yo[2 + j] : yo[j]) + __shfl_xor_sync(0xffffffffu, up ? yo[j] : yo[2 + j], SG == 4 ? 2 : 4);
          if (SG == 4) {
#pragma unroll
            for (int j = 0; j < 2; ++j) out[0][j % kOwn] = a[j];
          } else {
            const bool hi = s & 2;
            float r = (hi ? a[1] : a[0]) + __shfl_xor_sync(0xffffffffu, hi ? a[0] : a[1], 2);
            if (SG == 16) r += __shfl_xor_sync(0xffffffffu, r, 8);
            out[0][0] = r;
          }
        }
      }
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        const int col = m ? l1 : l0;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
          const int r = t + mine + k;
          float v = fmaf(skip[m], xx[m][k], out[m][k]);
          if (gate_on) {
            const float zz = to_f(sm.z[st][r][col]);
            v *= zz * sigmoid(zz);
          }
          if (r < nt && cw + col < p.dim && (SG < 16 || s < 8)) y[static_cast<long long>(t0 + r) * p.dim + col] = from_f<T>(v);
        }
      }
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
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      float v = total[m];  // this lane's tokens; the others of the channel lie in the other lanes of the same parity
      if (SG >= 4) v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (SG >= 8) v += __shfl_xor_sync(0xffffffffu, v, 4);
      const int ch = m ? c1 : c0;
      if (s < 2 && ch < p.dim) totals[q * per_chunk + b * p.dim + ch] = v;
    }
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
};

constexpr int kStepBatch = 4;  // sequences per thread: they share A, D and the bias

// SG lanes share a channel, 4 states each.  The states' traffic bounds it: 8 bytes per state.
template <class T, int SG>
__global__ void __launch_bounds__(128) scan_step_kernel(const ScanStepParams p) {
  grid_dependency_wait();
  const long long idx = static_cast<long long>(blockIdx.x) * 128 + threadIdx.x;
  const long long per_group = (static_cast<long long>(p.dim) * SG + 31) / 32 * 32;  // whole warps: the exchange below needs all lanes
  const long long bg = idx / per_group;
  const int in = static_cast<int>(idx - bg * per_group);
  const int d = in / SG, s = in % SG, n0 = 4 * s;
  if (bg * kStepBatch >= p.batch) return;
  const bool ok = d < p.dim;
  const int dd = ok ? d : p.dim - 1;
  float A[4], h[kStepBatch][4], Bn[kStepBatch][4], Cn[kStepBatch][4], x[kStepBatch], v[kStepBatch], z[kStepBatch];
  const int nb = min(kStepBatch, p.batch - static_cast<int>(bg) * kStepBatch);
  const long long b0 = bg * kStepBatch;
#pragma unroll
  for (int i = 0; i < kStepBatch; ++i) {
    if (i >= nb) break;
    const long long b = b0 + i;
    load_states(h[i], p.state + (b * p.dim + dd) * p.N, n0, p.N);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      Bn[i][k] = n0 + k < p.N ? to_f(static_cast<const T*>(p.B)[b * p.ld_B + n0 + k]) : 0.f;
      Cn[i][k] = n0 + k < p.N ? to_f(static_cast<const T*>(p.C)[b * p.ld_C + n0 + k]) : 0.f;
    }
    x[i] = to_f(static_cast<const T*>(p.x)[b * p.ld_x + dd]);
    v[i] = to_f(static_cast<const T*>(p.delta)[b * p.ld_d + dd]);
    z[i] = p.z ? to_f(static_cast<const T*>(p.z)[b * p.ld_z + dd]) : 0.f;
  }
  load_states(A, p.A + static_cast<long long>(dd) * p.N, n0, p.N);
  const float bias = p.bias ? p.bias[dd] : 0.f, skip = p.D ? p.D[dd] : 0.f;
#pragma unroll
  for (int i = 0; i < kStepBatch; ++i) {
    if (i >= nb) break;
    const long long b = b0 + i;
    float de = v[i] + bias;
    if (p.softplus) de = softplus(de);
    const float u = de * x[i];
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[i][k] = fmaf(ex2(de * (A[k] * kLog2e)), h[i][k], u * Bn[i][k]);
      if (n0 + k < p.N) y = fmaf(Cn[i][k], h[i][k], y);
    }
#pragma unroll
    for (int o = SG / 2; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (!ok) continue;
    store_states(p.state_out + (b * p.dim + dd) * p.N, h[i], n0, p.N);
    if (s == 0) {
      y = fmaf(skip, x[i], y);
      if (p.z) y *= z[i] * sigmoid(z[i]);
      static_cast<T*>(p.y)[b * p.dim + d] = from_f<T>(y);
    }
  }
}

}  // namespace btp_scan
