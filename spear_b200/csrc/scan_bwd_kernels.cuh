// Selective state space scan, backward (sm_100a).  Notation as in scan_kernels.cuh; dy is the gradient of the ungated output
// (the gradient of the gated one times z sigmoid(z)).
//
//   g_t  = C_t dy_t + a_{t+1} g_{t+1}                 gradient of h_t; g after the last token is the final state's
//   dC_t[n] = sum_d dy_t h_t       dB_t[n] = sum_d g_t u_t       du_t = sum_n g_t B_t       w_t = g_t a_t h_{t-1}
//   dA = sum_{b,t} w_t Delta_t     dDelta_t = sum_n w_t A + du_t x_t     dx_t = du_t Delta_t + dy_t D     dinitial = a_1 g_1
//
// The states are needed backwards in time.  The forward kept one every 16 tokens; a tile runs forward from there in steps of 4
// tokens and parks the state before each step in shared memory, then takes the steps from the last to the first: 4 tokens
// forward again with a_t and a_t h_{t-1} in registers (never a quotient by a_t), then 4 tokens backward.  So each exponential is
// taken twice.
// A CTA's warps hold neighbouring channels of the same tokens and add up dB and dC over them: a lane over its 4 channels, the
// lanes of a state group by exchanging halves (7 exchanges for 8 sums), the warps in shared memory.  Sums over the CTAs' channels
// and over sequences go through a buffer and a second kernel in a fixed order: the same call gives the same bits.
//
// Bound: the two-wide multiply-adds (about 13 per token, channel and state) and two exponentials.  Measured at 8 x 2048 tokens x 2048
// channels x 16 states, bfloat16: 816 us, and 169 us for the carries of its 16 chunks; 385 instructions per token and warp at 0.44 per
// cycle with the two warps that registers and shared memory leave a scheduler.  A thread would want more than the 255 registers that
// there are: 170 to 260 bytes of it spill.  In float a tile takes 144 KB (120 with 8 or 64 states), so one CTA fits: 1317 and 221 us.
#pragma once

#include "scan_kernels.cuh"

namespace btp_scan {

constexpr int kStep = 4;  // tokens whose decays and states are in registers at a time

struct ScanBwdParams {
  ScanParams f;             // inputs; y, state unused; carry: [splits - 1][B][dim][N] gradients, then the sums of step sizes
  const void* dy;           // [B, L, dim] gradient of the (gated) output
  const float* dstate;      // [B, dim, N] or nullptr
  void* dx;                 // [B, L, dim]
  void* ddelta;
  void* dz;                 // where there is a gate
  float* dinitial;          // [B, dim, N] or nullptr
  float* partial_bc;        // [channel blocks][B][L][2 N]
  float* partial_par;       // [splits][B] rows of par_pitch: dA, dD, dbias
  long long par_pitch;      // dim (N + 2) rounded up to 4: rows of dA are written 16 bytes at a time
  bool al_dy, al_out;       // al_out: pairs of the dense outputs
};

template <int SG>
struct BwdShape {
  static constexpr int kWarps = SG == 2 ? 2 : 4;  // 64-channel warps: two, so that a float tile fits
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kChannels = kWarps * 128 / SG;
  static constexpr int kStates = 4 * SG;
};

template <class T, int SG>
struct BwdTile {
  static constexpr int CW = BwdShape<SG>::kChannels, NP = BwdShape<SG>::kStates;
  T x[2][kTile][CW];
  T d[2][kTile][CW];
  T z[2][kTile][CW];
  T dy[2][kTile][CW];
  T B[2][kTile][NP];
  T C[2][kTile][NP];
  float delta[kTile][CW];
  float u[kTile][CW];    // then du
  float gy[kTile][CW];   // dy of the ungated output, then sum C h
  float wa[kTile][CW];   // sum_n w A (times log2 e)
  float B2[kTile][NP * 2];
  float C2[kTile][NP * 2];
  float red[BwdShape<SG>::kWarps][kTile][NP * 2];  // dB, dC of one warp's channels
  float4 park[kTile / kStep][4][BwdShape<SG>::kThreads];
};

// dB, dC of this lane's channels, v = (dB of states n0..n0+3, dC of the same), summed over the warp's channel groups: lanes exchange halves
// until each holds kHeld of the eight sums, at place channel_slot() of a row (dB of all states, dC of all states).
template <int SG>
struct ChannelSums {
  static constexpr int kHeld = SG == 16 ? 4 : SG == 8 ? 2 : 1;
  float v[kHeld];
};
template <int SG>
__device__ __forceinline__ int channel_slot(int lane, int n0) {
  return (lane & 16 ? 4 * SG : 0) + n0 + (SG <= 8 && lane & 8 ? 2 : 0) + (SG <= 4 && lane & 4 ? 1 : 0);
}
template <int SG>
__device__ __forceinline__ ChannelSums<SG> reduce_channels(const float (&v)[8], int lane) {
  ChannelSums<SG> r;
  float a[4];
  const bool hi = lane & 16;
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = (hi ? v[4 + k] : v[k]) + __shfl_xor_sync(0xffffffffu, hi ? v[k] : v[4 + k], 16);
  if constexpr (SG == 16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) r.v[k] = a[k];
  } else {
    const bool b3 = lane & 8;
    float c[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) c[k] = (b3 ? a[2 + k] : a[k]) + __shfl_xor_sync(0xffffffffu, b3 ? a[k] : a[2 + k], 8);
    if constexpr (SG == 8) {
      r.v[0] = c[0], r.v[1] = c[1];
    } else {
      const bool b2 = lane & 4;
      r.v[0] = (b2 ? c[1] : c[0]) + __shfl_xor_sync(0xffffffffu, b2 ? c[0] : c[1], 4);
      if (SG == 2) r.v[0] += __shfl_xor_sync(0xffffffffu, r.v[0], 2);
    }
  }
  return r;
}

// One warp per (channels, chunk from the second on, sequence): the gradient that the chunk hands to the state before it when none
// comes in from behind, and its sum of step sizes.  Uses Tile's x slot for dy.
template <class T, int SG>
__global__ void __launch_bounds__(32) scan_backward_carry_kernel(const ScanBwdParams bp) {
  using S = Tile<T, SG>;
  constexpr int WC = S::kChannels, NP = S::kStates, CP = WC / 2, RPI = 32 / CP;
  const ScanParams& p = bp.f;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  grid_dependency_wait();
  const int lane = threadIdx.x, g = lane / SG, s = lane % SG;
  const int cblocks = (p.dim + WC - 1) / WC;
  const int cb = blockIdx.x % cblocks;
  const int rest = blockIdx.x / cblocks;
  const int q = rest % (p.splits - 1) + 1;
  const long long b = rest / (p.splits - 1);
  const int cw = cb * WC, c0 = cw + 4 * g, n0 = 4 * s;
  const int n_tok = tokens_of(p.lengths, b, p.L);
  const int first = q * p.chunk, live = min(min(p.L, first + p.chunk), n_tok);
  const int cols = min(WC, p.dim - cw);
  const bool full = p.N == NP;
  LaneState A2, G;
  load_rates(A2, p.A, c0, p.dim, n0, p.N);
#pragma unroll
  for (int n = 0; n < 4; ++n) G.r[0][n] = G.r[1][n] = 0ull;
  const int cp = lane % CP, row0 = lane / CP, pc = cw + 2 * cp;
  const f32x2 bias = channel_pair(p.bias, pc, p.dim);
  for (int i = lane; i < 2 * kTile * (WC - cols); i += 32) {  // channels that are not there: never copied, read as zeros
    const int at = i / (WC - cols) * WC + cols + i % (WC - cols);
    (&sm.x[0][0][0])[at] = (&sm.d[0][0][0])[at] = (&sm.z[0][0][0])[at] = from_f<T>(0.f);
  }
  const T* dl = static_cast<const T*>(p.delta) + b * p.d_b + cw;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.z_b + cw : nullptr;
  const T* Cm = static_cast<const T*>(p.C) + b * p.C_b;
  const T* dy = static_cast<const T*>(bp.dy) + (b * p.L) * p.dim + cw;
  const auto load_tile = [&](int st, int t0) {
    const int rows = min(kTile, live - t0);
    fetch<T, kTile, WC, 32>(sm.x[st], dy + static_cast<long long>(t0) * p.dim, p.dim, rows, cols, bp.al_dy, lane);
    fetch<T, kTile, WC, 32>(sm.d[st], dl + t0 * p.d_t, p.d_t, rows, cols, p.al_d, lane);
    fetch<T, kTile, NP, 32>(sm.C[st], Cm + t0 * p.C_t, p.C_t, rows, p.N, p.al_C, lane);
    if (z) fetch<T, kTile, WC, 32>(sm.z[st], z + t0 * p.z_t, p.z_t, rows, cols, p.al_z, lane);
  };
  f32x2 sum0 = 0ull, sum1 = 0ull;
  const int tiles = live > first ? (live - first + kTile - 1) / kTile : 0;
  if (tiles) load_tile(0, first + (tiles - 1) * kTile);
  copy_commit();
  int st = 0;
  for (int i_t = tiles - 1; i_t >= 0; --i_t, st ^= 1) {
    const int t0 = first + i_t * kTile, nt = min(kTile, live - t0);
    if (i_t) load_tile(st ^ 1, t0 - kTile);
    copy_commit();
    copy_wait<1>();
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kTile; i += RPI) {
      const int r = i + row0;
      f32x2 v = add2(load_pair(&sm.d[st][r][2 * cp]), bias), e = load_pair(&sm.x[st][r][2 * cp]);
      if (p.softplus) v = softplus2(v);
      if (z) {
        const f32x2 zz = load_pair(&sm.z[st][r][2 * cp]);
        e = mul2(e, mul2(zz, sigmoid2(zz)));
      }
      if (r >= nt) v = e = 0ull;
      *reinterpret_cast<f32x2*>(&sm.delta[r][2 * cp]) = v;
      *reinterpret_cast<f32x2*>(&sm.u[r][2 * cp]) = e;
    }
#pragma unroll
    for (int i = 0; i < kTile * NP / 2; i += 32) {
      const int r = (i + lane) / (NP / 2), n = (i + lane) % (NP / 2) * 2;
      const float e0 = r < nt && n < p.N ? to_f(sm.C[st][r][n]) : 0.f, e1 = r < nt && n + 1 < p.N ? to_f(sm.C[st][r][n + 1]) : 0.f;
      *reinterpret_cast<float4*>(&sm.C2[r][2 * n]) = make_float4(e0, e0, e1, e1);
    }
    __syncwarp();
    const auto walk = [&](auto usual) {
      for (int t = (nt - 1) & ~3; t >= 0; t -= 4) {
#pragma unroll
        for (int j = 3; j >= 0; --j) {  // rows behind the last token hold zeros: they leave the gradient as it is
          const ulonglong2 d2 = *reinterpret_cast<const ulonglong2*>(&sm.delta[t + j][4 * g]);
          const ulonglong2 e2 = *reinterpret_cast<const ulonglong2*>(&sm.u[t + j][4 * g]);
          const ulonglong2 ca = *reinterpret_cast<const ulonglong2*>(&sm.C2[t + j][8 * s]);
          const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&sm.C2[t + j][8 * s + 4]);
          const f32x2 cn[4] = {ca.x, ca.y, cc.x, cc.y};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            G.r[0][n] = mul2(decay2(d2.x, A2.r[0][n]), fma2(cn[n], e2.x, G.r[0][n]));
            G.r[1][n] = mul2(decay2(d2.y, A2.r[1][n]), fma2(cn[n], e2.y, G.r[1][n]));
          }
          if (!decltype(usual)::value) clear_padding(G, n0, p.N);
          sum0 = add2(sum0, d2.x);
          sum1 = add2(sum1, d2.y);
        }
      }
    };
    if (full)
      walk(std::true_type{});
    else
      walk(std::false_type{});
    __syncwarp();
  }
  copy_wait<0>();
  const long long per_chunk = static_cast<long long>(p.batch) * p.dim;
  float* totals = p.carry + (p.splits - 1) * per_chunk * p.N;
  store_lane(p.carry + ((q - 1) * per_chunk + b * p.dim) * p.N, G, c0, p.dim, n0, p.N);
  if (s == 0) {
    float t[4];
    unpack2(t[0], t[1], sum0);
    unpack2(t[2], t[3], sum1);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c0 + k < p.dim) totals[(q - 1) * per_chunk + b * p.dim + c0 + k] = t[k];
  }
}

template <class T, int SG>
__global__ void __launch_bounds__(BwdShape<SG>::kThreads) scan_backward_kernel(const ScanBwdParams bp) {
  using S = BwdTile<T, SG>;
  constexpr int WC = 128 / SG, NP = S::NP, CW = S::CW, NT = BwdShape<SG>::kThreads, CP = CW / 2, RPI = NT / CP;
  const ScanParams& p = bp.f;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  S& sm = *reinterpret_cast<S*>(smem_raw);
  grid_dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane / SG, s = lane % SG;
  const int cblocks = (p.dim + CW - 1) / CW;
  const int cb = blockIdx.x % cblocks;
  const int rest = blockIdx.x / cblocks;
  const int q = rest % p.splits;
  const long long b = rest / p.splits;
  const int cw = cb * CW, cl = warp * WC + 4 * g, c0 = cw + cl, n0 = 4 * s;  // cl: this lane's channels within the CTA's
  const int n_tok = tokens_of(p.lengths, b, p.L);
  const int first = q * p.chunk, end = min(p.L, first + p.chunk), live = min(end, n_tok);
  const int cols = min(CW, p.dim - cw);
  const bool full = p.N == NP;

  LaneState A2, G, dA;
  load_rates(A2, p.A, c0, p.dim, n0, p.N);
#pragma unroll
  for (int n = 0; n < 4; ++n) G.r[0][n] = G.r[1][n] = dA.r[0][n] = dA.r[1][n] = 0ull;
  const long long per_chunk = static_cast<long long>(p.batch) * p.dim;
  if (bp.dstate) load_lane(G, bp.dstate + b * p.dim * p.N, c0, p.dim, n0, p.N, 1.f);
  {
    const float* totals = p.carry + (p.splits - 1) * per_chunk * p.N;
    for (int k = p.splits - 1; k > q; --k) {
      LaneState last;
      f32x2 t0, t1;
      load_lane(last, p.carry + ((k - 1) * per_chunk + b * p.dim) * p.N, c0, p.dim, n0, p.N, 1.f);
      load_totals(t0, t1, totals + (k - 1) * per_chunk + b * p.dim, c0, p.dim);
      apply_chunk(G, A2, last, t0, t1);
    }
  }
  const int cp = tid % CP, row0 = tid / CP, pc = cw + 2 * cp;
  const f32x2 bias = channel_pair(p.bias, pc, p.dim), skip = channel_pair(p.D, pc, p.dim);
  f32x2 sum_d = 0ull, sum_b = 0ull;
  for (int i = tid; i < 2 * kTile * (CW - cols); i += NT) {  // channels that are not there: never copied, read as zeros
    const int at = i / (CW - cols) * CW + cols + i % (CW - cols);
    (&sm.x[0][0][0])[at] = (&sm.d[0][0][0])[at] = (&sm.z[0][0][0])[at] = (&sm.dy[0][0][0])[at] = from_f<T>(0.f);
  }
  const T* x = static_cast<const T*>(p.x) + b * p.x_b + cw;
  const T* dl = static_cast<const T*>(p.delta) + b * p.d_b + cw;
  const T* z = p.z ? static_cast<const T*>(p.z) + b * p.z_b + cw : nullptr;
  const T* Bm = static_cast<const T*>(p.B) + b * p.B_b;
  const T* Cm = static_cast<const T*>(p.C) + b * p.C_b;
  const long long dense = (b * p.L) * p.dim + cw;
  const T* dy = static_cast<const T*>(bp.dy) + dense;
  T* dx = static_cast<T*>(bp.dx) + dense;
  T* dd = static_cast<T*>(bp.ddelta) + dense;
  T* dz = z ? static_cast<T*>(bp.dz) + dense : nullptr;
  const auto load_tile = [&](int st, int t0) {
    const int rows = min(kTile, live - t0);
    fetch<T, kTile, CW, NT>(sm.x[st], x + t0 * p.x_t, p.x_t, rows, cols, p.al_x, tid);
    fetch<T, kTile, CW, NT>(sm.d[st], dl + t0 * p.d_t, p.d_t, rows, cols, p.al_d, tid);
    fetch<T, kTile, CW, NT>(sm.dy[st], dy + static_cast<long long>(t0) * p.dim, p.dim, rows, cols, bp.al_dy, tid);
    if (z) fetch<T, kTile, CW, NT>(sm.z[st], z + t0 * p.z_t, p.z_t, rows, cols, p.al_z, tid);
    fetch<T, kTile, NP, NT>(sm.B[st], Bm + t0 * p.B_t, p.B_t, rows, p.N, p.al_B, tid);
    fetch<T, kTile, NP, NT>(sm.C[st], Cm + t0 * p.C_t, p.C_t, rows, p.N, p.al_C, tid);
  };
  const long long ck_rows = (p.L + kCheckpoint - 1) / kCheckpoint;
  const int tiles = live > first ? (live - first + kTile - 1) / kTile : 0;
  if (tiles) load_tile(0, first + (tiles - 1) * kTile);
  copy_commit();
  int st = 0;
  for (int i_t = tiles - 1; i_t >= 0; --i_t, st ^= 1) {
    const int t0 = first + i_t * kTile, nt = min(kTile, live - t0);
    copy_wait<0>();
    __syncthreads();  // this tile has arrived everywhere; the tile before has been read to the end
    if (i_t) load_tile(st ^ 1, t0 - kTile);
    copy_commit();
    LaneState h;
    load_lane(h, p.checkpoints + (b * ck_rows + t0 / kCheckpoint) * p.dim * p.N, c0, p.dim, n0, p.N, 1.f);
#pragma unroll
    for (int i = 0; i < kTile; i += RPI) {
      const int r = i + row0;
      f32x2 v = add2(load_pair(&sm.d[st][r][2 * cp]), bias), e = load_pair(&sm.dy[st][r][2 * cp]);
      if (p.softplus) v = softplus2(v);
      f32x2 w = mul2(v, load_pair(&sm.x[st][r][2 * cp]));
      if (z) {
        const f32x2 zz = load_pair(&sm.z[st][r][2 * cp]);
        e = mul2(e, mul2(zz, sigmoid2(zz)));
      }
      if (r >= nt) v = w = e = 0ull;  // rows behind the last token: zeros leave the state and its gradient as they are
      *reinterpret_cast<f32x2*>(&sm.delta[r][2 * cp]) = v;
      *reinterpret_cast<f32x2*>(&sm.u[r][2 * cp]) = w;
      *reinterpret_cast<f32x2*>(&sm.gy[r][2 * cp]) = e;
    }
    for (int i = tid; i < kTile * NP / 2; i += NT) {
      const int r = i / (NP / 2), n = i % (NP / 2) * 2;
      const bool ok0 = r < nt && n < p.N, ok1 = r < nt && n + 1 < p.N;
      const float b0 = ok0 ? to_f(sm.B[st][r][n]) : 0.f, b1 = ok1 ? to_f(sm.B[st][r][n + 1]) : 0.f;
      const float e0 = ok0 ? to_f(sm.C[st][r][n]) : 0.f, e1 = ok1 ? to_f(sm.C[st][r][n + 1]) : 0.f;
      *reinterpret_cast<float4*>(&sm.B2[r][2 * n]) = make_float4(b0, b0, b1, b1);
      *reinterpret_cast<float4*>(&sm.C2[r][2 * n]) = make_float4(e0, e0, e1, e1);
    }
    __syncthreads();
    const int steps = (nt + kStep - 1) / kStep;
    LaneState dA_tile;
#pragma unroll
    for (int n = 0; n < 4; ++n) dA_tile.r[0][n] = dA_tile.r[1][n] = 0ull;
    const auto walk = [&](auto usual, auto gated) {
      constexpr bool kFull = decltype(usual)::value, kGate = decltype(gated)::value;
      // forward over the tile: park the state before each step of 4 tokens
      for (int k = 0; k < steps; ++k) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float4 v;
          unpack2(v.x, v.y, h.r[0][n]);
          unpack2(v.z, v.w, h.r[1][n]);
          sm.park[k][n][tid] = v;
        }
        if (k + 1 == steps) break;
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
          const int t = k * kStep + j;
          const ulonglong2 d2 = *reinterpret_cast<const ulonglong2*>(&sm.delta[t][cl]);
          const ulonglong2 u2 = *reinterpret_cast<const ulonglong2*>(&sm.u[t][cl]);
          const ulonglong2 ba = *reinterpret_cast<const ulonglong2*>(&sm.B2[t][8 * s]);
          const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B2[t][8 * s + 4]);
          const f32x2 bn[4] = {ba.x, ba.y, bb.x, bb.y};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            h.r[0][n] = fma2(decay2(d2.x, A2.r[0][n]), h.r[0][n], mul2(u2.x, bn[n]));
            h.r[1][n] = fma2(decay2(d2.y, A2.r[1][n]), h.r[1][n], mul2(u2.y, bn[n]));
          }
          if (!kFull) clear_padding(h, n0, p.N);
        }
      }
      for (int k = steps - 1; k >= 0; --k) {
        LaneState a[kStep], w[kStep];  // decays, decayed states before the token's own input
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float4 v = sm.park[k][n][tid];
          h.r[0][n] = pack2(v.x, v.y);
          h.r[1][n] = pack2(v.z, v.w);
        }
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
          const int t = k * kStep + j;
          const ulonglong2 d2 = *reinterpret_cast<const ulonglong2*>(&sm.delta[t][cl]);
          const ulonglong2 u2 = *reinterpret_cast<const ulonglong2*>(&sm.u[t][cl]);
          const ulonglong2 ba = *reinterpret_cast<const ulonglong2*>(&sm.B2[t][8 * s]);
          const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B2[t][8 * s + 4]);
          const f32x2 bn[4] = {ba.x, ba.y, bb.x, bb.y};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            a[j].r[0][n] = decay2(d2.x, A2.r[0][n]);
            a[j].r[1][n] = decay2(d2.y, A2.r[1][n]);
            w[j].r[0][n] = mul2(a[j].r[0][n], h.r[0][n]);
            w[j].r[1][n] = mul2(a[j].r[1][n], h.r[1][n]);
            h.r[0][n] = fma2(u2.x, bn[n], w[j].r[0][n]);
            h.r[1][n] = fma2(u2.y, bn[n], w[j].r[1][n]);
          }
          if (!kFull) {
            clear_padding(h, n0, p.N);
            clear_padding(w[j], n0, p.N);
          }
        }
        // the step's results stay in registers until its last token: a store in between would order the next token's loads behind it
        float oy[kStep][2], ou[kStep][2], ow[kStep][2];
        ChannelSums<SG> sums[kStep];
#pragma unroll
        for (int j = kStep - 1; j >= 0; --j) {
          const int t = k * kStep + j;
          const ulonglong2 d2 = *reinterpret_cast<const ulonglong2*>(&sm.delta[t][cl]);
          const ulonglong2 u2 = *reinterpret_cast<const ulonglong2*>(&sm.u[t][cl]);
          const ulonglong2 e2 = *reinterpret_cast<const ulonglong2*>(&sm.gy[t][cl]);
          const ulonglong2 ba = *reinterpret_cast<const ulonglong2*>(&sm.B2[t][8 * s]);
          const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(&sm.B2[t][8 * s + 4]);
          const ulonglong2 ca = *reinterpret_cast<const ulonglong2*>(&sm.C2[t][8 * s]);
          const ulonglong2 cc = *reinterpret_cast<const ulonglong2*>(&sm.C2[t][8 * s + 4]);
          const f32x2 bn[4] = {ba.x, ba.y, bb.x, bb.y}, cn[4] = {ca.x, ca.y, cc.x, cc.y};
          const f32x2 dp[2] = {d2.x, d2.y}, up[2] = {u2.x, u2.y}, ep[2] = {e2.x, e2.y};
          f32x2 y[2] = {}, du[2] = {}, wa[2] = {};
          float bc[8];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            f32x2 db = 0ull, dc = 0ull;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              f32x2 gg = fma2(cn[n], ep[c], G.r[c][n]);
              if (!kFull && n0 + n >= p.N) gg = 0ull;
              const f32x2 hh = fma2(up[c], bn[n], w[j].r[c][n]);
              if (kGate) y[c] = fma2(cn[n], hh, y[c]);
              dc = fma2(ep[c], hh, dc);
              db = fma2(gg, up[c], db);
              du[c] = fma2(gg, bn[n], du[c]);
              const f32x2 ww = mul2(gg, w[j].r[c][n]);
              dA_tile.r[c][n] = fma2(ww, dp[c], dA_tile.r[c][n]);
              wa[c] = fma2(ww, A2.r[c][n], wa[c]);
              G.r[c][n] = mul2(gg, a[j].r[c][n]);
            }
            bc[n] = lo2(db) + hi2(db);
            bc[4 + n] = lo2(dc) + hi2(dc);
          }
          sums[j] = reduce_channels<SG>(bc, lane);
          if (kGate) reduce_states<SG>(oy[j], y[0], y[1], s);
          reduce_states<SG>(ou[j], du[0], du[1], s);
          reduce_states<SG>(ow[j], wa[0], wa[1], s);
        }
        __syncwarp();  // all lanes have read the step's u and dy: their places take du and sum C h
        const int slot = channel_slot<SG>(lane, n0);
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
          const int t = k * kStep + j;
          if (SG > 2 || !(lane & 2)) {
#pragma unroll
            for (int i = 0; i < ChannelSums<SG>::kHeld; ++i) sm.red[warp][t][slot + i] = sums[j].v[i];
          }
          if (SG == 2) {
            if (kGate) *reinterpret_cast<float2*>(&sm.gy[t][cl + 2 * s]) = make_float2(oy[j][0], oy[j][1]);
            *reinterpret_cast<float2*>(&sm.u[t][cl + 2 * s]) = make_float2(ou[j][0], ou[j][1]);
            *reinterpret_cast<float2*>(&sm.wa[t][cl + 2 * s]) = make_float2(ow[j][0], ow[j][1]);
          } else if (SG == 4 || s < 4) {
            if (kGate) sm.gy[t][cl + (s & 3)] = oy[j][0];
            sm.u[t][cl + (s & 3)] = ou[j][0];
            sm.wa[t][cl + (s & 3)] = ow[j][0];
          }
        }
      }
    };
    if (full) {
      if (z)
        walk(std::true_type{}, std::true_type{});
      else
        walk(std::true_type{}, std::false_type{});
    } else {
      walk(std::false_type{}, std::true_type{});
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      dA.r[0][n] = add2(dA.r[0][n], dA_tile.r[0][n]);
      dA.r[1][n] = add2(dA.r[1][n], dA_tile.r[1][n]);
    }
    __syncthreads();
    f32x2 tile_d = 0ull, tile_b = 0ull;
#pragma unroll
    for (int i = 0; i < kTile; i += RPI) {
      const int r = i + row0, c = 2 * cp;
      if (r >= nt || pc >= p.dim) continue;
      const f32x2 xx = load_pair(&sm.x[st][r][c]), up = load_pair(&sm.dy[st][r][c]);
      const f32x2 du = *reinterpret_cast<const f32x2*>(&sm.u[r][c]), one = both(1.f);
      const long long at = static_cast<long long>(t0 + r) * p.dim + c;
      f32x2 e = up;
      if (z) {
        const f32x2 zz = load_pair(&sm.z[st][r][c]), sg = sigmoid2(zz);
        e = mul2(up, mul2(zz, sg));
        const f32x2 y0 = fma2(skip, xx, *reinterpret_cast<const f32x2*>(&sm.gy[r][c]));
        const f32x2 slope = mul2(sg, fma2(zz, fma2(sg, both(-1.f), one), one));
        store_pair<T>(dz + at, mul2(mul2(up, y0), slope), bp.al_out, p.dim - pc);
      }
      const f32x2 ox = fma2(du, *reinterpret_cast<const f32x2*>(&sm.delta[r][c]), mul2(e, skip));
      f32x2 v = fma2(du, xx, mul2(*reinterpret_cast<const f32x2*>(&sm.wa[r][c]), both(kLn2)));
      if (p.softplus) v = mul2(v, softplus_slope2(add2(load_pair(&sm.d[st][r][c]), bias)));
      store_pair<T>(dx + at, ox, bp.al_out, p.dim - pc);
      store_pair<T>(dd + at, v, bp.al_out, p.dim - pc);
      tile_d = fma2(e, xx, tile_d);
      tile_b = add2(tile_b, v);
    }
    sum_d = add2(sum_d, tile_d);
    sum_b = add2(sum_b, tile_b);
    float* bc = bp.partial_bc + ((cb * static_cast<long long>(p.batch) + b) * p.L + t0) * 2 * p.N;
    for (int i = tid; i < nt * 2 * NP; i += NT) {
      const int r = i / (2 * NP), j = i % (2 * NP), n = j % NP;
      if (n >= p.N) continue;
      float v = sm.red[0][r][j];
#pragma unroll
      for (int k = 1; k < BwdShape<SG>::kWarps; ++k) v += sm.red[k][r][j];
      bc[static_cast<long long>(r) * 2 * p.N + (j < NP ? 0 : p.N) + n] = v;
    }
  }
  copy_wait<0>();
  const float zero[2] = {};
  if (pc < p.dim)
    for (int t = max(first, live) + row0; t < end; t += RPI) {
      const long long at = static_cast<long long>(t) * p.dim + 2 * cp;
      store_run<T, 2>(dx + at, zero, bp.al_out, p.dim - pc);
      store_run<T, 2>(dd + at, zero, bp.al_out, p.dim - pc);
      if (z) store_run<T, 2>(dz + at, zero, bp.al_out, p.dim - pc);
    }
  float* par = bp.partial_par + (q * static_cast<long long>(p.batch) + b) * bp.par_pitch;
  store_lane(par, dA, c0, p.dim, n0, p.N);
  if (bp.dinitial && q == 0) store_lane(bp.dinitial + b * p.dim * p.N, G, c0, p.dim, n0, p.N);
  __syncthreads();
  // the threads of one channel pair add up their rows
  float* strip = &sm.delta[0][0];  // [RPI][CW] and again for the bias
  *reinterpret_cast<f32x2*>(&strip[row0 * CW + 2 * cp]) = sum_d;
  *reinterpret_cast<f32x2*>(&strip[(RPI + row0) * CW + 2 * cp]) = sum_b;
  __syncthreads();
  for (int c = tid; c < cols; c += NT) {
    float a = 0.f, e = 0.f;
#pragma unroll
    for (int r = 0; r < RPI; ++r) {
      a += strip[r * CW + c];
      e += strip[(RPI + r) * CW + c];
    }
    float* to = par + static_cast<long long>(p.dim) * p.N;
    to[cw + c] = a;
    to[p.dim + cw + c] = e;
  }
}

// dB, dC [B, L, N] from partial[blocks][B][L][2 N]; 0 from each sequence's end on, where nothing was written.
template <class T>
__global__ void __launch_bounds__(256) scan_bc_sum_kernel(const float* part, void* dB, void* dC, const int* lengths, int batch, int L, int N,
                                                          int blocks) {
  grid_dependency_wait();
  const long long total = static_cast<long long>(batch) * L * 2 * N;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= total) return;
  const long long row = i / (2 * N);
  const int j = static_cast<int>(i - row * 2 * N);
  const long long b = row / L;
  float v = 0.f;
  if (row - b * L < tokens_of(lengths, b, L))
#pragma unroll 4
    for (int k = 0; k < blocks; ++k) v += part[k * total + i];
  if (j < N)
    static_cast<T*>(dB)[row * N + j] = from_f<T>(v);
  else
    static_cast<T*>(dC)[row * N + j - N] = from_f<T>(v);
}

}  // namespace btp_scan
