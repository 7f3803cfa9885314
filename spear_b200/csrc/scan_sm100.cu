// C entries of the selective scan: argument checks, launch shapes, launches.
#include "elem_host.cuh"
#include "scan_bwd_kernels.cuh"
#include "scan_kernels.cuh"
#include "sum_kernels.cuh"

namespace {

using namespace btp_host;
using namespace btp_scan;

// State groups per warp: 4 states each, so 8, 16, 32 or 64 states; fewer are padded.
int state_groups(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

struct Split {
  int splits;
  int chunk;
};
// Chunks that the tokens are split into, by a model of the time in cycles.  With w warps on the fullest scheduler a token takes
// 60 + 112 w cycles (measured 285 at w = 2, 1570 at w = 14), in the pass for the carries 60 + 75 w; every chunk before its own costs a
// warp about 300 cycles.  So a split pays where one pass leaves schedulers with one or two warps over a long stretch.
Split split_tokens(long long batch, int L, int dim, int N, int sms) {
  const int wc = 64 / state_groups(N);
  const long long units = batch * ((dim + wc - 1) / wc), schedulers = static_cast<long long>(sms) * 4;
  const auto warps = [&](long long n) { return static_cast<double>((n + schedulers - 1) / schedulers); };
  Split best{};
  double best_cost = 0;
  for (int s = 1; s <= 256; s = s < 4 ? s + 1 : s * 5 / 4) {
    const int chunk = ((L + s - 1) / s + 31) / 32 * 32;
    if (s > 1 && chunk < 64) break;
    const int n = (L + chunk - 1) / chunk;
    double cost = (60 + 112 * warps(units * n)) * (chunk + 16);
    if (n > 1) cost += (60 + 75 * warps(units * (n - 1))) * (chunk + 16) + 300.0 * n + 8000;
    if (s == 1 || cost < best_cost) {
      best_cost = cost;
      best = Split{n, chunk};
    }
  }
  return best;
}

// The same for the backward, whose CTAs of four warps (two per SM: registers and shared memory) take about 2.6 times as long per token as
// a pass for the carries, which splitting adds.  Measured at 8 x 2048 tokens x 2048 channels x 16 states, main pass and carries: one
// chunk 1373 us, 2 chunks 875 + 196, 4 chunks 877 + 167, 16 chunks (the rule's choice) 800 + 180, all in bfloat16.  In float one CTA
// fits an SM, which the rule does not take into account.
Split split_backward(long long batch, int L, int dim, int N, int sms) {
  const int sg = state_groups(N), wc = 128 / sg, cw = (sg == 2 ? 2 : 4) * wc;
  const long long ctas = batch * ((dim + cw - 1) / cw), warps = batch * ((dim + wc - 1) / wc);
  const long long slots = static_cast<long long>(sms) * 2, wslots = static_cast<long long>(sms) * 8;
  Split best{1, (L + 31) / 32 * 32};
  double best_cost = static_cast<double>((ctas + slots - 1) / slots) * 2.6 * best.chunk;
  for (int s = 2; s <= 256; s = s * 3 / 2 + (s == 2)) {
    const int chunk = ((L + s - 1) / s + 31) / 32 * 32;
    if (chunk < 64) break;
    const int n = (L + chunk - 1) / chunk;
    if (n < 2) continue;
    const double main = static_cast<double>((ctas * n + slots - 1) / slots) * 2.6 * (chunk + 16);
    const double carry = static_cast<double>((warps * (n - 1) + wslots - 1) / wslots) * (chunk + 24);
    const double cost = main + carry + n * 4.0;
    if (cost < best_cost) {
      best_cost = cost;
      best = Split{n, chunk};
    }
  }
  return best;
}

// The backward's buffer: carries and their sums of step sizes, partial dB and dC, partial dA, dD and dbias.
struct BwdBuffer {
  long long bc, par, total, pitch;  // offsets in floats; pitch of a row of parameter sums
  int blocks;
};
BwdBuffer backward_buffer(const Split& s, long long B, long long L, long long dim, int N) {
  const int sg = state_groups(N), cw = (sg == 2 ? 2 : 4) * 128 / sg;
  const auto round4 = [](long long n) { return (n + 3) / 4 * 4; };
  BwdBuffer w{};
  w.blocks = static_cast<int>((dim + cw - 1) / cw);
  w.bc = round4((s.splits - 1) * B * dim * (N + 1));
  w.par = w.bc + round4(w.blocks * B * L * 2 * N);
  w.pitch = round4(dim * (N + 2));
  w.total = w.par + s.splits * B * w.pitch;
  return w;
}

int check(const char* fn, long long B, int L, int dim, int N, int dtype) {
  if (B <= 0 || L <= 0 || dim <= 0) return fail(BTP_ERR_BAD_SHAPE, "%s: B, L and dim must be positive (got %lld, %d, %d)", fn, B, L, dim);
  if (N < 1 || N > 64) return fail(BTP_ERR_BAD_SHAPE, "%s: the number of states must be in 1 ... 64 (got %d)", fn, N);
  if (L > (1 << 30)) return fail(BTP_ERR_BAD_SHAPE, "%s: L exceeds the 2^30 limit", fn);
  if (!known_dtype(dtype)) return fail(BTP_ERR_BAD_DTYPE, "%s: unknown dtype tag %d", fn, dtype);
  return BTP_OK;
}

// f(value of the type, state groups)
template <class F>
cudaError_t dispatch(int dtype, int N, F&& f) {
  return by_type(dtype, [&](auto tag) {
    switch (state_groups(N)) {
      case 2: return f(tag, std::integral_constant<int, 2>{});
      case 4: return f(tag, std::integral_constant<int, 4>{});
      case 8: return f(tag, std::integral_constant<int, 8>{});
      default: return f(tag, std::integral_constant<int, 16>{});
    }
  });
}

bool copies16(const void* p, long long sb, long long st, int e, int cols) {
  return aligned16(p) && (sb * e) % 16 == 0 && (st * e) % 16 == 0 && (cols * e) % 16 == 0;
}

}  // namespace

extern "C" {

long long btp_sm100_scan_carry_floats(int B, int L, int dim, int N) {
  const char* fn = "btp_sm100_scan_carry_floats";
  int rc = check(fn, B, L, dim, N, BTP_DTYPE_F32);
  if (rc) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  const Split s = split_tokens(B, L, dim, N, info.sms);
  return static_cast<long long>(s.splits - 1) * B * dim * (N + 1);
}

int btp_sm100_scan_forward(const void* x, const void* delta, const float* A, const void* Bm, const void* Cm, const float* D,
                           const void* z, const float* delta_bias, const float* initial, const int* lengths, void* y, float* state,
                           float* checkpoints, float* carry, int B, int L, int dim, int N, long long x_b, long long x_t,
                           long long d_b, long long d_t, long long B_b, long long B_t, long long C_b, long long C_t, long long z_b,
                           long long z_t, int delta_softplus, int dtype, void* stream) {
  const char* fn = "btp_sm100_scan_forward";
  int rc = check(fn, B, L, dim, N, dtype);
  if (rc) return rc;
  if (!x || !delta || !A || !Bm || !Cm || !y) return fail(BTP_ERR_NULL_POINTER, "%s: x, delta, A, B, C and y must not be NULL", fn);
  if (x_b < 0 || x_t < 0 || d_b < 0 || d_t < 0 || B_b < 0 || B_t < 0 || C_b < 0 || C_t < 0 || z_b < 0 || z_t < 0)
    return fail(BTP_ERR_BAD_SHAPE, "%s: strides must not be negative", fn);
  for (const void* q : {static_cast<const void*>(A), static_cast<const void*>(initial), static_cast<const void*>(state),
                        static_cast<const void*>(checkpoints), static_cast<const void*>(carry)})
    if (q && !aligned16(q)) return fail(BTP_ERR_MISALIGNED, "%s: A and the float states must be 16-byte aligned", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  const Split s = split_tokens(B, L, dim, N, info.sms);
  if (s.splits > 1 && !carry) return fail(BTP_ERR_NULL_POINTER, "%s: this shape needs the carry buffer", fn);
  const int e = elem_bytes(dtype);
  ScanParams p{};
  p.x = x; p.delta = delta; p.B = Bm; p.C = Cm; p.z = z; p.A = A; p.D = D; p.bias = delta_bias; p.initial = initial; p.lengths = lengths;
  p.y = y; p.state = state; p.checkpoints = checkpoints; p.carry = carry;
  p.x_b = x_b; p.x_t = x_t; p.d_b = d_b; p.d_t = d_t; p.z_b = z_b; p.z_t = z_t; p.B_b = B_b; p.B_t = B_t; p.C_b = C_b; p.C_t = C_t;
  p.batch = B; p.L = L; p.dim = dim; p.N = N; p.splits = s.splits; p.chunk = s.chunk; p.softplus = delta_softplus != 0;
  p.al_x = copies16(x, x_b, x_t, e, dim);
  p.al_d = copies16(delta, d_b, d_t, e, dim);
  p.al_z = z && copies16(z, z_b, z_t, e, dim);
  p.al_B = copies16(Bm, B_b, B_t, e, N);
  p.al_C = copies16(Cm, C_b, C_t, e, N);
  const int wc = 64 / state_groups(N);
  const long long per_split = static_cast<long long>(B) * ((dim + wc - 1) / wc);
  if (per_split * s.splits > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto run = [&](auto tag, auto groups, auto carry_pass) {
    using T = decltype(tag);
    constexpr int SG = decltype(groups)::value;
    constexpr bool kCarry = decltype(carry_pass)::value;
    static_assert(sizeof(FwdTile<T, SG>) <= 48 * 1024, "fits without a larger limit");
    return launch_kernel(scan_forward_kernel<T, SG, kCarry>, static_cast<int>(per_split * (kCarry ? s.splits - 1 : s.splits)), 32,
                         static_cast<int>(sizeof(FwdTile<T, SG>)), st, p);
  };
  if (s.splits > 1) {
    rc = launched(fn, dispatch(dtype, N, [&](auto tag, auto groups) { return run(tag, groups, std::true_type{}); }));
    if (rc) return rc;
  }
  return launched(fn, dispatch(dtype, N, [&](auto tag, auto groups) { return run(tag, groups, std::false_type{}); }));
}

long long btp_sm100_scan_backward_floats(int B, int L, int dim, int N) {
  const char* fn = "btp_sm100_scan_backward_floats";
  int rc = check(fn, B, L, dim, N, BTP_DTYPE_F32);
  if (rc) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  return backward_buffer(split_backward(B, L, dim, N, info.sms), B, L, dim, N).total;
}

int btp_sm100_scan_backward(const void* x, const void* delta, const float* A, const void* Bm, const void* Cm, const float* D,
                            const void* z, const float* delta_bias, const int* lengths, const float* checkpoints, const void* dy,
                            const float* dstate, void* dx, void* ddelta, float* dparams, void* dB, void* dC, void* dz,
                            float* dinitial, float* buffer, int B, int L, int dim, int N, long long x_b, long long x_t, long long d_b,
                            long long d_t, long long B_b, long long B_t, long long C_b, long long C_t, long long z_b, long long z_t,
                            int delta_softplus, int dtype, void* stream) {
  const char* fn = "btp_sm100_scan_backward";
  int rc = check(fn, B, L, dim, N, dtype);
  if (rc) return rc;
  if (!x || !delta || !A || !Bm || !Cm || !checkpoints || !dy || !dx || !ddelta || !dparams || !dB || !dC || (z && !dz) || !buffer)
    return fail(BTP_ERR_NULL_POINTER, "%s: only D, z with dz, delta_bias, lengths, dstate and dinitial may be NULL", fn);
  if (x_b < 0 || x_t < 0 || d_b < 0 || d_t < 0 || B_b < 0 || B_t < 0 || C_b < 0 || C_t < 0 || z_b < 0 || z_t < 0)
    return fail(BTP_ERR_BAD_SHAPE, "%s: strides must not be negative", fn);
  for (const void* q : {static_cast<const void*>(A), static_cast<const void*>(checkpoints), static_cast<const void*>(dstate),
                        static_cast<const void*>(dinitial), static_cast<const void*>(buffer)})
    if (q && !aligned16(q)) return fail(BTP_ERR_MISALIGNED, "%s: A, the float states and the buffer must be 16-byte aligned", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  const Split s = split_backward(B, L, dim, N, info.sms);
  const BwdBuffer w = backward_buffer(s, B, L, dim, N);
  const int e = elem_bytes(dtype);
  ScanBwdParams bp{};
  ScanParams& p = bp.f;
  p.x = x; p.delta = delta; p.B = Bm; p.C = Cm; p.z = z; p.A = A; p.D = D; p.bias = delta_bias; p.lengths = lengths;
  p.checkpoints = const_cast<float*>(checkpoints); p.carry = buffer;
  p.x_b = x_b; p.x_t = x_t; p.d_b = d_b; p.d_t = d_t; p.z_b = z_b; p.z_t = z_t; p.B_b = B_b; p.B_t = B_t; p.C_b = C_b; p.C_t = C_t;
  p.batch = B; p.L = L; p.dim = dim; p.N = N; p.splits = s.splits; p.chunk = s.chunk; p.softplus = delta_softplus != 0;
  p.al_x = copies16(x, x_b, x_t, e, dim);
  p.al_d = copies16(delta, d_b, d_t, e, dim);
  p.al_z = z && copies16(z, z_b, z_t, e, dim);
  p.al_B = copies16(Bm, B_b, B_t, e, N);
  p.al_C = copies16(Cm, C_b, C_t, e, N);
  bp.dy = dy; bp.dstate = dstate; bp.dx = dx; bp.ddelta = ddelta; bp.dz = dz; bp.dinitial = dinitial;
  bp.partial_bc = buffer + w.bc; bp.partial_par = buffer + w.par; bp.par_pitch = w.pitch;
  bp.al_dy = aligned16(dy) && (static_cast<long long>(dim) * e) % 16 == 0;
  bp.al_out = dim % 2 == 0 && aligned16(dx) && aligned16(ddelta) && (!z || aligned16(dz));
  const int wc = 128 / state_groups(N);
  const long long ctas = static_cast<long long>(B) * w.blocks * s.splits;
  const long long warps = static_cast<long long>(B) * ((dim + wc - 1) / wc) * (s.splits - 1);
  const long long bc_ctas = (static_cast<long long>(B) * L * 2 * N + 255) / 256;
  const long long cols = w.pitch;
  if (ctas > 0x7fffffffll || warps > 0x7fffffffll || bc_ctas > 0x7fffffffll || cols > 0x7fffffffll)
    return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s.splits > 1) {
    rc = launched(fn, dispatch(dtype, N, [&](auto tag, auto groups) {
      using T = decltype(tag);
      constexpr int SG = decltype(groups)::value;
      static_assert(sizeof(Tile<T, SG>) <= 48 * 1024, "fits without a larger limit");
      return launch_kernel(scan_backward_carry_kernel<T, SG>, static_cast<int>(warps), 32, static_cast<int>(sizeof(Tile<T, SG>)), st, bp);
    }));
    if (rc) return rc;
  }
  rc = launched(fn, dispatch(dtype, N, [&](auto tag, auto groups) {
    using T = decltype(tag);
    constexpr int SG = decltype(groups)::value;
    constexpr int kSmem = static_cast<int>(sizeof(BwdTile<T, SG>));
    static_assert(kSmem <= 227 * 1024, "the tile must fit into shared memory");
    // per device and process: the same value every time, so a race of two threads is harmless
    const cudaError_t err = cudaFuncSetAttribute(scan_backward_kernel<T, SG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err != cudaSuccess) return err;
    return launch_kernel(scan_backward_kernel<T, SG>, static_cast<int>(ctas), BwdShape<SG>::kThreads, kSmem, st, bp);
  }));
  if (rc) return rc;
  rc = launched(fn, by_type(dtype, [&](auto tag) {
    return launch_kernel(scan_bc_sum_kernel<decltype(tag)>, static_cast<int>(bc_ctas), 256, 0, st,
                         static_cast<const float*>(bp.partial_bc), dB, dC, lengths, B, L, N, w.blocks);
  }));
  if (rc) return rc;
  return launched(fn, launch_kernel(column_sum_kernel<float, 8>, static_cast<int>((cols + 31) / 32), 256, 0, st,
                                    static_cast<const float*>(bp.partial_par), static_cast<void*>(dparams), s.splits * B, cols, true));
}

int btp_sm100_scan_step(const void* x, const void* delta, const float* A, const void* Bm, const void* Cm, const float* D,
                        const void* z, const float* delta_bias, const float* state, void* y, float* state_out, int B, int dim, int N,
                        long long ld_x, long long ld_d, long long ld_B, long long ld_C, long long ld_z, int delta_softplus, int dtype,
                        void* stream) {
  const char* fn = "btp_sm100_scan_step";
  int rc = check(fn, B, 1, dim, N, dtype);
  if (rc) return rc;
  if (!x || !delta || !A || !Bm || !Cm || !state || !y || !state_out)
    return fail(BTP_ERR_NULL_POINTER, "%s: x, delta, A, B, C, state, y and state_out must not be NULL", fn);
  if (ld_x < 0 || ld_d < 0 || ld_B < 0 || ld_C < 0 || ld_z < 0) return fail(BTP_ERR_BAD_SHAPE, "%s: strides must not be negative", fn);
  if (!aligned16(A) || !aligned16(state) || !aligned16(state_out))
    return fail(BTP_ERR_MISALIGNED, "%s: A and the states must be 16-byte aligned", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  ScanStepParams p{};
  p.x = x; p.delta = delta; p.B = Bm; p.C = Cm; p.z = z; p.A = A; p.D = D; p.bias = delta_bias; p.state = state; p.state_out = state_out; p.y = y;
  p.ld_x = ld_x; p.ld_d = ld_d; p.ld_z = ld_z; p.ld_B = ld_B; p.ld_C = ld_C;
  p.batch = B; p.dim = dim; p.N = N; p.softplus = delta_softplus != 0;
  const auto quads = [&](const void* q, long long ld) {
    return N % 4 == 0 && ld % 4 == 0 && (reinterpret_cast<uintptr_t>(q) & static_cast<uintptr_t>(4 * elem_bytes(dtype) - 1)) == 0;
  };
  p.al_B = quads(Bm, ld_B);
  p.al_C = quads(Cm, ld_C);
  const long long over = (static_cast<long long>(dim) * state_groups(N) + 127) / 128;
  const long long ctas = over * ((B + kStepBatch - 1) / kStepBatch);
  p.ctas = static_cast<int>(over);
  if (ctas > 0x7fffffffll || static_cast<long long>(dim) * 16 > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launched(fn, dispatch(dtype, N, [&](auto tag, auto groups) {
    return launch_kernel(scan_step_kernel<decltype(tag), decltype(groups)::value>, static_cast<int>(ctas), 128, 0, st, p);
  }));
}

}  // extern "C"
