// C entries of the root-mean-square norm: argument checks, launch shapes, launches.
#include "elem_host.cuh"
#include "norm_kernels.cuh"
#include "sum_kernels.cuh"

namespace {

using namespace btp_host;
using namespace btp_norm;

// How a row is dealt to threads.  One run of 8 columns per thread up to 2048 columns and where there are too few rows to fill the device
// (a row's latency is shortest then); two up to 8192 columns (fewer warps to add up), four beyond.  Measured: 16384 rows of 4096
// columns in 8 bits take 90 us with two and 95 with one, 16384 of 2048 with a float residual 69 with two and 62 with one.  A row of at
// most 32 threads' columns goes to one warp, which needs no barrier.
struct Shape {
  int vpt;
  bool warp_row;
  int threads;
  int grid;
};
Shape row_shape(long long rows, int dim, int sms, bool heavy) {
  Shape s{};
  s.vpt = dim > kMaxRowThreads * kRun * 2 ? 4 : dim > (rows < sms ? 4096 : 2048) ? 2 : 1;
  const int threads = (dim + kRun * s.vpt - 1) / (kRun * s.vpt);
  s.warp_row = threads <= 32;
  s.threads = s.warp_row ? 128 : (threads + 31) / 32 * 32;
  // as many CTAs as 1024 threads per SM give; each takes rows in turn and fetches one ahead
  const long long want = s.warp_row ? (rows + 3) / 4 : rows, cap = static_cast<long long>(sms) * (s.vpt == 4 && heavy ? 1 : 1024 / s.threads);  // see kCtas
  s.grid = static_cast<int>(want < cap ? want : cap);
  return s;
}
// Backward: one run of 8 columns per thread up to 4096 columns (the weight and its gradient stay in registers besides the row), as many
// CTAs as 1024 threads per SM give (measured best of 512 ... 2048); every one keeps its share of the weight's gradient for all its rows.
Shape backward_shape(int dim) {
  Shape s{};
  s.vpt = dim <= kMaxRowThreads * kRun ? 1 : dim <= kMaxRowThreads * kRun * 2 ? 2 : 4;
  const int threads = (dim + kRun * s.vpt - 1) / (kRun * s.vpt);
  s.warp_row = threads <= 32;
  s.threads = s.warp_row ? 128 : (threads + 31) / 32 * 32;
  return s;
}
int backward_grid(long long rows, const Shape& s, int sms) {
  const int fit = (s.vpt == 1 ? 1024 : 512) / s.threads;
  const long long want = s.warp_row ? (rows + 3) / 4 : rows;
  const long long cap = static_cast<long long>(sms) * (fit > 0 ? fit : 1);
  return static_cast<int>(want < cap ? want : cap);
}

template <class T, int RES, int OUT, int VPT>
cudaError_t launch_fwd(const FwdParams& p, const Shape& s, cudaStream_t stream) {
  if constexpr (VPT == 1)  // a row of one warp has one run per thread
    if (s.warp_row) return launch_kernel(rms_norm_forward_kernel<T, RES, OUT, VPT, true>, s.grid, 128, 0, stream, p);
  return launch_kernel(rms_norm_forward_kernel<T, RES, OUT, VPT, false>, s.grid, s.threads, 0, stream, p);
}
template <class T, int RES, int OUT>
cudaError_t launch_fwd_v(const FwdParams& p, const Shape& s, cudaStream_t stream) {
  return s.vpt == 1 ? launch_fwd<T, RES, OUT, 1>(p, s, stream) : s.vpt == 2 ? launch_fwd<T, RES, OUT, 2>(p, s, stream) : launch_fwd<T, RES, OUT, 4>(p, s, stream);
}
template <class T, int RES>
cudaError_t launch_fwd_o(const FwdParams& p, const Shape& s, int out, cudaStream_t stream) {
  return out == kSame ? launch_fwd_v<T, RES, kSame>(p, s, stream)
                      : out == kRow8 ? launch_fwd_v<T, RES, kRow8>(p, s, stream) : launch_fwd_v<T, RES, kBlock8>(p, s, stream);
}
template <class T, int RES, int VPT>
cudaError_t launch_bwd(const BwdParams& p, const Shape& s, int grid, cudaStream_t stream) {
  if constexpr (VPT == 1)
    if (s.warp_row) return launch_kernel(rms_norm_backward_kernel<T, RES, VPT, true>, grid, 128, 0, stream, p);
  return launch_kernel(rms_norm_backward_kernel<T, RES, VPT, false>, grid, s.threads, 0, stream, p);
}
template <class T, int RES>
cudaError_t launch_bwd_v(const BwdParams& p, const Shape& s, int grid, cudaStream_t stream) {
  return s.vpt == 1 ? launch_bwd<T, RES, 1>(p, s, grid, stream) : s.vpt == 2 ? launch_bwd<T, RES, 2>(p, s, grid, stream) : launch_bwd<T, RES, 4>(p, s, grid, stream);
}

int check_rows(const char* fn, long long rows, int dim, int dtype) {
  if (rows <= 0 || dim <= 0) return fail(BTP_ERR_BAD_SHAPE, "%s: rows and dim must be positive (got %lld, %d)", fn, rows, dim);
  if (rows > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: %lld rows exceed the 2^31-1 limit", fn, rows);
  if (dim > kMaxDim) return fail(BTP_ERR_BAD_SHAPE, "%s: dim must be at most %d (got %d)", fn, kMaxDim, dim);
  if (!known_dtype(dtype)) return fail(BTP_ERR_BAD_DTYPE, "%s: unknown dtype tag %d", fn, dtype);
  return BTP_OK;
}

}  // namespace

extern "C" {

int btp_sm100_rms_norm_forward(const void* x, const void* residual, const void* weight, void* y, void* h, float* rstd,
                               float* scale, long long rows, int dim, long long ld_x, long long ld_r, float eps, int dtype,
                               int residual_dtype, int weight_dtype, int out_mode, void* stream) {
  const char* fn = "btp_sm100_rms_norm_forward";
  int rc = check_rows(fn, rows, dim, dtype);
  if (rc) return rc;
  if (out_mode < 0 || out_mode > 2) return fail(BTP_ERR_BAD_ORDER, "%s: out_mode must be 0, 1 or 2 (got %d)", fn, out_mode);
  if (!x || !y || (residual && !h) || (out_mode && !scale))
    return fail(BTP_ERR_NULL_POINTER, "%s: x, y, h (with a residual) and scale (with 8-bit output) must not be NULL", fn);
  if (residual && residual_dtype != dtype && residual_dtype != BTP_DTYPE_F32)
    return fail(BTP_ERR_BAD_DTYPE, "%s: the residual must have x's type or be float32", fn);
  if (weight && weight_dtype != dtype && weight_dtype != BTP_DTYPE_F32)
    return fail(BTP_ERR_BAD_DTYPE, "%s: the weight must have x's type or be float32", fn);
  if (ld_x < dim || (residual && ld_r < dim)) return fail(BTP_ERR_BAD_SHAPE, "%s: a row pitch is smaller than its row", fn);
  if (!(eps >= 0.f)) return fail(BTP_ERR_BAD_SHAPE, "%s: eps must not be negative", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  const Shape s = row_shape(rows, dim, info.sms, residual || dtype == BTP_DTYPE_F32);
  const int e = elem_bytes(dtype), er = residual ? elem_bytes(residual_dtype) : e;
  FwdParams p{};
  p.x = x; p.residual = residual; p.weight = weight; p.y = y; p.h = h; p.rstd = rstd; p.scale = scale;
  p.rows = rows; p.ld_x = ld_x; p.ld_r = ld_r; p.dim = dim; p.eps = eps;
  p.weight_f32 = weight && weight_dtype == BTP_DTYPE_F32;
  p.al_x = aligned16(x) && (ld_x * e) % 16 == 0;
  p.al_r = residual && aligned16(residual) && (ld_r * er) % 16 == 0;
  p.al_w = weight && aligned16(weight);
  p.al_out = aligned16(y) && (!h || aligned16(h)) && dim % kRun == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int res = !residual ? kNone : (residual_dtype == dtype ? kResSame : kResF32);
  return launched(fn, by_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (res == kNone) return launch_fwd_o<T, kNone>(p, s, out_mode, st);
    if constexpr (sizeof(T) == 2)
      if (res == kResF32) return launch_fwd_o<T, kResF32>(p, s, out_mode, st);
    return launch_fwd_o<T, kResSame>(p, s, out_mode, st);
  }));
}

int btp_sm100_rms_norm_partial_rows(long long rows, int dim) {
  const char* fn = "btp_sm100_rms_norm_partial_rows";
  int rc = check_rows(fn, rows, dim, BTP_DTYPE_F32);
  if (rc) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  const Shape s = backward_shape(dim);
  return backward_grid(rows, s, info.sms) * (s.warp_row ? 4 : 1);
}

int btp_sm100_rms_norm_backward(const void* h, const void* weight, const void* dy, const void* dh, const float* rstd, void* dx,
                                void* dresidual, void* dweight, float* partial, long long rows, int dim, long long ld_h,
                                int dtype, int residual_dtype, int weight_dtype, void* stream) {
  const char* fn = "btp_sm100_rms_norm_backward";
  int rc = check_rows(fn, rows, dim, dtype);
  if (rc) return rc;
  if (!h || !dy || !rstd) return fail(BTP_ERR_NULL_POINTER, "%s: h, dy and rstd must not be NULL", fn);
  if (dweight && (!weight || !partial)) return fail(BTP_ERR_NULL_POINTER, "%s: dweight needs the weight and the partial sums", fn);
  if (residual_dtype != dtype && residual_dtype != BTP_DTYPE_F32)
    return fail(BTP_ERR_BAD_DTYPE, "%s: the residual must have x's type or be float32", fn);
  if (weight && weight_dtype != dtype && weight_dtype != BTP_DTYPE_F32)
    return fail(BTP_ERR_BAD_DTYPE, "%s: the weight must have x's type or be float32", fn);
  if (ld_h < dim) return fail(BTP_ERR_BAD_SHAPE, "%s: a row pitch is smaller than its row", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  const Shape s = backward_shape(dim);
  const int grid = backward_grid(rows, s, info.sms);
  BwdParams p{};
  p.h = h; p.weight = weight; p.dy = dy; p.dh = dh; p.rstd = rstd; p.dx = dx; p.dres = dresidual;
  p.partial = dweight ? partial : nullptr;
  p.rows = rows; p.ld_h = ld_h; p.dim = dim;
  p.weight_f32 = weight && weight_dtype == BTP_DTYPE_F32;
  p.al_h = aligned16(h) && (ld_h * elem_bytes(residual_dtype)) % 16 == 0;
  p.al_w = weight && aligned16(weight);
  p.al_dense = dim % kRun == 0 && aligned16(dy) && (!dh || aligned16(dh)) && (!dx || aligned16(dx)) && (!dresidual || aligned16(dresidual)) &&
               (!partial || aligned16(partial));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = launched(fn, by_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    if constexpr (sizeof(T) == 2)
      if (residual_dtype != dtype) return launch_bwd_v<T, kResF32>(p, s, grid, st);
    return launch_bwd_v<T, kResSame>(p, s, grid, st);
  }));
  if (rc || !dweight) return rc;
  const int parts = grid * (s.warp_row ? 4 : 1);
  return launched(fn, by_type(dtype, [&](auto tag) {
    return launch_kernel(column_sum_kernel<decltype(tag), 32>, (dim + 31) / 32, 1024, 0, st, static_cast<const float*>(partial), dweight,
                         parts, static_cast<long long>(dim), p.weight_f32);
  }));
}

}  // extern "C"
