// C entries of the short causal convolution: argument checks, launch shapes, launches.
#include "conv_kernels.cuh"
#include "elem_host.cuh"

#include <initializer_list>

namespace {

using namespace btp_host;
using namespace btp_conv;

constexpr int kStepChannels = 4;  // per thread of the step

// Tokens per CTA: whole tiles, as many as leave the device about `per_sm` CTAs per SM (each reads W-1 tokens of its neighbour's run
// again and fills its ring anew); at least 4 tiles.
int tokens_per_run(long long B, int L, int dim, int sms, int per_sm) {
  const long long cblocks = (dim + kCols - 1) / kCols, slots = static_cast<long long>(sms) * per_sm;
  long long runs = slots / (B * cblocks);
  if (runs < 1) runs = 1;
  long long run = ((L + runs - 1) / runs + kTile - 1) / kTile * kTile;
  if (run < 4 * kTile) run = 4 * kTile;
  return static_cast<int>(run);
}
constexpr int kForwardCtas = 20, kBackwardCtas = 8;  // per SM; measured best of 10 ... 40 and 6 ... 16

int check(const char* fn, long long B, int L, int dim, int width, int dtype, int weight_dtype) {
  if (B <= 0 || L <= 0 || dim <= 0) return fail(BTP_ERR_BAD_SHAPE, "%s: B, L and dim must be positive (got %lld, %d, %d)", fn, B, L, dim);
  if (B > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: B exceeds the 2^31-1 limit", fn);
  if (L > (1 << 30)) return fail(BTP_ERR_BAD_SHAPE, "%s: L exceeds the 2^30 limit", fn);
  if (width < 2 || width > 4) return fail(BTP_ERR_BAD_ORDER, "%s: width must be 2, 3 or 4 (got %d)", fn, width);
  if (!known_dtype(dtype)) return fail(BTP_ERR_BAD_DTYPE, "%s: unknown dtype tag %d", fn, dtype);
  if (weight_dtype != dtype && weight_dtype != BTP_DTYPE_F32)
    return fail(BTP_ERR_BAD_DTYPE, "%s: weight and bias must have x's type or be float32", fn);
  return BTP_OK;
}

// Whether `n` channels are one word everywhere: rows `dim` and the given strides apart, from each of the pointers.
bool one_word(int n, int e, int dim, long long sb, long long st, std::initializer_list<const void*> ptrs) {
  if (dim % n || sb % n || st % n) return false;
  for (const void* q : ptrs)
    if (q && (reinterpret_cast<uintptr_t>(q) & static_cast<uintptr_t>(n * e - 1))) return false;
  return true;
}
// f(value of the type, taps)
template <class F>
cudaError_t dispatch(int dtype, int width, F&& f) {
  return by_type(dtype, [&](auto tag) {
    if (width == 2) return f(tag, std::integral_constant<int, 2>{});
    if (width == 3) return f(tag, std::integral_constant<int, 3>{});
    return f(tag, std::integral_constant<int, 4>{});
  });
}

}  // namespace

extern "C" {

int btp_sm100_causal_conv_forward(const void* x, const void* weight, const void* bias, const void* initial, const int* lengths,
                                  void* y, void* state, int B, int L, int dim, int width, long long sx_b, long long sx_t, int silu,
                                  int dtype, int weight_dtype, void* stream) {
  const char* fn = "btp_sm100_causal_conv_forward";
  int rc = check(fn, B, L, dim, width, dtype, weight_dtype);
  if (rc) return rc;
  if (!x || !weight || !y) return fail(BTP_ERR_NULL_POINTER, "%s: x, weight and y must not be NULL", fn);
  if (sx_b < 0 || sx_t < 0) return fail(BTP_ERR_BAD_SHAPE, "%s: strides must not be negative", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  ConvParams p{};
  const int e = elem_bytes(dtype);
  p.aligned = one_word(2, e, dim, sx_b, sx_t, {x, y, initial, state});
  p.copies = one_word(16 / e, e, dim, sx_b, sx_t, {x});
  p.whole_w = aligned16(weight);
  p.x = x; p.weight = weight; p.bias = bias; p.initial = initial; p.lengths = lengths; p.y = y; p.state = state;
  p.sx_b = sx_b; p.sx_t = sx_t; p.B = B; p.L = L; p.dim = dim; p.silu = silu != 0; p.weight_f32 = weight_dtype == BTP_DTYPE_F32;
  p.run = tokens_per_run(B, L, dim, info.sms, kForwardCtas);
  p.runs = (L + p.run - 1) / p.run;
  const long long ctas = static_cast<long long>(B) * p.runs * ((dim + kCols - 1) / kCols);
  if (ctas > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launched(fn, dispatch(dtype, width, [&](auto tag, auto taps) {
    using T = decltype(tag);
    constexpr int W = decltype(taps)::value;
    return launch_kernel(conv_forward_kernel<T, W>, static_cast<int>(ctas), kThreads, static_cast<int>(sizeof(ConvTile<T, 1>)), st, p);
  }));
}

int btp_sm100_causal_conv_partial_rows(int B, int L, int dim) {
  const char* fn = "btp_sm100_causal_conv_partial_rows";
  int rc = check(fn, B, L, dim, 4, BTP_DTYPE_F32, BTP_DTYPE_F32);
  if (rc) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  const int run = tokens_per_run(B, L, dim, info.sms, kBackwardCtas);
  const long long parts = static_cast<long long>(B) * ((L + run - 1) / run);
  if (parts > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  return static_cast<int>(parts);
}

int btp_sm100_causal_conv_backward(const void* x, const void* weight, const void* bias, const void* initial, const int* lengths,
                                   const void* dy, const void* dstate, void* dx, void* dweight, void* dbias, void* dinitial,
                                   float* partial, int B, int L, int dim, int width, long long sx_b, long long sx_t, int silu,
                                   int dtype, int weight_dtype, void* stream) {
  const char* fn = "btp_sm100_causal_conv_backward";
  int rc = check(fn, B, L, dim, width, dtype, weight_dtype);
  if (rc) return rc;
  if (!x || !weight || !dy || !dx) return fail(BTP_ERR_NULL_POINTER, "%s: x, weight, dy and dx must not be NULL", fn);
  if ((dweight || dbias) && !partial) return fail(BTP_ERR_NULL_POINTER, "%s: dweight and dbias need the partial sums", fn);
  if (partial && (reinterpret_cast<uintptr_t>(partial) & 7u)) return fail(BTP_ERR_MISALIGNED, "%s: the partial sums must be 8-byte aligned", fn);
  if (sx_b < 0 || sx_t < 0) return fail(BTP_ERR_BAD_SHAPE, "%s: strides must not be negative", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  ConvParams p{};
  p.x = x; p.weight = weight; p.bias = bias; p.initial = initial; p.lengths = lengths; p.dy = dy; p.dstate = dstate; p.dx = dx;
  p.dinitial = dinitial; p.partial = dweight || dbias ? partial : nullptr;
  p.sx_b = sx_b; p.sx_t = sx_t; p.B = B; p.L = L; p.dim = dim; p.silu = silu != 0; p.weight_f32 = weight_dtype == BTP_DTYPE_F32;
  const int e = elem_bytes(dtype);
  p.aligned = one_word(2, e, dim, sx_b, sx_t, {x, dy, dx, initial, dstate, dinitial});
  p.copies = one_word(16 / e, e, dim, sx_b, sx_t, {x});
  p.copies_dy = one_word(16 / e, e, dim, 0, 0, {dy});
  p.whole_w = aligned16(weight);
  p.run = tokens_per_run(B, L, dim, info.sms, kBackwardCtas);
  p.runs = (L + p.run - 1) / p.run;
  const long long parts = static_cast<long long>(B) * p.runs;
  const long long ctas = parts * ((dim + kCols - 1) / kCols);
  if (ctas > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = launched(fn, dispatch(dtype, width, [&](auto tag, auto taps) {
    using T = decltype(tag);
    constexpr int W = decltype(taps)::value;
    constexpr int kSmem = static_cast<int>(sizeof(ConvTile<T, 2>));
    // per device and process: the same value every time, so a race of two threads is harmless
    const cudaError_t err = cudaFuncSetAttribute(conv_backward_kernel<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (err != cudaSuccess) return err;
    return launch_kernel(conv_backward_kernel<T, W>, static_cast<int>(ctas), kThreads, kSmem, st, p);
  }));
  if (rc || !p.partial) return rc;
  const long long cols = static_cast<long long>(width + 1) * dim;
  return launched(fn, by_type(dtype, [&](auto tag) {
    return launch_kernel(conv_weight_sum_kernel<decltype(tag)>, static_cast<int>((cols + 31) / 32), 256, 0, st,
                         static_cast<const float*>(partial), dweight, dbias, parts, dim, width, p.weight_f32);
  }));
}

int btp_sm100_causal_conv_step(const void* x, const void* state, const void* weight, const void* bias, void* y, void* state_out,
                               int B, int dim, int width, long long ld_x, int silu, int dtype, int weight_dtype, void* stream) {
  const char* fn = "btp_sm100_causal_conv_step";
  int rc = check(fn, B, 1, dim, width, dtype, weight_dtype);
  if (rc) return rc;
  if (!x || !state || !weight || !y || !state_out)
    return fail(BTP_ERR_NULL_POINTER, "%s: x, state, weight, y and state_out must not be NULL", fn);
  if (ld_x < 0) return fail(BTP_ERR_BAD_SHAPE, "%s: strides must not be negative", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  ConvStepParams p{};
  p.aligned = one_word(kStepChannels, elem_bytes(dtype), dim, ld_x, 0, {x, y, state, state_out});
  p.whole_w = aligned16(weight);
  p.x = x; p.state = state; p.weight = weight; p.bias = bias; p.y = y; p.state_out = state_out;
  p.ld_x = ld_x; p.B = B; p.dim = dim; p.silu = silu != 0; p.weight_f32 = weight_dtype == BTP_DTYPE_F32;
  const long long ctas = (static_cast<long long>(B) * ((dim + kStepChannels - 1) / kStepChannels) + 127) / 128;
  if (ctas > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launched(fn, dispatch(dtype, width, [&](auto tag, auto taps) {
    using T = decltype(tag);
    constexpr int W = decltype(taps)::value;
    return launch_kernel(conv_step_kernel<T, W>, static_cast<int>(ctas), 128, 0, st, p);
  }));
}

}  // extern "C"
