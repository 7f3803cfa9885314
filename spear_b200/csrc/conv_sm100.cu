// C entries of the short causal convolution: argument checks, launch shapes, launches.
#include "conv_kernels.cuh"
#include "elem_host.cuh"

namespace {

using namespace btp_host;
using namespace btp_conv;

// Tokens per thread: as long as the device still gets about two threads per slot (148 SMs x 2048), since every run reads W-1
// tokens of the one before it again; 4 to 64.
int forward_run(long long B, int L, int dim, int vec, int sms) {
  const long long want = B * L * (dim / vec) / (static_cast<long long>(sms) * 2048 * 2);
  int run = 4;
  while (run < 64 && run < want) run *= 2;
  return run;
}
// Backward: a CTA takes 8 runs of 32 lanes' channels.
int backward_run(long long B, int L, int dim, int vec, int sms) {
  const long long want = B * L * (dim / vec) / (static_cast<long long>(sms) * 512 * 2);
  int run = 8;
  while (run < 64 && run < want) run *= 2;
  return run;
}

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

template <class T>
constexpr int vec_of() { return 16 / static_cast<int>(sizeof(T)); }

// f(value of the type, vector width, taps)
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
  const int e = elem_bytes(dtype), vec = 16 / e;
  const bool al = dim % vec == 0 && (sx_b * e) % 16 == 0 && (sx_t * e) % 16 == 0 && aligned16(x) && aligned16(y) &&
                  (!initial || aligned16(initial)) && (!state || aligned16(state));
  ConvParams p{};
  p.x = x; p.weight = weight; p.bias = bias; p.initial = initial; p.lengths = lengths; p.y = y; p.state = state;
  p.sx_b = sx_b; p.sx_t = sx_t; p.B = B; p.L = L; p.dim = dim; p.silu = silu != 0; p.weight_f32 = weight_dtype == BTP_DTYPE_F32;
  const int v = al ? vec : 1;
  p.run = forward_run(B, L, dim, v, info.sms);
  p.runs = (L + p.run - 1) / p.run;
  const long long ctas = (static_cast<long long>(B) * p.runs * (dim / v) + 255) / 256;
  if (ctas > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launched(fn, dispatch(dtype, width, [&](auto tag, auto taps) {
    using T = decltype(tag);
    constexpr int W = decltype(taps)::value;
    if (al) return launch_kernel(conv_forward_kernel<T, vec_of<T>(), W>, static_cast<int>(ctas), 256, 0, st, p);
    return launch_kernel(conv_forward_kernel<T, 1, W>, static_cast<int>(ctas), 256, 0, st, p);
  }));
}

int btp_sm100_causal_conv_partial_rows(int B, int L, int dim) {
  const char* fn = "btp_sm100_causal_conv_partial_rows";
  int rc = check(fn, B, L, dim, 4, BTP_DTYPE_F32, BTP_DTYPE_F32);
  if (rc) return rc;
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  // the most that either vector width takes
  long long most = 0;
  for (int v : {1, 4}) {
    const int run = backward_run(B, L, dim, v, info.sms);
    const long long parts = static_cast<long long>(B) * ((L + run * kRunsPerCta - 1) / (run * kRunsPerCta));
    if (parts > most) most = parts;
  }
  if (most > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  return static_cast<int>(most);
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
  if (sx_b < 0 || sx_t < 0) return fail(BTP_ERR_BAD_SHAPE, "%s: strides must not be negative", fn);
  int dev;
  DeviceInfo info;
  if ((rc = device_info(&dev, &info))) return rc;
  // four channels per thread (8 bytes at 16 bits): filter, windows and sums of W = 4 taps are 20 registers a channel
  const int e = elem_bytes(dtype);
  const auto al4 = [&](const void* q) { return !q || (reinterpret_cast<uintptr_t>(q) & static_cast<uintptr_t>(4 * e - 1)) == 0; };
  const bool al = dim % 4 == 0 && sx_b % 4 == 0 && sx_t % 4 == 0 && al4(x) && al4(dy) && al4(dx) && al4(initial) && al4(dstate) && al4(dinitial);
  ConvParams p{};
  p.x = x; p.weight = weight; p.bias = bias; p.initial = initial; p.lengths = lengths; p.dy = dy; p.dstate = dstate; p.dx = dx;
  p.dinitial = dinitial; p.partial = dweight || dbias ? partial : nullptr;
  p.sx_b = sx_b; p.sx_t = sx_t; p.B = B; p.L = L; p.dim = dim; p.silu = silu != 0; p.weight_f32 = weight_dtype == BTP_DTYPE_F32;
  const int v = al ? 4 : 1;
  p.run = backward_run(B, L, dim, v, info.sms);
  p.runs = (L + p.run - 1) / p.run;
  const long long parts = static_cast<long long>(B) * ((p.runs + kRunsPerCta - 1) / kRunsPerCta);
  const long long ctas = parts * ((dim + 32 * v - 1) / (32 * v));
  if (ctas > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = launched(fn, dispatch(dtype, width, [&](auto tag, auto taps) {
    using T = decltype(tag);
    constexpr int W = decltype(taps)::value;
    if (al) return launch_kernel(conv_backward_kernel<T, 4, W>, static_cast<int>(ctas), 256, 0, st, p);
    return launch_kernel(conv_backward_kernel<T, 1, W>, static_cast<int>(ctas), 256, 0, st, p);
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
  const int e = elem_bytes(dtype), vec = 16 / e;
  const bool al = dim % vec == 0 && (ld_x * e) % 16 == 0 && aligned16(x) && aligned16(y) && aligned16(state) && aligned16(state_out);
  ConvStepParams p{};
  p.x = x; p.state = state; p.weight = weight; p.bias = bias; p.y = y; p.state_out = state_out;
  p.ld_x = ld_x; p.B = B; p.dim = dim; p.silu = silu != 0; p.weight_f32 = weight_dtype == BTP_DTYPE_F32;
  const long long ctas = (static_cast<long long>(B) * (dim / (al ? vec : 1)) + 127) / 128;
  if (ctas > 0x7fffffffll) return fail(BTP_ERR_BAD_SHAPE, "%s: too many elements for one launch", fn);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launched(fn, dispatch(dtype, width, [&](auto tag, auto taps) {
    using T = decltype(tag);
    constexpr int W = decltype(taps)::value;
    if (al) return launch_kernel(conv_step_kernel<T, vec_of<T>(), W>, static_cast<int>(ctas), 128, 0, st, p);
    return launch_kernel(conv_step_kernel<T, 1, W>, static_cast<int>(ctas), 128, 0, st, p);
  }));
}

}  // extern "C"
