// The token-major operators (norm, convolution, scan) on torch tensors, in C++ on top of the C ABI: outputs and workspaces, launches, and
// the autograd nodes of training passes.
//
// A backward pass runs on autograd's device thread, where every Python call costs several times what it costs on the caller's (cold caches
// and the hand-over of the interpreter lock).  Measured for 64 x 512 float32 through torch.autograd.grad, whole pass of the norm: 63 us
// with these nodes, 108 with the same steps in Python, 84 for elementary torch operations without autograd.
//
// The callers in spear_b200/ops have checked every argument and made every tensor dense where the kernels need it.  They do not come
// here while somebody records the call (torch.compile, make_fx, torch.jit.trace, tensor subclasses): then the Python functions beside them
// run the registered ops.  A backward pass may be recorded although its forward was not; it then runs the registered op too.
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/btp_sm100.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kCheckpoint = 16;  // tokens between the states that the scan's forward keeps

int tag(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? BTP_DTYPE_BF16 : t.scalar_type() == at::kHalf ? BTP_DTYPE_F16 : BTP_DTYPE_F32;
}
template <class T = void>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
Tensor plain(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor option(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor floats(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().dtype(at::kFloat)); }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
// Channels dense, other strides free.
Tensor dense_last(const Tensor& t) { return t.is_contiguous() || t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
bool trains(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
Tensor aligned(const Tensor& t) { return t.defined() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 ? t.clone() : t; }

// The tensors' device is current and its stream is the one to launch on.
struct On {
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
  c10::cuda::CUDAGuard guard;
  void* stream;
};
void check(int rc, const char* name) {
  TORCH_CHECK(rc == BTP_OK, name, " failed: ", btp_sm100_status_string(rc), ": ", btp_sm100_last_error());
}
template <class I>
I sized(I n, const char* name) {
  if (n < 0) check(static_cast<int>(n), name);
  return n;
}

// Whether somebody records or interprets this backward pass.
bool recorded(const variable_list& grads) {
  if (c10::impl::TorchDispatchModeTLS::stack_len() > 0 || torch::jit::tracer::isTracing()) return true;
  for (const auto& g : grads)
    if (g.defined() && g.key_set().has(c10::DispatchKey::Python)) return true;
  return false;
}
template <class... Args>
void run_op(const char* name, Args&&... args) {
  auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "");
  torch::jit::Stack stack;
  (stack.emplace_back(std::forward<Args>(args)), ...);
  op.callBoxed(stack);
}

// Gradients that cannot be differentiated again: under create_graph each says so when somebody tries.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads) {
    if (!g.defined()) continue;
    auto error = std::make_shared<torch::autograd::DelayedError>("this operator has no second derivative", 1);
    g = (*error)({g.detach().set_requires_grad(true)})[0];
  }
  return grads;
}

// What a node keeps besides tensors, as one number: an option, and which of its tensor arguments were given.
int64_t kept(int64_t option, std::initializer_list<bool> given) {
  int64_t bits = 0, i = 0;
  for (bool g : given) bits |= static_cast<int64_t>(g) << i++;
  return option << 16 | bits;
}
// Which of the arguments need a gradient: autograd counts its edges over those that were given.
class Needs {
 public:
  explicit Needs(AutogradContext* ctx) : ctx_(ctx) {
    const int64_t k = ctx->saved_data["kept"].toInt();
    option = k >> 16;
    given_ = k & 0xffff;
  }
  bool operator()(int arg) const {
    if (!(given_ >> arg & 1)) return false;
    size_t edge = 0;
    for (int i = 0; i < arg; ++i) edge += given_ >> i & 1;
    return ctx_->needs_input_grad(edge);
  }
  int64_t option;

 private:
  AutogradContext* ctx_;
  int64_t given_;
};

// ---------------------------------------------------------------------------------------------------- norm
// t as [rows, D] with dense rows at one pitch; copied only where its strides allow no such view.
Tensor rows_of(const Tensor& t) {
  const int64_t d = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, d});
  if ((d > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < d)) r = r.contiguous();
  return r;
}
int64_t pitch(const Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }

// y [like x] and, with a residual, h [like it]; rstd [rows] or undefined.
std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& x2, const Tensor& w, const Tensor& residual, const Tensor& rstd, double eps) {
  const Tensor r = residual.defined() ? rows_of(residual) : residual;
  const int64_t rows = x2.size(0), dim = x2.size(1);
  Tensor y = at::empty(x.sizes(), x.options()), h = r.defined() ? at::empty(residual.sizes(), residual.options()) : r;
  if (rows) {
    const On on(x);
    check(btp_sm100_rms_norm_forward(x2.data_ptr(), ptr(r), ptr(w), y.data_ptr(), ptr(h), ptr<float>(rstd), nullptr, rows, static_cast<int>(dim),
                                     pitch(x2), r.defined() ? pitch(r) : dim, static_cast<float>(eps), tag(x), r.defined() ? tag(r) : 0,
                                     w.defined() ? tag(w) : 0, BTP_NORM_SAME, on.stream),
          "btp_sm100_rms_norm_forward");
  }
  return {y, h};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static constexpr bool is_traceable = true;  // a recorded backward pass runs the registered op

  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
    const Tensor x2 = rows_of(x), w = plain(weight), rstd = floats({x2.size(0)}, x);
    const auto [y, h] = norm_forward(x, x2, w, plain(residual), rstd, eps);
    ctx->save_for_backward({h.defined() ? h : x2, w, rstd});
    ctx->saved_data["kept"] = kept(static_cast<int64_t>(x.scalar_type()), {true, weight.has_value(), residual.has_value()});
    ctx->set_materialize_grads(false);
    return h.defined() ? variable_list{y, h} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto saved = ctx->get_saved_variables();
    const Needs need(ctx);
    const auto dtype = static_cast<at::ScalarType>(need.option);
    const bool need_x = need(0), need_w = need(1), need_r = need(2);
    const Tensor &h = saved[0], &w = saved[1], &rstd = saved[2];
    Tensor dx, dw, dr, dh = up.size() > 1 ? up[1] : Tensor();
    if (!up[0].defined()) {  // y was not used: the sum passes its gradient on
      if (dh.defined()) dx = need_x ? dh.to(dtype) : dx, dr = need_r ? dh : dr;
      return once({dx, dw, dr, Tensor()});
    }
    const Tensor dy = up[0].contiguous();
    dh = dense(dh);
    const bool one = h.scalar_type() == dtype;  // one tensor serves as the gradient of both terms of the sum
    if (need_x || (one && need_r)) dx = at::empty_like(dy);
    if (need_r && !one) dr = at::empty_like(dy, dy.options().dtype(h.scalar_type()));
    if (need_w) dw = at::empty_like(w);
    if (dx.defined() || dr.defined() || dw.defined()) {
      const Tensor h2 = rows_of(h);
      const int64_t rows = h2.size(0);
      const int dim = static_cast<int>(h2.size(1));
      if (recorded(up)) {
        run_op("spear_btp::rms_norm_backward", h2, option(w), dy, option(dh), rstd, option(dx), option(dr), option(dw));
      } else if (!rows) {
        if (dw.defined()) dw.zero_();
      } else {
        const On on(dy);
        const Tensor partial = need_w ? floats({sized(btp_sm100_rms_norm_partial_rows(rows, dim), "btp_sm100_rms_norm_partial_rows"), dim}, dy) : Tensor();
        check(btp_sm100_rms_norm_backward(h2.data_ptr(), ptr(w), dy.data_ptr(), ptr(dh), ptr<float>(rstd), ptr(dx), ptr(dr), ptr(dw),
                                          ptr<float>(partial), rows, dim, pitch(h2), tag(dy), tag(h2), w.defined() ? tag(w) : 0, on.stream),
              "btp_sm100_rms_norm_backward");
      }
    }
    if (need_r && one) dr = dx;
    return once({need_x ? dx : Tensor(), dw, dr, Tensor()});
  }
};

std::tuple<Tensor, OptTensor> rms_norm(const Tensor& x, const OptTensor& weight, const OptTensor& residual, double eps) {
  const Tensor w = plain(weight), r = plain(residual);
  if (!trains({&x, &w, &r})) {
    const auto [y, h] = norm_forward(x, rows_of(x), w, r, Tensor(), eps);
    return {y, option(h)};
  }
  auto out = NormNode::apply(x, weight, residual, eps);
  return {out[0], out.size() > 1 ? OptTensor(out[1]) : std::nullopt};
}

// ---------------------------------------------------------------------------------------------------- token-major sequences
// What a function takes besides the tensors that may need gradients.
struct Options {
  Tensor lengths;
  bool on;     // silu, softplus
  bool state;  // whether the final state is returned
};
// Batch and token strides of [B, L, D]; a dimension of one element has none of its own.
struct Strides {
  explicit Strides(const Tensor& t) {
    if (!t.defined()) return;
    token = t.size(1) > 1 ? t.stride(1) : t.size(2);
    batch = t.size(0) > 1 ? t.stride(0) : t.size(1) * token;
  }
  int64_t batch = 0, token = 0;
};

// [B, D] with dense rows, and its pitch.
struct Row {
  explicit Row(const Tensor& t) {
    if (!t.defined()) return;
    rows = dense_last(t);
    pitch = rows.is_contiguous() ? rows.size(1) : rows.stride(0);
  }
  Tensor rows;
  int64_t pitch = 0;
};

std::pair<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& i, const Options& opt) {
  const int B = static_cast<int>(x.size(0)), L = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2)), W = static_cast<int>(w.size(1));
  Tensor y = at::empty({B, L, D}, x.options()), state = opt.state ? at::empty({B, W - 1, D}, x.options()) : Tensor();
  const Strides s(x);
  const On on(x);
  check(btp_sm100_causal_conv_forward(x.data_ptr(), w.data_ptr(), ptr(b), ptr(i), ptr<int>(opt.lengths), y.data_ptr(), ptr(state), B, L, D, W,
                                      s.batch, s.token, opt.on, tag(x), tag(w), on.stream),
        "btp_sm100_causal_conv_forward");
  return {y, state};
}

struct ConvNode : torch::autograd::Function<ConvNode> {
  static constexpr bool is_traceable = true;  // a recorded backward pass runs the registered op

  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& initial,
                               const Options& opt) {
    const Tensor b = plain(bias), i = plain(initial);
    const auto [y, state] = conv_forward(x, weight, b, i, opt);
    ctx->save_for_backward({x, weight, b, i, opt.lengths});
    ctx->saved_data["kept"] = kept(opt.on, {true, true, bias.has_value(), initial.has_value()});
    ctx->set_materialize_grads(false);
    return opt.state ? variable_list{y, state} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    Tensor dw, db, di, dstate = dense(up.size() > 1 ? up[1] : Tensor());
    if (!up[0].defined() && !dstate.defined()) return variable_list(5);
    const auto saved = ctx->get_saved_variables();
    const Needs need(ctx);
    const bool silu = need.option;
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &i = saved[3], &lengths = saved[4];
    const int B = static_cast<int>(x.size(0)), L = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2)), W = static_cast<int>(w.size(1));
    const Tensor dy = up[0].defined() ? up[0].contiguous() : at::zeros(x.sizes(), x.options());
    Tensor dx = at::empty(x.sizes(), x.options());
    if (need(1)) dw = at::empty(w.sizes(), w.options());
    if (need(2)) db = at::empty(b.sizes(), b.options());
    if (need(3)) di = at::empty(i.sizes(), i.options());
    if (recorded(up)) {
      run_op("spear_btp::causal_conv_backward", x, w, option(b), option(i), option(lengths), dy, option(dstate), dx, option(dw), option(db),
             option(di), silu);
    } else {
      const Strides s(x);
      const On on(x);
      const Tensor partial = dw.defined() || db.defined()
                                 ? floats({sized(btp_sm100_causal_conv_partial_rows(B, L, D), "btp_sm100_causal_conv_partial_rows"), W + 1, D}, x)
                                 : Tensor();
      check(btp_sm100_causal_conv_backward(x.data_ptr(), w.data_ptr(), ptr(b), ptr(i), ptr<int>(lengths), dy.data_ptr(), ptr(dstate),
                                           dx.data_ptr(), ptr(dw), ptr(db), ptr(di), ptr<float>(partial), B, L, D, W, s.batch, s.token, silu,
                                           tag(x), tag(w), on.stream),
            "btp_sm100_causal_conv_backward");
    }
    return once({need(0) ? dx : Tensor(), dw, db, di, Tensor()});
  }
};

std::tuple<Tensor, OptTensor> causal_conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& initial,
                                          const OptTensor& lengths, bool silu, bool state) {
  const Tensor b = plain(bias), i = plain(initial);
  const Options opt{plain(lengths), silu, state};
  if (!trains({&x, &weight, &b, &i})) {
    const auto [y, last] = conv_forward(x, weight, b, i, opt);
    return {y, option(last)};
  }
  auto out = ConvNode::apply(x, weight, bias, initial, opt);
  return {out[0], state ? OptTensor(out[1]) : std::nullopt};
}

// One token: (y, the new state), which goes to state_out where that is given.
std::tuple<Tensor, Tensor> causal_conv_step(const Tensor& x, const Tensor& state, const Tensor& weight, const OptTensor& bias,
                                            const OptTensor& state_out, bool silu) {
  const Tensor y = at::empty(x.sizes(), x.options()), out = state_out ? *state_out : at::empty(state.sizes(), state.options());
  if (x.size(0)) {
    const Tensor w = weight.contiguous(), b = dense(plain(bias));
    const Row r(x);
    const On on(x);
    check(btp_sm100_causal_conv_step(r.rows.data_ptr(), state.data_ptr(), w.data_ptr(), ptr(b), y.data_ptr(), out.data_ptr(),
                                     static_cast<int>(x.size(0)), static_cast<int>(x.size(1)), static_cast<int>(w.size(1)), r.pitch, silu, tag(x),
                                     tag(w), on.stream),
          "btp_sm100_causal_conv_step");
  }
  return {y, out};
}

// y, the final state and the checkpoints (where a backward pass will want them).
std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                                                const Tensor& d, const Tensor& z, const Tensor& bias, const Tensor& initial, const Options& opt,
                                                bool keep) {
  const int B = static_cast<int>(x.size(0)), L = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2)), N = static_cast<int>(A.size(1));
  const Tensor A16 = aligned(A), i16 = aligned(initial);
  Tensor y = at::empty({B, L, D}, x.options()), state = opt.state ? floats({B, D, N}, x) : Tensor();
  const Tensor checkpoints = keep ? floats({B, (L + kCheckpoint - 1) / kCheckpoint, D, N}, x) : Tensor();
  const Strides sx(x), sd(delta), sb(Bm), sc(Cm), sz(z);
  const On on(x);
  const auto n = sized(btp_sm100_scan_carry_floats(B, L, D, N), "btp_sm100_scan_carry_floats");
  const Tensor carry = n ? floats({n}, x) : Tensor();
  check(btp_sm100_scan_forward(x.data_ptr(), delta.data_ptr(), ptr<float>(A16), Bm.data_ptr(), Cm.data_ptr(), ptr<float>(d), ptr(z),
                               ptr<float>(bias), ptr<float>(i16), ptr<int>(opt.lengths), y.data_ptr(), ptr<float>(state),
                               ptr<float>(checkpoints), ptr<float>(carry), B, L, D, N, sx.batch, sx.token, sd.batch, sd.token, sb.batch, sb.token,
                               sc.batch, sc.token, sz.batch, sz.token, opt.on, tag(x), on.stream),
        "btp_sm100_scan_forward");
  return {y, state, checkpoints};
}

struct ScanNode : torch::autograd::Function<ScanNode> {
  static constexpr bool is_traceable = true;  // a recorded backward pass runs the registered op

  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                               const OptTensor& skip, const OptTensor& gate, const OptTensor& delta_bias, const OptTensor& initial,
                               const Options& opt) {
    const Tensor d = plain(skip), z = plain(gate), bias = plain(delta_bias);
    const auto [y, state, checkpoints] = scan_forward(x, delta, A, Bm, Cm, d, z, bias, plain(initial), opt, true);
    ctx->save_for_backward({x, delta, A, Bm, Cm, d, z, bias, opt.lengths, checkpoints});
    ctx->saved_data["kept"] =
        kept(opt.on, {true, true, true, true, true, skip.has_value(), gate.has_value(), delta_bias.has_value(), initial.has_value()});
    ctx->set_materialize_grads(false);
    return opt.state ? variable_list{y, state} : variable_list{y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    Tensor dstate = dense(up.size() > 1 ? up[1] : Tensor());
    if (!up[0].defined() && !dstate.defined()) return variable_list(10);
    const auto saved = ctx->get_saved_variables();
    const Needs need(ctx);
    const bool softplus = need.option;
    const Tensor &x = saved[0], &delta = saved[1], &A = saved[2], &Bm = saved[3], &Cm = saved[4], &d = saved[5], &z = saved[6], &bias = saved[7],
                 &lengths = saved[8], &checkpoints = saved[9];
    const int B = static_cast<int>(x.size(0)), L = static_cast<int>(x.size(1)), D = static_cast<int>(x.size(2)), N = static_cast<int>(A.size(1));
    const Tensor dy = up[0].defined() ? up[0].contiguous() : at::zeros(x.sizes(), x.options());
    Tensor dx = at::empty(x.sizes(), x.options()), ddelta = at::empty(x.sizes(), x.options()), dz = z.defined() ? at::empty(x.sizes(), x.options()) : z;
    Tensor dB = at::empty(Bm.sizes(), Bm.options()), dC = at::empty(Cm.sizes(), Cm.options());
    const int64_t rates = static_cast<int64_t>(D) * N;
    const Tensor dparams = floats({(rates + 2 * D + 3) / 4 * 4}, x);  // dA, dD and the bias's, one after the other
    Tensor dinitial = need(8) ? floats({B, D, N}, x) : Tensor();
    if (recorded(up)) {
      run_op("spear_btp::scan_backward", x, delta, A, Bm, Cm, option(d), option(z), option(bias), option(lengths), checkpoints, dy, option(dstate),
             dx, ddelta, dparams, dB, dC, option(dz), option(dinitial), softplus);
    } else {
      const Tensor A16 = aligned(A), s16 = aligned(dstate);
      const Strides sx(x), sd(delta), sb(Bm), sc(Cm), sz(z);
      const On on(x);
      const Tensor buffer = floats({sized(btp_sm100_scan_backward_floats(B, L, D, N), "btp_sm100_scan_backward_floats")}, x);
      check(btp_sm100_scan_backward(x.data_ptr(), delta.data_ptr(), ptr<float>(A16), Bm.data_ptr(), Cm.data_ptr(), ptr<float>(d), ptr(z),
                                    ptr<float>(bias), ptr<int>(lengths), ptr<float>(checkpoints), dy.data_ptr(), ptr<float>(s16), dx.data_ptr(),
                                    ddelta.data_ptr(), ptr<float>(dparams), dB.data_ptr(), dC.data_ptr(), ptr(dz), ptr<float>(dinitial),
                                    ptr<float>(buffer), B, L, D, N, sx.batch, sx.token, sd.batch, sd.token, sb.batch, sb.token, sc.batch, sc.token,
                                    sz.batch, sz.token, softplus, tag(x), on.stream),
            "btp_sm100_scan_backward");
    }
    variable_list grads{dx, ddelta, dparams.narrow(0, 0, rates).view({D, N}), dB, dC, dparams.narrow(0, rates, D), dz,
                        dparams.narrow(0, rates + D, D), dinitial, Tensor()};
    for (int i = 0; i < 9; ++i)
      if (!need(i)) grads[i] = Tensor();
    return once(std::move(grads));
  }
};

std::tuple<Tensor, OptTensor> selective_scan(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C,
                                             const OptTensor& D, const OptTensor& z, const OptTensor& delta_bias, const OptTensor& initial,
                                             const OptTensor& lengths, bool softplus, bool state) {
  const Tensor d = plain(D), gate = plain(z), bias = plain(delta_bias), i = plain(initial);
  const Options opt{plain(lengths), softplus, state};
  if (!trains({&x, &delta, &A, &B, &C, &d, &gate, &bias, &i})) {
    const auto [y, last, none] = scan_forward(x, delta, A, B, C, d, gate, bias, i, opt, false);
    return {y, option(last)};
  }
  auto out = ScanNode::apply(x, delta, A, B, C, D, z, delta_bias, initial, opt);
  return {out[0], state ? OptTensor(out[1]) : std::nullopt};
}

std::tuple<Tensor, Tensor> selective_scan_step(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                                               const Tensor& state, const OptTensor& D, const OptTensor& z, const OptTensor& delta_bias,
                                               const OptTensor& state_out, bool softplus) {
  const Tensor y = at::empty(x.sizes(), x.options()), out = state_out ? *state_out : at::empty(state.sizes(), state.options());
  if (x.size(0)) {
    TORCH_CHECK_VALUE((reinterpret_cast<uintptr_t>(state.data_ptr()) | reinterpret_cast<uintptr_t>(out.data_ptr())) % 16 == 0,
                      "selective_scan_step: state and state_out must be 16-byte aligned");
    const Tensor A16 = aligned(A.contiguous()), d = dense(plain(D)), bias = dense(plain(delta_bias));
    const Row rx(x), rd(delta), rB(Bm), rC(Cm), rz(plain(z));
    const On on(x);
    check(btp_sm100_scan_step(rx.rows.data_ptr(), rd.rows.data_ptr(), ptr<float>(A16), rB.rows.data_ptr(), rC.rows.data_ptr(), ptr<float>(d),
                              ptr(rz.rows), ptr<float>(bias), ptr<float>(state), y.data_ptr(), ptr<float>(out), static_cast<int>(x.size(0)),
                              static_cast<int>(x.size(1)), static_cast<int>(A.size(1)), rx.pitch, rd.pitch, rB.pitch, rC.pitch, rz.pitch, softplus,
                              tag(x), on.stream),
          "btp_sm100_scan_step");
  }
  return {y, out};
}

}  // namespace

PYBIND11_MODULE(btp_torch, m) {
  namespace py = pybind11;
  m.doc() = "The token-major operators on tensors that spear_b200.ops has checked.";
  m.def("rms_norm", &rms_norm, py::call_guard<py::gil_scoped_release>());
  m.def("causal_conv", &causal_conv, py::call_guard<py::gil_scoped_release>());
  m.def("selective_scan", &selective_scan, py::call_guard<py::gil_scoped_release>());
  m.def("causal_conv_step", &causal_conv_step, py::call_guard<py::gil_scoped_release>());
  m.def("selective_scan_step", &selective_scan_step, py::call_guard<py::gil_scoped_release>());
}
