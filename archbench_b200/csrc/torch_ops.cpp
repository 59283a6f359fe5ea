// The selective-state-space operators and the fused linear layer as functions of torch tensors: argument checks, output
// and workspace allocation, and the autograd nodes, around the C entry points of gdn_b200.h.  A call costs a few
// microseconds of host time (as Python over ctypes it cost 12 to 18, which bound every call of a few rows).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <functional>
#include <optional>
#include <string>

#include "gdn_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using Opt = std::optional<Tensor>;

// Message parts as text.  Not through streams: on a machine with the CUDA driver's libraries loaded, streaming a number
// from this module ends in another library's copy of the C++ locale and crashes.
std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(const c10::Device& d) { return d.str(); }
std::string text(at::IntArrayRef v) {
  std::string r = "(";
  for (size_t i = 0; i < v.size(); ++i) r += (i ? ", " : "") + std::to_string(v[i]);
  return r + (v.size() == 1 ? ",)" : ")");
}
template <typename... P>
std::string message(const P&... parts) {
  return (std::string() + ... + text(parts));
}
// Refusals are ValueErrors.
#define VALUE(cond, ...) \
  do { \
    if (C10_UNLIKELY(!(cond))) C10_THROW_ERROR(ValueError, message(__VA_ARGS__)); \
  } while (0)

// A library status: sizes that no kernel serves as a ValueError, the rest as archbench_b200.native.GdnError.
void check(int status) {
  if (status == GDN_OK) return;
  if (status == GDN_ERR_SHAPE || status == GDN_ERR_UNSUPPORTED) C10_THROW_ERROR(ValueError, message("sizes out of range: ", gdn_status_string(status)));
  py::gil_scoped_acquire gil;  // an autograd thread may be here without it
  py::module_::import("archbench_b200.native").attr("_check")(status);
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T* ptr_as(const Tensor& t) {
  return static_cast<T*>(ptr(t));
}
Tensor get(const Opt& t) { return t ? *t : Tensor(); }
Opt opt(const Tensor& t) { return t.defined() ? Opt(t) : std::nullopt; }  // autograd nodes take what may be absent so
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

int dtype_code(const Tensor& t, const char* name) {
  VALUE(t.is_cuda(), "archbench_b200 ops run on CUDA tensors only (no CPU path)");
  const auto s = t.scalar_type();
  VALUE(s == at::kFloat || s == at::kBFloat16, name, " must be float32 or bfloat16, got ", s);
  return s == at::kFloat ? GDN_DTYPE_F32 : GDN_DTYPE_BF16;
}

// `t` checked against a shape and a device, in `dtype` with a unit last stride.
Tensor token(const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType dtype, int64_t device) {
  VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
  VALUE(t.is_cuda() && t.get_device() == device, name, " must be on cuda:", device, ", got ", t.device());
  Tensor r = t.scalar_type() == dtype ? t : t.to(dtype);
  return r.stride(-1) == 1 || shape.back() == 1 ? r : r.contiguous();
}
Tensor dense(const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType dtype, int64_t device) {
  return t.defined() ? token(t, name, shape, dtype, device).contiguous() : t;
}

// Token counts as int32; the kernels take min(max(n, 0), T).  Wider types are brought into range first: their low 32 bits alone
// may be any count.
Tensor row_lengths(const Opt& lengths, int64_t B, int64_t T, int64_t device) {
  if (!lengths) return Tensor();
  VALUE(!lengths->is_floating_point() && !lengths->is_complex() && lengths->dim() == 1 && lengths->size(0) == B && lengths->is_cuda() && lengths->get_device() == device,
        "lengths must be an integer tensor of shape (", B, ",) on cuda:", device);
  Tensor n = *lengths;
  if (n.element_size() > 4 || n.scalar_type() == at::kUInt32) n = n.to(at::kLong).clamp(0, T);
  return n.to(at::kInt).contiguous();
}

// The first of `ts` (absent ones among them) that wants a gradient, or NULL.
using Tensors = std::initializer_list<const Tensor*>;
const Tensor* wants_grad(Tensors ts) {
  for (const Tensor* t : ts)  // the kernels would drop a tangent
    if (t->defined() && C10_UNLIKELY(t->_fw_grad(/*level=*/0).defined()))
      C10_THROW_ERROR(NotImplementedError, "the kernels have no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return nullptr;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return t;
  return nullptr;
}

// A kernel wrote `t` in place: a graph that keeps the old values refuses its backward.  (Tensors of inference mode are in no
// graph and have no counter.)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The one-token forms have no gradient.  Where one would be wanted their output says so in its backward, as a node on
// `source`; `run` makes the output.
struct OneTokenNode : torch::autograd::Function<OneTokenNode> {
  static Tensor forward(AutogradContext*, const Tensor&, const std::function<Tensor()>& run) {
    at::AutoDispatchBelowADInplaceOrView below;
    return run();
  }
  static variable_list backward(AutogradContext*, variable_list) {
    C10_THROW_ERROR(Error, "the one-token forms are not differentiable: call the prompt's form on one token");
  }
};
template <typename F>
Tensor one_token(Tensors inputs, const Tensor& state, const F& run) {
  VALUE(!wants_grad({&state}), "state is updated in place and must not require a gradient: detach it");
  const Tensor* source = wants_grad(inputs);
  return source ? OneTokenNode::apply(*source, std::function<Tensor()>(run)) : run();
}

int activation_code(const std::optional<std::string>& a, bool gelu) {
  if (!a) return GDN_ACT_NONE;
  if (*a == "silu") return GDN_ACT_SILU;
  VALUE(gelu && *a == "gelu", "activation must be None, 'silu'", gelu ? " or 'gelu'" : "", ", got '", *a, "'");
  return GDN_ACT_GELU;
}

// A workspace of `bytes` from torch's allocator, for one call on the current stream.
Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

void first_order() {
  if (at::GradMode::is_enabled()) C10_THROW_ERROR(Error, "the kernels' gradients are not differentiable themselves (create_graph)");
}

Tensor empty_like_dense(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }
Tensor zeros_like_dense(const Tensor& t) { return t.defined() ? at::zeros(t.sizes(), t.options()) : Tensor(); }

// ---- causal convolution -----------------------------------------------------------------------

gdn_conv_args conv_block(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, int act, const Tensor& lengths) {
  gdn_conv_args a = {};
  const bool tok = x.dim() == 3;
  a.x = ptr(x); a.weight = ptr(w); a.bias = ptr(bias); a.state_in = ptr(state); a.lengths = ptr_as<int32_t>(lengths);
  a.sx_b = x.stride(0); a.sx_t = tok ? x.stride(1) : 0;
  a.B = x.size(0); a.T = tok ? x.size(1) : 1; a.C = x.size(-1);
  a.width = (int)w.size(1); a.act = act;
  a.dtype = x.scalar_type() == at::kFloat ? GDN_DTYPE_F32 : GDN_DTYPE_BF16;
  a.w_dtype = w.scalar_type() == at::kFloat ? GDN_DTYPE_F32 : GDN_DTYPE_BF16;
  return a;
}

std::pair<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, int act, bool want,
                                       const Tensor& lengths) {
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options()), last;
  if (want) last = at::empty({x.size(0), x.size(2), w.size(1) - 1}, x.options());
  gdn_conv_args a = conv_block(x, w, bias, state, act, lengths);
  a.y = ptr(y); a.sy_b = y.stride(0); a.sy_t = y.stride(1); a.state_out = ptr(last);
  check(gdn_conv_fwd(&a, stream_of(x)));
  return {y, last};
}

// Gradients of x, the weight, the bias and the initial state, in the order and form of the forward's arguments; dy or dlast
// may be absent.
variable_list conv_backward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, const Tensor& lengths, int act,
                            Tensor dy, Tensor dlast) {
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  if (x.numel() == 0)
    return {zeros_like_dense(x), zeros_like_dense(w), zeros_like_dense(bias), !state.defined() ? Tensor() : dlast.defined() ? dlast.clone() : zeros_like_dense(state)};
  dy = dy.defined() ? token(dy, "dy", x.sizes(), x.scalar_type(), x.get_device()) : at::zeros(x.sizes(), x.options());
  if (dlast.defined()) dlast = dlast.contiguous();
  variable_list out = {empty_like_dense(x), empty_like_dense(w), empty_like_dense(bias), empty_like_dense(state)};
  gdn_conv_bwd_args a = {};
  a.fwd = conv_block(x, w, bias, state, act, lengths);
  a.dy = ptr(dy); a.sdy_b = dy.stride(0); a.sdy_t = dy.stride(1);
  a.dstate_out = ptr(dlast); a.dx = ptr(out[0]); a.dweight = ptr(out[1]); a.dbias = ptr(out[2]); a.dstate_in = ptr(out[3]);
  size_t need = 0;
  check(gdn_conv_bwd_workspace_bytes(&a, &need));
  const Tensor ws = workspace(need, x);
  a.workspace = ptr(ws); a.workspace_bytes = need;
  check(gdn_conv_bwd(&a, stream_of(x)));
  return out;
}

struct ConvNode : torch::autograd::Function<ConvNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& bias0, const Opt& state0, const Opt& lengths0,
                               int64_t act, bool want) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor bias = get(bias0), state = get(state0), lengths = get(lengths0);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, bias, state, lengths});
    ctx->saved_data["act"] = act;
    auto [y, last] = conv_forward(x, w, bias, state, (int)act, want, lengths);
    return want ? variable_list{y, last} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order();
    const auto s = ctx->get_saved_variables();
    const Tensor dy = g[0], dlast = g.size() > 1 ? g[1] : Tensor();
    if (!dy.defined() && !dlast.defined()) return variable_list(7);
    variable_list out = conv_backward(s[0], s[1], s[2], s[3], s[4], (int)ctx->saved_data["act"].toInt(), dy, dlast);
    out.resize(7);
    return out;
  }
};

std::pair<Tensor, Tensor> conv_params(Tensor w, const Opt& bias, int64_t C, int64_t device) {
  if (w.dim() == 3 && w.size(1) == 1) w = w.select(1, 0);  // nn.Conv1d's (C, 1, W)
  VALUE(w.dim() == 2 && w.size(0) == C, "weight must be (", C, ", W) or (", C, ", 1, W), got ", w.sizes());
  VALUE(w.size(1) >= 2 && w.size(1) <= 4, "the convolution kernels serve widths 2 to 4, got ", w.size(1));
  dtype_code(w, "weight");
  const int64_t wide[] = {C, w.size(1)}, one[] = {C};
  return {dense(w, "weight", wide, w.scalar_type(), device), dense(get(bias), "bias", one, w.scalar_type(), device)};
}

std::pair<Tensor, Opt> causal_conv(const Tensor& x0, const Tensor& weight, const Opt& bias0, const std::optional<std::string>& activation,
                                   const Opt& initial_state, bool output_final_state, const Opt& lengths0) {
  dtype_code(x0, "x");
  VALUE(x0.dim() == 3, "x must be (B, T, C), got ", x0.sizes());
  const int64_t device = x0.get_device(), B = x0.size(0), C = x0.size(2);
  const int act = activation_code(activation, false);
  const Tensor x = token(x0, "x", x0.sizes(), x0.scalar_type(), device);
  const auto [w, bias] = conv_params(weight, bias0, C, device);
  const int64_t st[] = {B, C, w.size(1) - 1};
  const Tensor state = dense(get(initial_state), "initial_state", st, x.scalar_type(), device), lengths = row_lengths(lengths0, B, x.size(1), device);
  Tensor y, last;
  if (wants_grad({&x, &w, &bias, &state})) {
    const variable_list r = ConvNode::apply(x, w, opt(bias), opt(state), opt(lengths), (int64_t)act, output_final_state);
    y = r[0];
    if (output_final_state) last = r[1];
  } else {
    std::tie(y, last) = conv_forward(x, w, bias, state, act, output_final_state, lengths);
  }
  return {y, last.defined() ? Opt(last) : std::nullopt};
}

Tensor causal_conv_step(const Tensor& x0, const Tensor& weight, const Tensor& state, const Opt& bias0, const std::optional<std::string>& activation) {
  dtype_code(x0, "x");
  VALUE(x0.dim() == 2, "x must be (B, C), got ", x0.sizes());
  const int64_t device = x0.get_device(), B = x0.size(0), C = x0.size(1);
  const int act = activation_code(activation, false);
  const Tensor x = token(x0, "x", x0.sizes(), x0.scalar_type(), device);
  const auto [w, bias] = conv_params(weight, bias0, C, device);
  const int64_t st[] = {B, C, w.size(1) - 1};
  VALUE(state.sizes() == at::IntArrayRef(st) && state.scalar_type() == x.scalar_type() && state.is_contiguous() && state.device() == x.device(),
        "state must be a contiguous ", at::IntArrayRef(st), " ", x.scalar_type(), " tensor on ", x.device(), ": it is updated in place");
  return one_token({&x, &w, &bias}, state, [&, &w = w, &bias = bias] {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const Tensor y = at::empty({B, C}, x.options());
    gdn_conv_args a = conv_block(x, w, bias, state, act, Tensor());
    a.y = ptr(y); a.sy_b = y.stride(0);
    check(gdn_conv_step(&a, stream_of(x)));
    written(state);
    return y;
  });
}

// ---- selective scan ---------------------------------------------------------------------------

struct ScanIn {
  Tensor x, dt, A, B, C, D, z, bias, h0, lengths;
  bool softplus;
};

gdn_scan_args scan_block(const ScanIn& s) {
  gdn_scan_args a = {};
  const bool tok = s.x.dim() == 3;
  const int g = tok ? 2 : 1;  // the group dimension of B and C
  a.x = ptr(s.x); a.dt = ptr(s.dt); a.Bm = ptr(s.B); a.Cm = ptr(s.C); a.z = ptr(s.z);
  a.A = ptr_as<float>(s.A); a.Dskip = ptr_as<float>(s.D); a.dt_bias = ptr_as<float>(s.bias); a.h0 = ptr_as<float>(s.h0);
  a.lengths = ptr_as<int32_t>(s.lengths);
  a.sx_b = s.x.stride(0); a.sdt_b = s.dt.stride(0); a.sB_b = s.B.stride(0); a.sC_b = s.C.stride(0);
  a.sB_g = s.B.stride(g); a.sC_g = s.C.stride(g);
  if (s.z.defined()) a.sz_b = s.z.stride(0);
  if (tok) {
    a.sx_t = s.x.stride(1); a.sdt_t = s.dt.stride(1); a.sB_t = s.B.stride(1); a.sC_t = s.C.stride(1);
    if (s.z.defined()) a.sz_t = s.z.stride(1);
  }
  a.B = s.x.size(0); a.T = tok ? s.x.size(1) : 1; a.D = s.x.size(-1); a.N = s.A.size(1); a.G = s.B.size(g);
  a.dtype = s.x.scalar_type() == at::kFloat ? GDN_DTYPE_F32 : GDN_DTYPE_BF16;
  a.softplus = s.softplus;
  return a;
}

struct ScanOut {
  Tensor y, h, ckpt;
};

ScanOut scan_forward(const ScanIn& s, bool want, bool train) {
  const Tensor& x = s.x;
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  const int64_t B = x.size(0), T = x.size(1), D = x.size(2), N = s.A.size(1);
  ScanOut o;
  o.y = at::empty({B, T, D}, x.options());
  if (want) o.h = at::empty({B, D, N}, f32);
  if (train) o.ckpt = at::empty({B, (T + GDN_SCAN_CKPT - 1) / GDN_SCAN_CKPT, D, N}, f32);
  gdn_scan_args a = scan_block(s);
  a.y = ptr(o.y); a.sy_b = o.y.stride(0); a.sy_t = o.y.stride(1); a.h_out = ptr_as<float>(o.h); a.ckpt = ptr_as<float>(o.ckpt);
  size_t need = 0;
  check(gdn_scan_workspace_bytes(&a, &need));
  const Tensor ws = workspace(need, x);
  a.workspace = ptr(ws); a.workspace_bytes = need;
  check(gdn_scan_fwd(&a, stream_of(x)));
  return o;
}

// Gradients of x, dt, A, B, C, D, z, the bias and the initial state, as for the convolution.
variable_list scan_backward(const ScanIn& s, const Tensor& ckpt, Tensor dy, Tensor dh) {
  const Tensor& x = s.x;
  const Tensor in[] = {s.x, s.dt, s.A, s.B, s.C, s.D, s.z, s.bias, s.h0};
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  variable_list out(9);
  if (x.numel() == 0) {
    for (int i = 0; i < 8; ++i) out[i] = zeros_like_dense(in[i]);
    out[8] = !s.h0.defined() ? Tensor() : dh.defined() ? dh.clone() : zeros_like_dense(s.h0);
    return out;
  }
  dy = dy.defined() ? token(dy, "dy", x.sizes(), x.scalar_type(), x.get_device()) : at::zeros(x.sizes(), x.options());
  if (dh.defined()) dh = dh.contiguous();
  for (int i = 0; i < 9; ++i) out[i] = empty_like_dense(in[i]);
  gdn_scan_bwd_args a = {};
  a.fwd = scan_block(s);
  a.fwd.ckpt = ptr_as<float>(ckpt);
  a.dy = ptr(dy); a.sdy_b = dy.stride(0); a.sdy_t = dy.stride(1); a.dh_out = ptr_as<float>(dh);
  a.dx = ptr(out[0]); a.ddt = ptr(out[1]); a.dA = ptr_as<float>(out[2]); a.dB = ptr(out[3]); a.dC = ptr(out[4]);
  a.dDskip = ptr_as<float>(out[5]); a.dz = ptr(out[6]); a.ddt_bias = ptr_as<float>(out[7]); a.dh0 = ptr_as<float>(out[8]);
  size_t need = 0;
  check(gdn_scan_bwd_workspace_bytes(&a, &need));
  const Tensor ws = workspace(need, x);
  a.fwd.workspace = ptr(ws); a.fwd.workspace_bytes = need;
  check(gdn_scan_bwd(&a, stream_of(x)));
  return out;
}

struct ScanNode : torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                               const Opt& D0, const Opt& z0, const Opt& bias0, const Opt& h00, const Opt& lengths0, bool softplus, bool want) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor D = get(D0), z = get(z0), bias = get(bias0), h0 = get(h00), lengths = get(lengths0);
    ctx->set_materialize_grads(false);
    const ScanOut o = scan_forward({x, dt, A, B, C, D, z, bias, h0, lengths, softplus}, want, true);
    ctx->save_for_backward({x, dt, A, B, C, D, z, bias, h0, lengths, o.ckpt});
    ctx->saved_data["softplus"] = softplus;
    return want ? variable_list{o.y, o.h} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order();
    const auto v = ctx->get_saved_variables();
    const Tensor dy = g[0], dh = g.size() > 1 ? g[1] : Tensor();
    if (!dy.defined() && !dh.defined()) return variable_list(12);
    variable_list out = scan_backward({v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9], ctx->saved_data["softplus"].toBool()}, v[10], dy, dh);
    out.resize(12);
    return out;
  }
};

// Checked inputs: token tensors in x's dtype with unit last strides, B and C (..., G, N), parameters fp32.
ScanIn scan_inputs(const Tensor& x, const Tensor& dt, const Tensor& A, Tensor B, Tensor C, const Opt& D, const Opt& z, const Opt& dt_bias,
                   bool softplus) {
  dtype_code(x, "x");
  const int64_t device = x.get_device(), nd = x.dim(), Dm = x.size(-1);
  const auto ty = x.scalar_type();
  VALUE(A.dim() == 2 && A.size(0) == Dm, "A must be (", Dm, ", N), got ", A.sizes());
  const int64_t N = A.size(1);
  VALUE(N >= 1 && N <= 64, "the scan kernels serve 1 to 64 states per channel, got ", N);
  if (B.dim() == nd) B = B.unsqueeze(-2);
  if (C.dim() == nd) C = C.unsqueeze(-2);
  const int64_t G = B.dim() == nd + 1 ? B.size(-2) : 0;
  VALUE(G >= 1 && Dm % G == 0, "B must be (..., ", N, ") or (..., G, ", N, ") with G a divisor of ", Dm, ", got ", B.sizes());
  c10::SmallVector<int64_t, 4> states(x.sizes().begin(), x.sizes().end() - 1);
  states.push_back(G);
  states.push_back(N);
  const int64_t one[] = {Dm}, two[] = {Dm, N};
  ScanIn s;
  s.x = token(x, "x", x.sizes(), ty, device);
  s.dt = token(dt, "dt", x.sizes(), ty, device);
  s.B = token(B, "B", states, ty, device);
  s.C = token(C, "C", states, ty, device);
  if (z) s.z = token(*z, "z", x.sizes(), ty, device);
  s.A = dense(A, "A", two, at::kFloat, device);
  s.D = dense(get(D), "D", one, at::kFloat, device);
  s.bias = dense(get(dt_bias), "dt_bias", one, at::kFloat, device);
  s.softplus = softplus;
  return s;
}

ScanIn scan_block_inputs(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D, const Opt& z,
                         const Opt& dt_bias, bool softplus, const Opt& h0, const Opt& lengths) {
  VALUE(x.dim() == 3, "x must be (B, T, D), got ", x.sizes());
  ScanIn s = scan_inputs(x, dt, A, B, C, D, z, dt_bias, softplus);
  const int64_t st[] = {x.size(0), x.size(2), s.A.size(1)};
  s.h0 = dense(get(h0), "initial_state", st, at::kFloat, x.get_device());
  s.lengths = row_lengths(lengths, x.size(0), x.size(1), x.get_device());
  return s;
}

std::pair<Tensor, Opt> selective_scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D,
                                      const Opt& z, const Opt& dt_bias, bool dt_softplus, const Opt& initial_state, bool output_final_state,
                                      const Opt& lengths) {
  const ScanIn s = scan_block_inputs(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, lengths);
  Tensor y, h;
  if (wants_grad({&s.x, &s.dt, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias, &s.h0})) {
    const variable_list r = ScanNode::apply(s.x, s.dt, s.A, s.B, s.C, opt(s.D), opt(s.z), opt(s.bias), opt(s.h0), opt(s.lengths),
                                             dt_softplus, output_final_state);
    y = r[0];
    if (output_final_state) h = r[1];
  } else {
    const ScanOut o = scan_forward(s, output_final_state, false);
    y = o.y;
    h = o.h;
  }
  return {y, h.defined() ? Opt(h) : std::nullopt};
}

Tensor selective_scan_step(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& state, const Opt& D,
                           const Opt& z, const Opt& dt_bias, bool dt_softplus) {
  VALUE(x.dim() == 2, "x must be (B, D), got ", x.sizes());
  const ScanIn s = scan_inputs(x, dt, A, B, C, D, z, dt_bias, dt_softplus);
  const int64_t st[] = {x.size(0), x.size(1), s.A.size(1)};
  VALUE(state.sizes() == at::IntArrayRef(st) && state.scalar_type() == at::kFloat && state.is_contiguous() && state.device() == x.device(),
        "state must be a contiguous ", at::IntArrayRef(st), " float32 tensor on ", x.device(), ": it is updated in place");
  return one_token({&s.x, &s.dt, &s.A, &s.B, &s.C, &s.D, &s.z, &s.bias}, state, [&] {
    const c10::cuda::OptionalCUDAGuard guard(x.device());
    const Tensor y = at::empty(x.sizes(), x.options());
    gdn_scan_args a = scan_block(s);
    a.y = ptr(y); a.sy_b = y.stride(0); a.h_out = ptr_as<float>(state);
    check(gdn_scan_step(&a, stream_of(x)));
    written(state);
    return y;
  });
}

// ---- linear -----------------------------------------------------------------------------------

std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& res, int act, bool want_pre) {
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  const Tensor y = at::empty({M, N}, x.options());
  Tensor pre;
  if (want_pre && act) pre = at::empty({M, N}, x.options().dtype(at::kHalf));  // act'(x W^T + b)
  gdn_linear_args a = {};
  a.x = ptr(x); a.weight = ptr(w); a.bias = ptr(bias); a.residual = ptr(res); a.y = ptr(y); a.pre = ptr(pre);
  a.sx = x.stride(0); a.sw = w.stride(0); a.sr = res.defined() ? res.stride(0) : 0; a.sy = N;
  a.M = M; a.N = N; a.K = K; a.act = act; a.keep = GDN_LINEAR_KEEP_SLOPE;
  size_t need = 0;
  check(gdn_linear_workspace_bytes(&a, &need));
  const Tensor ws = workspace(need, x);
  a.workspace = ptr(ws); a.workspace_bytes = need;
  check(gdn_linear_fwd(&a, stream_of(x)));
  return {y, pre};
}

// Gradients of x, the weight and the bias, those whose bit is set in `needs`.
variable_list linear_backward(const Tensor& x, const Tensor& w, const Tensor& pre, Tensor dy, int act, int64_t needs) {
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  variable_list out(3);
  auto make = [&](int i, at::IntArrayRef shape) {
    if (needs >> i & 1) out[i] = M ? at::empty(shape, x.options()) : at::zeros(shape, x.options());
  };
  make(0, {M, K});
  make(1, {N, K});
  make(2, {N});
  if (M == 0 || !(needs & 7)) return out;
  if (dy.stride(-1) != 1) dy = dy.contiguous();
  gdn_linear_bwd_args a = {};
  a.x = ptr(x); a.weight = ptr(w); a.pre = ptr(pre); a.dy = ptr(dy);
  a.dx = ptr(out[0]); a.dweight = ptr(out[1]); a.dbias = ptr(out[2]);
  a.sx = x.stride(0); a.sw = w.stride(0); a.sdy = dy.stride(0);
  a.M = M; a.N = N; a.K = K; a.act = act; a.keep = GDN_LINEAR_KEEP_SLOPE;
  size_t need = 0;
  check(gdn_linear_bwd_workspace_bytes(&a, &need));
  const Tensor ws = workspace(need, x);
  a.workspace = ptr(ws); a.workspace_bytes = need;
  check(gdn_linear_bwd(&a, stream_of(x)));
  return out;
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& bias0, const Opt& res0, int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor bias = get(bias0), res = get(res0);
    auto [y, pre] = linear_forward(x, w, bias, res, (int)act, true);
    ctx->save_for_backward({x, w, pre});
    ctx->saved_data["act"] = act;
    ctx->saved_data["needs"] = (int64_t)(x.requires_grad() | (w.requires_grad() << 1) | ((bias.defined() && bias.requires_grad()) << 2) |
                                         ((res.defined() && res.requires_grad()) << 3));
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order();
    const auto s = ctx->get_saved_variables();
    const Tensor dy = g[0];
    variable_list out(5);
    if (!dy.defined()) return out;
    const int64_t needs = ctx->saved_data["needs"].toInt();
    const variable_list made = linear_backward(s[0], s[1], s[2], dy, (int)ctx->saved_data["act"].toInt(), needs);
    std::copy(made.begin(), made.end(), out.begin());
    if (needs & 8) out[3] = dy;
    return out;
  }
};

// A bf16 tensor as rows with a unit last stride.
Tensor rows(const Tensor& t, const char* name, at::IntArrayRef shape, int64_t device) {
  VALUE(t.sizes() == shape, name, " must be ", shape, ", got ", t.sizes());
  VALUE(t.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  VALUE(t.is_cuda() && t.get_device() == device, name, " must be on cuda:", device, ", got ", t.device());
  const Tensor r = t.dim() == 2 ? t : t.reshape({-1, shape.back()});
  return r.stride(-1) == 1 || shape.back() == 1 ? r : r.contiguous();
}

struct LinearIn {
  Tensor x, w, bias, residual;
};

// x as (M, K) rows, the weight, the bias and the residual as (M, N) rows, checked.
LinearIn linear_inputs(const Tensor& x0, const Tensor& weight, const Opt& bias0, const Opt& residual0) {
  VALUE(x0.is_cuda(), "archbench_b200 ops run on CUDA tensors only (no CPU path)");
  VALUE(x0.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x0.size(-1) && weight.numel() > 0, "x must be (..., K) and weight (N, K), got ",
        x0.sizes(), " and ", weight.sizes());
  const int64_t device = x0.get_device(), N = weight.size(0);
  c10::SmallVector<int64_t, 5> shape(x0.sizes().begin(), x0.sizes().end());
  LinearIn in;
  in.x = rows(x0, "x", shape, device);
  in.w = rows(weight, "weight", weight.sizes(), device);
  shape.back() = N;
  in.bias = get(bias0);
  if (in.bias.defined()) {
    const int64_t one[] = {N};
    VALUE(in.bias.sizes() == at::IntArrayRef(one) && in.bias.scalar_type() == at::kBFloat16 && in.bias.is_cuda() && in.bias.get_device() == device,
          "bias must be a bfloat16 (", N, ",) tensor on cuda:", device);
    in.bias = in.bias.contiguous();
  }
  if (residual0) in.residual = rows(*residual0, "residual", shape, device);
  return in;
}

Tensor linear(const Tensor& x0, const Tensor& weight, const Opt& bias0, const std::optional<std::string>& activation, const Opt& residual0) {
  const LinearIn in = linear_inputs(x0, weight, bias0, residual0);
  const auto& [x, w, bias, residual] = in;
  const int act = activation_code(activation, true);
  Tensor y = wants_grad({&x, &w, &bias, &residual}) ? LinearNode::apply(x, w, opt(bias), opt(residual), (int64_t)act)
                                                : linear_forward(x, w, bias, residual, act, false).first;
  if (x0.dim() == 2) return y;
  c10::SmallVector<int64_t, 5> shape(x0.sizes().begin(), x0.sizes().end());
  shape.back() = w.size(0);
  return y.reshape(shape);
}

// ---- the same in parts, for the registered forms (traced_ops.py) -----------------------------

std::vector<Opt> causal_conv_backward(const Tensor& x0, const Tensor& weight, const Opt& bias0, const std::optional<std::string>& activation,
                                      const Opt& state0, const Opt& lengths0, const Opt& dy, const Opt& dlast) {
  dtype_code(x0, "x");
  VALUE(x0.dim() == 3, "x must be (B, T, C), got ", x0.sizes());
  const int64_t device = x0.get_device(), B = x0.size(0), C = x0.size(2);
  const Tensor x = token(x0, "x", x0.sizes(), x0.scalar_type(), device);
  const auto [w, bias] = conv_params(weight, bias0, C, device);
  const int64_t st[] = {B, C, w.size(1) - 1};
  const Tensor state = dense(get(state0), "initial_state", st, x.scalar_type(), device);
  const variable_list g = conv_backward(x, w, bias, state, row_lengths(lengths0, B, x.size(1), device), activation_code(activation, false), get(dy), get(dlast));
  return {opt(g[0]), opt(g[1]), opt(g[2]), opt(g[3])};
}

// y, the final state and the states that the backward reads.
std::vector<Opt> selective_scan_forward(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D,
                                        const Opt& z, const Opt& dt_bias, bool softplus, const Opt& h0, bool want, const Opt& lengths, bool train) {
  const ScanOut o = scan_forward(scan_block_inputs(x, dt, A, B, C, D, z, dt_bias, softplus, h0, lengths), want, train);
  return {opt(o.y), opt(o.h), opt(o.ckpt)};
}

std::vector<Opt> selective_scan_backward(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D,
                                         const Opt& z, const Opt& dt_bias, bool softplus, const Opt& h0, const Opt& lengths, const Tensor& ckpt,
                                         const Opt& dy, const Opt& dh) {
  std::vector<Opt> out;
  for (const Tensor& g : scan_backward(scan_block_inputs(x, dt, A, B, C, D, z, dt_bias, softplus, h0, lengths), ckpt, get(dy), get(dh)))
    out.push_back(opt(g));
  return out;
}

// y (M, N) and what the backward reads of the activation, for x (M, K).
std::vector<Opt> linear_forward_parts(const Tensor& x, const Tensor& weight, const Opt& bias, const std::optional<std::string>& activation,
                                      const Opt& residual, bool train) {
  const LinearIn in = linear_inputs(x, weight, bias, residual);
  const auto [y, pre] = linear_forward(in.x, in.w, in.bias, in.residual, activation_code(activation, true), train);
  return {opt(y), opt(pre)};
}

std::vector<Opt> linear_backward_parts(const Tensor& x, const Tensor& weight, const Opt& pre, const Tensor& dy,
                                       const std::optional<std::string>& activation, int64_t needs) {
  const LinearIn in = linear_inputs(x, weight, std::nullopt, std::nullopt);
  const int64_t shape[] = {in.x.size(0), in.w.size(0)};
  const variable_list g = linear_backward(in.x, in.w, get(pre), rows(dy, "dy", shape, x.get_device()), activation_code(activation, true), needs);
  return {opt(g[0]), opt(g[1]), opt(g[2])};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("linear", &linear);
  m.def("causal_conv_backward", &causal_conv_backward);
  m.def("selective_scan_forward", &selective_scan_forward);
  m.def("selective_scan_backward", &selective_scan_backward);
  m.def("linear_forward", &linear_forward_parts);
  m.def("linear_backward", &linear_backward_parts);
}
