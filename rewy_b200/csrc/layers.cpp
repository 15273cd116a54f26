// Torch operators of the kernels around a recurrence: arguments checked, outputs allocated, the C ABI called, and the autograd
// nodes of those that train.  Each operator is one function for every backend key: it refuses what it does not take, tensors on
// the CPU last, so that its checks run anywhere.  Launches go to torch's current stream of the tensors' device, on which
// outputs and workspaces are allocated.  Gradients are first order and reverse mode: differentiating them again raises, and so does an
// operand or incoming gradient with a forward-mode derivative.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>
#include <algorithm>
#include <atomic>
#include <optional>
#include <string>
#include <tuple>
#include <vector>
#include "../../include/rewy_b200.h"

namespace {
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

#define WANT(ok, ...) TORCH_CHECK(ok, "rewy_b200 ", __VA_ARGS__)

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
Tensor value(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
const void* in(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const void* in(const OptTensor& t) { return has(t) ? t->data_ptr() : nullptr; }
template <class X>
X* at_ptr(const Tensor& t) { return t.defined() ? static_cast<X*>(t.data_ptr()) : nullptr; }
template <class X>
X* at_ptr(const OptTensor& t) { return has(t) ? static_cast<X*>(t->data_ptr()) : nullptr; }

int dtype_of(const Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return REWY_BF16;
    case at::kHalf: return REWY_F16;
    case at::kFloat: return REWY_F32;
    default: TORCH_CHECK(false, "rewy_b200 ", op, ": ", name, " must be BF16, FP16 or FP32, got ", t.scalar_type());
  }
}
std::string shape(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); i++) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}
void want_shape(const char* op, const char* name, const Tensor& t, at::IntArrayRef sizes) {
  if (t.sizes() == sizes) return;
  std::string s;
  for (size_t i = 0; i < sizes.size(); i++) s += (i ? ", " : "") + std::to_string(sizes[i]);
  TORCH_CHECK(false, "rewy_b200 ", op, ": ", name, " must have the shape [", s, "], got ", shape(t));
}
void want_shape(const char* op, const char* name, const OptTensor& t, at::IntArrayRef sizes) {
  if (has(t)) want_shape(op, name, *t, sizes);
}
void want_type(const char* op, const char* name, const OptTensor& t, at::ScalarType type) {
  WANT(!has(t) || t->scalar_type() == type, op, ": ", name, " must be ", type, ", got ", t->scalar_type());
}
// What the kernels' 32-bit counts hold (the C entries' limits), asked before a size is narrowed to one
constexpr int64_t MOST_TOKENS = int64_t(1) << 30, MOST_CHANNELS = int64_t(1) << 24, MOST_ROWS = (int64_t(1) << 31) - 1;
void want_most(const char* op, const char* what, int64_t n, int64_t most) { WANT(n <= most, op, ": takes up to ", most, " ", what, ", got ", n); }
void want_tokens(const char* op, const Tensor& x) {   // [B, T, channels]
  want_most(op, "sequences", x.size(0), MOST_TOKENS);
  want_most(op, "tokens per sequence", x.size(1), MOST_TOKENS);
  want_most(op, "tokens", x.size(0) * x.size(1), MOST_TOKENS);
  want_most(op, "channels", x.size(2), MOST_CHANNELS);
}

// no derivative that travels with the values: the kernels would drop it
template <class Tensors>
void want_no_tangent(const char* op, const Tensors& tensors) {
  for (const OptTensor& t : tensors) WANT(!has(t) || !t->_fw_grad(0).defined(), op, ": has no forward-mode derivative, and an input carries one");
}
// Tensors that only stand for others have no address: an optional one would be taken for one that is not there.
bool in_memory(const Tensor& t) {
  const auto* impl = t.unsafeGetTensorImpl();
  return impl->has_storage() && (t.numel() == 0 || impl->storage().data() != nullptr);
}
// one CUDA device for all of them
void want_cuda(const char* op, std::initializer_list<OptTensor> tensors) {
  want_no_tangent(op, tensors);
  c10::Device device(c10::kCPU);
  for (const auto& t : tensors) {
    if (!has(t)) continue;
    WANT(t->is_cuda(), op, ": needs CUDA tensors (there is no CPU fallback)");
    WANT(t->layout() == at::kStrided, op, ": needs dense tensors");
    WANT(in_memory(*t), op, ": needs tensors with memory of their own, not fake ones, wrappers or a transform's");
    if (!device.is_cuda()) device = t->device();
    WANT(t->device() == device, op, ": tensors are on ", device, " and ", t->device());
  }
}
void check(int status, const char* what) { WANT(status == REWY_OK, what, " failed with status ", status, ": ", rewy_last_error()); }
rewy_stream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

Tensor rows_of(const Tensor& t) { return t.defined() && t.stride(-1) != 1 && t.size(-1) != 1 ? t.contiguous() : t; }  // last dimension dense
OptTensor dense(const OptTensor& t) { return has(t) ? OptTensor(t->contiguous()) : std::nullopt; }
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// Offsets of packed sequences on the device, checked on the host: from the host copy if there is one.
Tensor packed_offsets(const char* op, const OptTensor& cu, const OptTensor& cu_cpu, const Tensor& x) {
  if (!has(cu)) {
    WANT(!has(cu_cpu), op, ": cu_seqlens_cpu goes with cu_seqlens");
    return Tensor();
  }
  WANT(cu->dim() == 1 && cu->numel() >= 2 && (cu->scalar_type() == at::kInt || cu->scalar_type() == at::kLong), op,
       ": cu_seqlens must hold the int32 or int64 offsets of one sequence or more");
  WANT(x.size(0) == 1, op, ": packed sequences need a batch of 1");
  const Tensor host = (has(cu_cpu) ? *cu_cpu : *cu).to(at::kCPU, at::kLong).contiguous();
  WANT(host.numel() == cu->numel(), op, ": cu_seqlens and cu_seqlens_cpu differ in length");
  const int64_t* h = host.data_ptr<int64_t>();
  bool good = h[0] == 0 && h[host.numel() - 1] == x.size(1);
  for (int64_t i = 1; i < host.numel(); i++) good = good && h[i] > h[i - 1];
  WANT(good, op, ": packed sequences need positive lengths that add up to the token count");
  return cu->to(x.device(), at::kInt).contiguous();
}

// `slots` of a step
void want_slots(const char* op, const OptTensor& slots, int64_t rows, int64_t pool) {
  if (has(slots)) {
    WANT(slots->scalar_type() == at::kInt || slots->scalar_type() == at::kLong, op, ": slots must be int32 or int64");
    want_shape(op, "slots", slots, {rows});
  } else {
    WANT(pool >= rows, op, ": ", pool, " states for ", rows, " rows");
  }
}
void want_state(const char* op, const Tensor& state) {
  WANT(state.is_contiguous(), op, ": the state is updated in place and must be contiguous");
}
void want_no_grad(const char* op, std::initializer_list<OptTensor> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const auto& t : tensors)
    WANT(!has(t) || !t->requires_grad(), op, ": a step has no gradient: call it under torch.no_grad() or with detached tensors");
}
void written(const Tensor& t) {   // in place, behind autograd's back
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor workspace(size_t bytes, const Tensor& like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }

bool any_grad(std::initializer_list<OptTensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : tensors)
    if (has(t) && t->requires_grad()) return true;
  return false;
}

// Backwards that have been launched, for the dispatch report: autograd runs them without passing through Python.
enum { CAUSAL_CONV, SELECTIVE_SCAN, GATED_RMS_NORM, RESIDUAL_RMS_NORM, NODES };
std::atomic<int64_t> backwards[NODES];
std::vector<int64_t> layer_backwards() {   // since the last call, in the order above
  std::vector<int64_t> n;
  for (auto& count : backwards) n.push_back(count.exchange(0));
  return n;
}

// The gradients a node gives, tied to its inputs by one that raises: only a backward that is itself recorded needs it.
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  const auto current = torch::autograd::get_current_node();
  if (current == nullptr) return grads;
  auto edges = current->next_edges();
  const auto error = std::make_shared<torch::autograd::Error>("the gradients of this rewy_b200 operator cannot be differentiated again", std::move(edges));
  for (Tensor& t : grads) {
    if (!t.defined()) continue;
    t = t.detach();
    torch::autograd::create_gradient_edge(t, error);
  }
  return grads;
}
Tensor grad_or_zeros(const Tensor& g, at::IntArrayRef sizes, const at::TensorOptions& o) {
  return g.defined() ? g.to(o.dtype().toScalarType()).contiguous() : at::zeros(sizes, o);
}

// ---- causal convolution ----------------------------------------------------------------------------------------------

RewyConvArgs conv_args(const Tensor& x, const Tensor& weight, const Tensor& bias, bool silu, const Tensor& initial, const Tensor& cu) {
  RewyConvArgs a{};
  a.dtype = dtype_of(x, "causal_conv", "x"); a.param_dtype = dtype_of(weight, "causal_conv", "weight"); a.activation = silu;
  a.B = (int32_t)x.size(0); a.T = (int32_t)x.size(1); a.D = (int32_t)x.size(2); a.W = (int32_t)weight.size(1);
  a.x_batch_stride = x.stride(0); a.x_token_stride = x.stride(1);
  a.x = in(x); a.weight = in(weight); a.bias = in(bias); a.initial_state = in(initial);
  if (cu.defined()) { a.cu_seqlens = cu.data_ptr<int32_t>(); a.num_seqs = (int32_t)cu.numel() - 1; }
  return a;
}
std::tuple<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, bool silu, const Tensor& initial, bool final_state,
                                        const Tensor& cu) {
  const c10::cuda::CUDAGuard guard(x.device());
  RewyConvArgs a = conv_args(x, weight, bias, silu, initial, cu);
  Tensor y = at::empty(x.sizes(), x.options()), fin;
  if (final_state) fin = at::empty({cu.defined() ? cu.numel() - 1 : x.size(0), weight.size(1) - 1, x.size(2)}, x.options());
  a.y = y.data_ptr();
  a.final_state = at_ptr<void>(fin);
  check(rewy_conv_fwd(&a, stream()), "causal_conv");
  return {y, fin};
}

struct Conv : torch::autograd::Function<Conv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& initial, bool silu,
                               bool final_state, const OptTensor& cu) {
    const Tensor xr = rows_of(x), w = weight.contiguous(), b = dense(value(bias)), i = dense(value(initial));
    auto [y, fin] = conv_forward(xr, w, b, silu, i, final_state, value(cu));
    ctx->save_for_backward({xr, w, b, i, value(cu)});
    ctx->saved_data["silu"] = silu;
    ctx->set_materialize_grads(false);
    if (fin.defined()) return {y, fin};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    want_no_tangent("causal_conv backward", grads);
    const auto saved = ctx->get_saved_variables();
    const Tensor x = rows_of(saved[0]), w = saved[1].contiguous(), b = dense(saved[2]), initial = dense(saved[3]), &cu = saved[4];
    const c10::cuda::CUDAGuard guard(x.device());
    RewyConvArgs a = conv_args(x, w, b, ctx->saved_data["silu"].toBool(), initial, cu);
    const Tensor dy = grad_or_zeros(grads[0], x.sizes(), x.options()), dfin = grads.size() > 1 && grads[1].defined() ? grads[1].to(x.scalar_type()).contiguous() : Tensor();
    Tensor dx = at::empty(x.sizes(), x.options()), dw = at::empty_like(w), db, di;
    if (b.defined()) db = at::empty_like(b);
    if (initial.defined()) di = at::empty_like(initial);
    Tensor ws = workspace(rewy_conv_bwd_workspace_bytes(a.B, a.T, a.D, a.W), x);
    a.dy = in(dy); a.dfinal_state = in(dfin);
    a.dx = dx.data_ptr(); a.dweight = dw.data_ptr(); a.dbias = at_ptr<void>(db); a.dinitial_state = at_ptr<void>(di);
    a.workspace = ws.data_ptr(); a.workspace_bytes = ws.nbytes();
    check(rewy_conv_bwd(&a, stream()), "causal_conv backward");
    backwards[CAUSAL_CONV]++;
    auto g = first_order({dx, dw, db, di});
    return {g[0], g[1], g[2], g[3], Tensor(), Tensor(), Tensor()};
  }
};

Tensor conv_weight(const char* op, const Tensor& weight, int64_t channels) {   // [D, W], or [D, 1, W] as convolution modules keep it
  Tensor w = weight.dim() == 3 && weight.size(1) == 1 ? weight.squeeze(1) : weight;
  WANT(w.dim() == 2 && w.size(0) == channels, op, ": weight must have the shape [", channels, ", W], got ", shape(weight));
  WANT(w.size(1) >= 2 && w.size(1) <= 4, op, ": takes 2 to 4 taps, got ", w.size(1));
  return w;
}

std::tuple<Tensor, Tensor> causal_conv(const Tensor& x, const Tensor& weight, const OptTensor& bias, bool silu, const OptTensor& initial_state,
                                       bool output_final_state, const OptTensor& cu_seqlens, const OptTensor& cu_seqlens_cpu) {
  const char* op = "causal_conv";
  WANT(x.dim() == 3, op, ": x must have the shape [B, T, D], got ", shape(x));
  dtype_of(x, op, "x");
  WANT(x.size(0) > 0 && x.size(1) > 0 && x.size(2) > 0, op, ": x must not be empty, got ", shape(x));
  want_tokens(op, x);
  const Tensor w = conv_weight(op, weight, x.size(2));
  dtype_of(w, op, "weight");
  want_shape(op, "bias", bias, {x.size(2)});
  want_type(op, "bias", bias, w.scalar_type());
  const int64_t sequences = has(cu_seqlens) ? cu_seqlens->numel() - 1 : x.size(0);
  want_shape(op, "initial_state", initial_state, {sequences, w.size(1) - 1, x.size(2)});
  want_type(op, "initial_state", initial_state, x.scalar_type());
  const Tensor cu = packed_offsets(op, cu_seqlens, cu_seqlens_cpu, x);
  want_cuda(op, {x, w, bias, initial_state});
  if (any_grad({x, w, bias, initial_state})) {
    auto out = Conv::apply(x, w, bias, initial_state, silu, output_final_state, cu.defined() ? OptTensor(cu) : std::nullopt);
    return {out[0], out.size() > 1 ? out[1] : Tensor()};
  }
  return conv_forward(rows_of(x), w.contiguous(), dense(value(bias)), silu, dense(value(initial_state)), output_final_state, cu);
}

Tensor causal_conv_step(const Tensor& x, Tensor state, const Tensor& weight, const OptTensor& bias, bool silu, const OptTensor& slots) {
  const char* op = "causal_conv_step";
  WANT(x.dim() == 2 && x.numel() > 0, op, ": x must have the shape [B, D], got ", shape(x));
  want_most(op, "rows", x.size(0), MOST_ROWS);
  want_most(op, "channels", x.size(1), MOST_CHANNELS);
  const Tensor w = conv_weight(op, weight, x.size(1)).contiguous(), xr = rows_of(x);
  WANT(state.dim() == 3 && state.size(0) > 0 && state.size(1) == w.size(1) - 1 && state.size(2) == x.size(1), op, ": state must have the shape [pool, ",
       w.size(1) - 1, ", ", x.size(1), "], got ", shape(state));
  want_type(op, "state", state, x.scalar_type());
  want_state(op, state);
  want_shape(op, "bias", bias, {x.size(1)});
  want_type(op, "bias", bias, w.scalar_type());
  want_slots(op, slots, x.size(0), state.size(0));
  want_no_grad(op, {x, state, weight, bias});
  RewyConvStepArgs a{};
  a.dtype = dtype_of(x, op, "x"); a.param_dtype = dtype_of(w, op, "weight");
  want_cuda(op, {x, state, weight, bias, slots});
  const c10::cuda::CUDAGuard guard(x.device());
  const OptTensor b = dense(bias), s = dense(slots);
  Tensor y = at::empty(x.sizes(), x.options());
  a.activation = silu; a.B = (int32_t)x.size(0); a.D = (int32_t)x.size(1); a.W = (int32_t)w.size(1);
  a.slots_i64 = has(s) && s->scalar_type() == at::kLong; a.x_stride = xr.stride(0); a.pool = state.size(0);
  a.x = in(xr); a.weight = in(w); a.bias = in(b); a.slots = in(s); a.state = state.data_ptr(); a.y = y.data_ptr();
  check(rewy_conv_step(&a, stream()), op);
  written(state);
  return y;
}

// ---- selective scan --------------------------------------------------------------------------------------------------

struct ScanInputs {
  Tensor u, dt, A, B, C, D, z, bias, initial, cu;
  bool softplus;
};
RewyScanArgs scan_args(const ScanInputs& s) {
  RewyScanArgs a{};
  a.dtype = dtype_of(s.u, "selective_scan", "u");
  a.B = (int32_t)s.u.size(0); a.T = (int32_t)s.u.size(1); a.M = (int32_t)s.u.size(2); a.N = (int32_t)s.A.size(1); a.G = (int32_t)s.B.size(2);
  a.softplus = s.softplus;
  for (int i = 0; i < 2; i++) {
    a.u_stride[i] = s.u.stride(i); a.dt_stride[i] = s.dt.stride(i);
    if (s.z.defined()) a.z_stride[i] = s.z.stride(i);
  }
  for (int i = 0; i < 3; i++) { a.B_stride[i] = s.B.stride(i); a.C_stride[i] = s.C.stride(i); }
  a.u = in(s.u); a.dt = in(s.dt); a.z = in(s.z); a.Bm = in(s.B); a.C = in(s.C);
  a.A = at_ptr<float>(s.A); a.D = at_ptr<float>(s.D); a.dt_bias = at_ptr<float>(s.bias); a.initial_state = at_ptr<float>(s.initial);
  if (s.cu.defined()) { a.cu_seqlens = s.cu.data_ptr<int32_t>(); a.num_seqs = (int32_t)s.cu.numel() - 1; }
  return a;
}
ScanInputs scan_inputs(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Tensor& D, const Tensor& z, const Tensor& bias,
                       const Tensor& initial, const Tensor& cu, bool softplus) {
  return {rows_of(u), rows_of(dt), A.contiguous(), rows_of(B), rows_of(C), dense(D), rows_of(z), dense(bias), dense(initial), cu, softplus};
}
std::tuple<Tensor, Tensor, Tensor> scan_forward(const ScanInputs& s, bool final_state, bool keep) {
  const c10::cuda::CUDAGuard guard(s.u.device());
  RewyScanArgs a = scan_args(s);
  const auto f32 = s.u.options().dtype(at::kFloat);
  Tensor y = at::empty(s.u.sizes(), s.u.options()), fin, kept;
  if (final_state) fin = at::empty({s.cu.defined() ? s.cu.numel() - 1 : s.u.size(0), a.M, a.N}, f32);
  if (keep) kept = at::empty({(int64_t)(rewy_scan_checkpoint_bytes(a.B, a.T, a.M, a.N) / sizeof(float))}, f32);
  Tensor ws = workspace(rewy_scan_workspace_bytes(a.B, a.T, a.M, a.N, a.G, 0), s.u);
  a.y = y.data_ptr(); a.final_state = at_ptr<float>(fin); a.checkpoints = at_ptr<float>(kept);
  a.workspace = ws.data_ptr(); a.workspace_bytes = ws.nbytes();
  check(rewy_scan_fwd(&a, stream()), "selective_scan");
  return {y, fin, kept};
}

struct Scan : torch::autograd::Function<Scan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& D,
                               const OptTensor& z, const OptTensor& bias, const OptTensor& initial, bool softplus, bool final_state, const OptTensor& cu) {
    const ScanInputs s = scan_inputs(u, dt, A, B, C, value(D), value(z), value(bias), value(initial), value(cu), softplus);
    auto [y, fin, kept] = scan_forward(s, final_state, true);
    ctx->save_for_backward({s.u, s.dt, s.A, s.B, s.C, s.D, s.z, s.bias, s.initial, s.cu, kept});
    ctx->saved_data["softplus"] = softplus;
    ctx->set_materialize_grads(false);
    if (fin.defined()) return {y, fin};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    want_no_tangent("selective_scan backward", grads);
    const auto v = ctx->get_saved_variables();
    const ScanInputs s = scan_inputs(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9], ctx->saved_data["softplus"].toBool());
    const c10::cuda::CUDAGuard guard(s.u.device());
    RewyScanArgs a = scan_args(s);
    const auto f32 = s.A.options();
    const Tensor dy = grad_or_zeros(grads[0], s.u.sizes(), s.u.options()), dfin = grads.size() > 1 && grads[1].defined() ? grads[1].to(at::kFloat).contiguous() : Tensor();
    const Tensor kept = v[10].contiguous();
    auto like = [](const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); };
    Tensor du = like(s.u), ddt = like(s.dt), dz = like(s.z), dB = like(s.B), dC = like(s.C), dA = like(s.A), dD = like(s.D), dbias = like(s.bias),
           di = like(s.initial);
    Tensor ws = workspace(rewy_scan_workspace_bytes(a.B, a.T, a.M, a.N, a.G, 1), s.u);
    a.dy = in(dy); a.dfinal_state = at_ptr<float>(dfin); a.checkpoints = at_ptr<float>(kept);
    a.du = du.data_ptr(); a.ddt = ddt.data_ptr(); a.dz = at_ptr<void>(dz); a.dB = dB.data_ptr(); a.dC = dC.data_ptr();
    a.dA = at_ptr<float>(dA); a.dD = at_ptr<float>(dD); a.ddt_bias = at_ptr<float>(dbias); a.dinitial_state = at_ptr<float>(di);
    a.workspace = ws.data_ptr(); a.workspace_bytes = ws.nbytes();
    check(rewy_scan_bwd(&a, stream()), "selective_scan backward");
    backwards[SELECTIVE_SCAN]++;
    auto g = first_order({du, ddt, dA, dB, dC, dD, dz, dbias, di});
    g.resize(12);
    return g;
  }
};

std::tuple<Tensor, Tensor> selective_scan(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& D,
                                          const OptTensor& z, const OptTensor& dt_bias, bool dt_softplus, const OptTensor& initial_state,
                                          bool output_final_state, const OptTensor& cu_seqlens, const OptTensor& cu_seqlens_cpu) {
  const char* op = "selective_scan";
  WANT(u.dim() == 3, op, ": u must have the shape [B, T, M], got ", shape(u));
  dtype_of(u, op, "u");
  WANT(u.numel() > 0, op, ": u must not be empty, got ", shape(u));
  want_tokens(op, u);
  want_shape(op, "dt", dt, u.sizes());
  want_shape(op, "z", z, u.sizes());
  const int64_t M = u.size(2);
  WANT(A.dim() == 2 && A.size(0) == M, op, ": A must have the shape [", M, ", N], got ", shape(A));
  const int64_t N = A.size(1);
  WANT(N >= 1 && N <= 64, op, ": takes 1 to 64 states per channel, got ", N);
  auto grouped = [&](const Tensor& t, const char* name) {
    const Tensor g = t.dim() == 3 ? t.unsqueeze(2) : t;
    WANT(g.dim() == 4 && g.size(0) == u.size(0) && g.size(1) == u.size(1) && g.size(2) > 0 && M % g.size(2) == 0 && g.size(3) == N, op, ": ", name,
         " must have the shape [B, T, G, N] or [B, T, N] with G a divisor of the channels, got ", shape(t));
    return g;
  };
  const Tensor Bg = grouped(B, "B"), Cg = grouped(C, "C");
  WANT(Bg.size(2) == Cg.size(2), op, ": B and C must have the same groups");
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor>("dt", dt), {"B", B}, {"C", C}, {"z", z}}) want_type(op, name, t, u.scalar_type());
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor>("A", A), {"D", D}, {"dt_bias", dt_bias}, {"initial_state", initial_state}})
    want_type(op, name, t, at::kFloat);
  want_shape(op, "D", D, {M});
  want_shape(op, "dt_bias", dt_bias, {M});
  const int64_t sequences = has(cu_seqlens) ? cu_seqlens->numel() - 1 : u.size(0);
  want_shape(op, "initial_state", initial_state, {sequences, M, N});
  const Tensor cu = packed_offsets(op, cu_seqlens, cu_seqlens_cpu, u);
  want_cuda(op, {u, dt, A, B, C, D, z, dt_bias, initial_state});
  if (any_grad({u, dt, A, B, C, D, z, dt_bias, initial_state})) {
    auto out = Scan::apply(u, dt, A, Bg, Cg, D, z, dt_bias, initial_state, dt_softplus, output_final_state, cu.defined() ? OptTensor(cu) : std::nullopt);
    return {out[0], out.size() > 1 ? out[1] : Tensor()};
  }
  const ScanInputs s = scan_inputs(u, dt, A, Bg, Cg, value(D), value(z), value(dt_bias), value(initial_state), cu, dt_softplus);
  auto [y, fin, kept] = scan_forward(s, output_final_state, false);
  return {y, fin};
}

Tensor selective_scan_step(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, Tensor state, const OptTensor& D,
                           const OptTensor& z, const OptTensor& dt_bias, bool dt_softplus, const OptTensor& slots) {
  const char* op = "selective_scan_step";
  WANT(u.dim() == 2 && u.numel() > 0, op, ": u must have the shape [B, M], got ", shape(u));
  const int64_t R = u.size(0), M = u.size(1);
  want_most(op, "rows", R, MOST_ROWS);
  want_most(op, "channels", M, MOST_CHANNELS);
  want_shape(op, "dt", dt, {R, M});
  want_shape(op, "z", z, {R, M});
  WANT(A.dim() == 2 && A.size(0) == M, op, ": A must have the shape [", M, ", N], got ", shape(A));
  const int64_t N = A.size(1);
  WANT(N >= 1 && N <= 64, op, ": takes 1 to 64 states per channel, got ", N);
  auto grouped = [&](const Tensor& t, const char* name) {
    const Tensor g = t.dim() == 2 ? t.unsqueeze(1) : t;
    WANT(g.dim() == 3 && g.size(0) == R && g.size(1) > 0 && M % g.size(1) == 0 && g.size(2) == N, op, ": ", name,
         " must have the shape [B, G, N] or [B, N] with G a divisor of the channels, got ", shape(t));
    return rows_of(g);
  };
  const Tensor Bg = grouped(B, "B"), Cg = grouped(C, "C");
  WANT(Bg.size(1) == Cg.size(1), op, ": B and C must have the same groups");
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor>("dt", dt), {"B", B}, {"C", C}, {"z", z}}) want_type(op, name, t, u.scalar_type());
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor>("A", A), {"D", D}, {"dt_bias", dt_bias}, {"state", state}}) want_type(op, name, t, at::kFloat);
  want_shape(op, "D", D, {M});
  want_shape(op, "dt_bias", dt_bias, {M});
  WANT(state.dim() == 3 && state.size(0) > 0 && state.size(1) == M && state.size(2) == N, op, ": state must have the shape [pool, ", M, ", ", N, "], got ",
       shape(state));
  want_state(op, state);
  want_slots(op, slots, R, state.size(0));
  want_no_grad(op, {u, dt, A, B, C, state, D, z, dt_bias});
  RewyScanStepArgs a{};
  a.dtype = dtype_of(u, op, "u");
  want_cuda(op, {u, dt, A, B, C, state, D, z, dt_bias, slots});
  const c10::cuda::CUDAGuard guard(u.device());
  const Tensor ur = rows_of(u), dr = rows_of(dt), Ar = A.contiguous(), zr = rows_of(value(z));
  const OptTensor Dr = dense(D), br = dense(dt_bias), s = dense(slots);
  Tensor y = at::empty({R, M}, u.options());
  a.B = (int32_t)R; a.M = (int32_t)M; a.N = (int32_t)N; a.G = (int32_t)Bg.size(1); a.softplus = dt_softplus;
  a.slots_i64 = has(s) && s->scalar_type() == at::kLong;
  a.u_stride = ur.stride(0); a.dt_stride = dr.stride(0); a.z_stride = zr.defined() ? zr.stride(0) : 0; a.pool = state.size(0);
  for (int i = 0; i < 2; i++) { a.B_stride[i] = Bg.stride(i); a.C_stride[i] = Cg.stride(i); }
  a.u = in(ur); a.dt = in(dr); a.z = in(zr); a.Bm = in(Bg); a.C = in(Cg); a.slots = in(s);
  a.A = at_ptr<float>(Ar); a.D = at_ptr<float>(Dr); a.dt_bias = at_ptr<float>(br); a.state = state.data_ptr<float>(); a.y = y.data_ptr();
  check(rewy_scan_step(&a, stream()), op);
  written(state);
  return y;
}

// ---- norms -----------------------------------------------------------------------------------------------------------

struct RowLayout { int64_t inner, stride[2]; };
// Rows of the last dimension as (r / inner) * stride[0] + (r % inner) * stride[1], or nothing if that takes more strides.
std::optional<RowLayout> row_layout(const Tensor& t) {
  if (t.size(-1) != 1 && t.stride(-1) != 1) return std::nullopt;
  int64_t sizes[2] = {1, 1}, strides[2] = {0, 0};   // innermost first
  int levels = 0;
  for (int64_t d = t.dim() - 2; d >= 0; d--) {
    if (t.size(d) == 1) continue;
    if (levels > 0 && t.stride(d) == sizes[levels - 1] * strides[levels - 1]) {
      sizes[levels - 1] *= t.size(d);
    } else {
      if (levels == 2) return std::nullopt;
      sizes[levels] = t.size(d);
      strides[levels++] = t.stride(d);
    }
  }
  return RowLayout{sizes[0], {strides[1], strides[0]}};
}
Tensor norm_rows(const Tensor& t) { return !t.defined() || row_layout(t) ? t : t.contiguous(); }

RewyNormArgs norm_args(const char* op, const Tensor& x, const Tensor& other, const Tensor& weight, double eps) {
  RewyNormArgs a{};
  a.dtype = a.residual_dtype = dtype_of(x, op, "x");
  a.param_dtype = a.scale_dtype = dtype_of(weight, op, "weight");
  a.D = (int32_t)x.size(-1);
  a.rows = x.numel() / x.size(-1);
  const RowLayout lx = *row_layout(x), lo = other.defined() ? *row_layout(other) : RowLayout{1, {0, 0}};
  a.x_inner = lx.inner; a.other_inner = lo.inner;
  for (int i = 0; i < 2; i++) { a.x_stride[i] = lx.stride[i]; a.other_stride[i] = lo.stride[i]; }
  a.eps = (float)eps; a.scale = 1.f;
  a.x = in(x); a.weight = in(weight);
  return a;
}
void check_norm(const char* op, const Tensor& x, const Tensor& weight) {
  WANT(x.dim() >= 1 && x.numel() > 0, op, ": x must have rows of values, got ", shape(x));
  dtype_of(x, op, "x");
  dtype_of(weight, op, "weight");
  WANT(x.size(-1) <= 16384, op, ": takes rows of up to 16384 values, got ", x.size(-1));
  want_shape(op, "weight", weight, {x.size(-1)});
}

RewyNormArgs gated_args(const Tensor& x, const Tensor& gate, const Tensor& weight, double eps, int64_t act, bool gate_first) {
  RewyNormArgs a = norm_args("gated_rms_norm", x, gate, weight, eps);
  a.activation = (int32_t)act; a.gate_first = gate_first; a.gate = in(gate);
  return a;
}
Tensor gated_forward(const Tensor& x, const Tensor& gate, const Tensor& weight, double eps, int64_t act, bool gate_first) {
  const c10::cuda::CUDAGuard guard(x.device());
  RewyNormArgs a = gated_args(x, gate, weight, eps, act, gate_first);
  Tensor y = at::empty(x.sizes(), x.options());
  a.y = y.data_ptr();
  check(rewy_gated_norm_fwd(&a, stream()), "gated_rms_norm");
  return y;
}
struct GatedNorm : torch::autograd::Function<GatedNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& weight, double eps, int64_t act, bool gate_first) {
    const Tensor xr = norm_rows(x), gr = norm_rows(gate), w = weight.contiguous();
    ctx->save_for_backward({xr, gr, w});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["act"] = act;
    ctx->saved_data["gate_first"] = gate_first;
    return gated_forward(xr, gr, w, eps, act, gate_first);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    want_no_tangent("gated_rms_norm backward", grads);
    const auto v = ctx->get_saved_variables();
    const Tensor x = norm_rows(v[0]), gate = norm_rows(v[1]), w = v[2].contiguous(), dy = grad_or_zeros(grads[0], x.sizes(), x.options());
    const c10::cuda::CUDAGuard guard(x.device());
    RewyNormArgs a = gated_args(x, gate, w, ctx->saved_data["eps"].toDouble(), ctx->saved_data["act"].toInt(), ctx->saved_data["gate_first"].toBool());
    Tensor dx = at::empty(x.sizes(), x.options()), dg = at::empty(x.sizes(), x.options()), dw = at::empty_like(w);
    Tensor ws = workspace(rewy_norm_bwd_workspace_bytes(a.rows, a.D), x);
    a.dy = in(dy); a.dx = dx.data_ptr(); a.dgate = dg.data_ptr(); a.dweight = dw.data_ptr();
    a.workspace = ws.data_ptr(); a.workspace_bytes = ws.nbytes();
    check(rewy_gated_norm_bwd(&a, stream()), "gated_rms_norm backward");
    backwards[GATED_RMS_NORM]++;
    auto g = first_order({dx, dg, dw});
    g.resize(6);
    return g;
  }
};
Tensor gated_rms_norm(const Tensor& x, const Tensor& gate, const Tensor& weight, double eps, int64_t activation, bool gate_first) {
  const char* op = "gated_rms_norm";
  check_norm(op, x, weight);
  want_shape(op, "gate", gate, x.sizes());
  want_type(op, "gate", gate, x.scalar_type());
  want_cuda(op, {x, gate, weight});
  if (any_grad({x, gate, weight})) return GatedNorm::apply(x, gate, weight, eps, activation, gate_first);
  return gated_forward(norm_rows(x), norm_rows(gate), weight.contiguous(), eps, activation, gate_first);
}

RewyNormArgs residual_args(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& scale_vector, double scale, double eps) {
  RewyNormArgs a = norm_args("residual_rms_norm", x, residual, weight, eps);
  a.residual = in(residual);
  if (residual.defined()) a.residual_dtype = dtype_of(residual, "residual_rms_norm", "residual");
  a.scale = (float)scale;
  if (scale_vector.defined()) { a.scale_vector = in(scale_vector); a.scale_dtype = dtype_of(scale_vector, "residual_rms_norm", "scale"); }
  return a;
}
std::tuple<Tensor, Tensor> residual_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& scale_vector, double scale, double eps) {
  const c10::cuda::CUDAGuard guard(x.device());
  RewyNormArgs a = residual_args(x, residual, weight, scale_vector, scale, eps);
  Tensor y = at::empty(x.sizes(), x.options()), out = at::empty(x.sizes(), residual.defined() ? residual.options() : x.options());
  a.y = y.data_ptr(); a.residual_out = out.data_ptr();
  check(rewy_residual_norm_fwd(&a, stream()), "residual_rms_norm");
  return {y, out};
}
struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& weight, const OptTensor& scale_vector, double scale,
                               double eps) {
    const Tensor xr = norm_rows(x), rr = norm_rows(value(residual)), w = weight.contiguous(), s = dense(value(scale_vector));
    ctx->save_for_backward({xr, rr, w, s});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    auto [y, out] = residual_forward(xr, rr, w, s, scale, eps);
    return {y, out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    want_no_tangent("residual_rms_norm backward", grads);
    const auto v = ctx->get_saved_variables();
    const Tensor x = norm_rows(v[0]), residual = norm_rows(v[1]), w = v[2].contiguous(), s = dense(v[3]);
    const c10::cuda::CUDAGuard guard(x.device());
    RewyNormArgs a = residual_args(x, residual, w, s, ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble());
    const auto ro = residual.defined() ? residual.options() : x.options();
    const Tensor dy = grad_or_zeros(grads[0], x.sizes(), x.options()), dro = grads[1].defined() ? grads[1].to(ro.dtype().toScalarType()).contiguous() : Tensor();
    Tensor dx = at::empty(x.sizes(), x.options()), dr, dw = at::empty_like(w), ds;
    if (residual.defined()) dr = at::empty(x.sizes(), ro);
    if (s.defined()) ds = at::empty_like(s);
    Tensor ws = workspace(rewy_norm_bwd_workspace_bytes(a.rows, a.D), x);
    a.dy = in(dy); a.dresidual_out = in(dro); a.dx = dx.data_ptr(); a.dresidual = at_ptr<void>(dr); a.dweight = dw.data_ptr(); a.dscale = at_ptr<void>(ds);
    a.workspace = ws.data_ptr(); a.workspace_bytes = ws.nbytes();
    check(rewy_residual_norm_bwd(&a, stream()), "residual_rms_norm backward");
    backwards[RESIDUAL_RMS_NORM]++;
    auto g = first_order({dx, dr, dw, ds});
    g.resize(6);
    return g;
  }
};
std::tuple<Tensor, Tensor> residual_rms_norm(const Tensor& x, const OptTensor& residual, const Tensor& weight, const OptTensor& scale_vector, double scale,
                                             double eps) {
  const char* op = "residual_rms_norm";
  check_norm(op, x, weight);
  want_shape(op, "residual", residual, x.sizes());
  WANT(!has(residual) || residual->scalar_type() == x.scalar_type() || residual->scalar_type() == at::kFloat, op, ": residual must have the type of x or FP32, got ",
       residual->scalar_type());
  want_shape(op, "scale", scale_vector, {x.size(-1)});
  if (has(scale_vector)) dtype_of(*scale_vector, op, "scale");
  want_cuda(op, {x, residual, weight, scale_vector});
  if (any_grad({x, residual, weight, scale_vector})) {
    auto out = ResidualNorm::apply(x, residual, weight, scale_vector, scale, eps);
    return {out[0], out[1]};
  }
  return residual_forward(norm_rows(x), norm_rows(value(residual)), weight.contiguous(), dense(value(scale_vector)), scale, eps);
}

// ---- delta-rule steps ------------------------------------------------------------------------------------------------

const char* const STEP_NAMES[] = {"step_delta_rule", "step_gated_delta_rule", "step_kda", "step_gdn2"};

Tensor delta_step(int64_t family, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& g, const OptTensor& beta, const OptTensor& b,
                  const OptTensor& w, Tensor state, std::optional<double> scale, const OptTensor& slots, bool qk_norm, double beta_scale, const OptTensor& A_log,
                  const OptTensor& dt_bias, bool state_v_first) {
  WANT(family >= REWY_DELTA && family <= REWY_GDN2, "delta_step: family must be 0 to 3, got ", family);
  const char* op = STEP_NAMES[family];
  WANT(q.dim() == 3 && v.dim() == 3 && q.numel() > 0 && v.numel() > 0, op, ": q, k must have the shape [B, H, K] and v [B, HV, V], got ", shape(q), " and ", shape(v));
  const int64_t B = q.size(0), H = q.size(1), K = q.size(2), HV = v.size(1), V = v.size(2);
  want_most(op, "rows", B, MOST_ROWS);
  want_most(op, "heads", std::max(H, HV), MOST_ROWS);
  want_shape(op, "k", k, {B, H, K});
  WANT(v.size(0) == B && HV % H == 0, op, ": the value heads (", HV, ") must be a multiple of the query/key heads (", H, ") of the same batch");
  WANT(K <= 128 && V <= 128, op, ": head dimensions above 128 are not supported");
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor>("k", k), {"v", v}, {"b", b}, {"w", w}}) want_type(op, name, t, q.scalar_type());
  if (family == REWY_GDN) want_shape(op, "g", g, {B, HV});
  else want_shape(op, "g", g, {B, HV, K});
  want_shape(op, "beta", beta, {B, HV});
  want_shape(op, "b", b, {B, HV, K});
  want_shape(op, "w", w, {B, HV, V});
  want_shape(op, "A_log", A_log, {HV});
  want_shape(op, "dt_bias", dt_bias, {HV * K});
  want_type(op, "A_log", A_log, at::kFloat);
  want_type(op, "dt_bias", dt_bias, at::kFloat);
  WANT(state.dim() == 4 && state.size(0) > 0 && state.size(1) == HV && state.size(2) == (state_v_first ? V : K) && state.size(3) == (state_v_first ? K : V), op,
       ": state must have the shape [pool, ", HV, ", ", state_v_first ? V : K, ", ", state_v_first ? K : V, "], got ", shape(state));
  want_type(op, "state", state, at::kFloat);
  want_state(op, state);
  want_slots(op, slots, B, state.size(0));
  want_no_grad(op, {q, k, v, g, beta, b, w, state, A_log, dt_bias});
  RewyDeltaStepArgs a{};
  a.dtype = dtype_of(q, op, "q");
  a.gate_dtype = has(g) ? dtype_of(*g, op, "g") : a.dtype;
  a.beta_dtype = has(beta) ? dtype_of(*beta, op, "beta") : a.dtype;
  want_cuda(op, {q, k, v, g, beta, b, w, state, slots, A_log, dt_bias});
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous();
  const OptTensor gc = dense(g), bc = dense(beta), ec = dense(b), wc = dense(w), sc = dense(slots), ac = dense(A_log), dc = dense(dt_bias);
  Tensor o = at::empty({B, HV, V}, q.options());
  a.family = (int32_t)family; a.B = (int32_t)B; a.H = (int32_t)H; a.HV = (int32_t)HV; a.K = (int32_t)K; a.V = (int32_t)V;
  a.state_v_first = state_v_first; a.qk_norm = qk_norm; a.slots_i64 = has(sc) && sc->scalar_type() == at::kLong;
  a.scale = (float)(scale.has_value() ? *scale : 1.0 / std::sqrt((double)K));
  a.beta_scale = (float)beta_scale; a.pool = state.size(0);
  a.q = in(qc); a.k = in(kc); a.v = in(vc); a.g = in(gc); a.beta = in(bc); a.b_gate = in(ec); a.w_gate = in(wc); a.slots = in(sc);
  a.A_log = at_ptr<float>(ac); a.dt_bias = at_ptr<float>(dc); a.state = state.data_ptr<float>(); a.o = o.data_ptr();
  check(rewy_delta_step(&a, stream()), op);
  written(state);
  return o;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rewy_b200, m) {
  m.def("causal_conv(Tensor x, Tensor weight, Tensor? bias, bool silu, Tensor? initial_state, bool output_final_state, Tensor? cu_seqlens, "
        "Tensor? cu_seqlens_cpu) -> (Tensor, Tensor)");
  m.def("causal_conv_step(Tensor x, Tensor(a!) state, Tensor weight, Tensor? bias, bool silu, Tensor? slots) -> Tensor");
  m.def("selective_scan(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, bool dt_softplus, Tensor? initial_state, "
        "bool output_final_state, Tensor? cu_seqlens, Tensor? cu_seqlens_cpu) -> (Tensor, Tensor)");
  m.def("selective_scan_step(Tensor u, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor(a!) state, Tensor? D, Tensor? z, Tensor? dt_bias, bool dt_softplus, "
        "Tensor? slots) -> Tensor");
  m.def("gated_rms_norm(Tensor x, Tensor gate, Tensor weight, float eps, int activation, bool gate_first) -> Tensor");
  m.def("residual_rms_norm(Tensor x, Tensor? residual, Tensor weight, Tensor? scale_vector, float scale, float eps) -> (Tensor, Tensor)");
  m.def("delta_step(int family, Tensor q, Tensor k, Tensor v, Tensor? g, Tensor? beta, Tensor? b, Tensor? w, Tensor(a!) state, float? scale, Tensor? slots, "
        "bool qk_norm, float beta_scale, Tensor? A_log, Tensor? dt_bias, bool state_v_first) -> Tensor");
  m.def("layer_backwards() -> int[]", &layer_backwards);
}
TORCH_LIBRARY_IMPL(rewy_b200, CompositeImplicitAutograd, m) {
  m.impl("causal_conv", &causal_conv);
  m.impl("causal_conv_step", &causal_conv_step);
  m.impl("selective_scan", &selective_scan);
  m.impl("selective_scan_step", &selective_scan_step);
  m.impl("gated_rms_norm", &gated_rms_norm);
  m.impl("residual_rms_norm", &residual_rms_norm);
  m.impl("delta_step", &delta_step);
}
