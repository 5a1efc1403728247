// murm_torch.cpp — torch binding of the block operators (fused_linear, qk_norm_rope, rotary).
//
// The operators' calls are short: a projection of a few tokens takes some microseconds on the GPU,
// so their host side (argument checks, allocation, autograd nodes) is compiled. It stays on top of
// the C ABI: the functions of include/murm.h are handed in by address from the one library the
// package has loaded (bind), and every kernel runs through them.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <array>

#include "murm.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---------------------------------------------------------------------------
// the library
// ---------------------------------------------------------------------------
struct Library {
  decltype(&murm_linear_fwd) linear_fwd = nullptr;
  decltype(&murm_linear_bwd) linear_bwd = nullptr;
  decltype(&murm_linear_workspace) linear_workspace = nullptr;
  decltype(&murm_linear_bwd_workspace) linear_bwd_workspace = nullptr;
  decltype(&murm_norm_rope_fwd) norm_rope_fwd = nullptr;
  decltype(&murm_norm_rope_bwd) norm_rope_bwd = nullptr;
  decltype(&murm_norm_rope_workspace) norm_rope_workspace = nullptr;
  decltype(&murm_last_error_message) last_error_message = nullptr;
  decltype(&murm_status_string) status_string = nullptr;
} g_lib;

void bind(const py::dict& addresses) {
  auto set = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::decay_t<decltype(fn)>>(addresses[name].cast<uintptr_t>());
  };
  set(g_lib.linear_fwd, "murm_linear_fwd");
  set(g_lib.linear_bwd, "murm_linear_bwd");
  set(g_lib.linear_workspace, "murm_linear_workspace");
  set(g_lib.linear_bwd_workspace, "murm_linear_bwd_workspace");
  set(g_lib.norm_rope_fwd, "murm_norm_rope_fwd");
  set(g_lib.norm_rope_bwd, "murm_norm_rope_bwd");
  set(g_lib.norm_rope_workspace, "murm_norm_rope_workspace");
  set(g_lib.last_error_message, "murm_last_error_message");
  set(g_lib.status_string, "murm_status_string");
}

void check(murm_status s) {
  if (s == MURM_OK) return;
  const std::string msg = g_lib.last_error_message();
  TORCH_CHECK_TYPE(s != MURM_ERR_DTYPE, msg);
  TORCH_CHECK(false, g_lib.status_string(s), ": ", msg);
}

int dtype_code(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "murmurative CUDA kernels require CUDA tensors; ", name, " is on ", t.device());
  switch (t.scalar_type()) {
    case at::kFloat: return MURM_F32;
    case at::kHalf: return MURM_F16;
    case at::kBFloat16: return MURM_BF16;
    default: TORCH_CHECK_TYPE(false, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  }
}

constexpr int64_t kMaxSize = INT32_MAX;  // of what the C ABI takes in 32 bits, checked before it is cut to them

void same_device(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device(), name, " must be on ", x.device(), ", got ", t.device());
}

// t (if there is one) has x's dtype and device.
void like(const Tensor& t, const Tensor& x, const char* name) {
  if (!t.defined()) return;
  TORCH_CHECK_TYPE(t.scalar_type() == x.scalar_type(), name, " must have x's dtype ", x.scalar_type(), ", got ",
                   t.scalar_type());
  same_device(t, x, name);
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

Tensor bytes_on(const Tensor& like, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

bool defined(const optional<Tensor>& t) { return t.has_value() && t->defined(); }
Tensor value(const optional<Tensor>& t) { return defined(t) ? *t : Tensor(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// The operators run below the dispatcher, which neither forward-mode tangents nor torch.jit.trace see:
// an output without its tangent, or an empty tensor in the traced graph, would pass for a result.
template <typename... T>
void refuse_unseen(const char* name, const T&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!((inputs.defined() && inputs._fw_grad(0).defined()) || ...), name,
                              " has no forward-mode derivative");
  TORCH_CHECK(!torch::jit::tracer::isTracing(), name, " cannot be recorded by torch.jit.trace; torch.compile can");
}

// Gradients of a node that is differentiable once: differentiating them again raises.
variable_list once(variable_list&& grads, const char* name) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  variable_list out;
  for (auto& g : grads) {
    if (!g.defined()) {
      out.emplace_back();
      continue;
    }
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once only", 1);
    out.push_back((*error)({g.detach().requires_grad_(true)})[0]);
  }
  return out;
}

template <typename N>
std::shared_ptr<N> make_node() {
  return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// ---------------------------------------------------------------------------
// fused_linear
// ---------------------------------------------------------------------------
// A 2-D tensor the C ABI reads in place: unit inner stride, rows that do not overlap.
Tensor rows_of(const Tensor& t) {
  const bool ok = (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) == 1 || t.stride(0) >= t.size(1));
  return ok ? t : t.contiguous();
}
int64_t row_stride(const Tensor& t) { return std::max(t.stride(0), t.size(1)); }

// x [M, K], weight [N, K], bias [N], residual [M, N] -> out [M, N], slopes (undefined unless saved)
std::pair<Tensor, Tensor> linear_forward(const Tensor& x_, const Tensor& weight_, const Tensor& bias_,
                                         const Tensor& residual_, int64_t act, bool save) {
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows_of(x_), weight = rows_of(weight_);
  const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
  Tensor out = at::empty({M, N}, x.options()), slope;
  if (save && act != MURM_ACT_NONE)
    slope = at::empty({M, N}, x.options().dtype(x.scalar_type() == at::kFloat ? at::kFloat : at::kShort));
  if (M == 0) return {out, slope};
  Tensor bias, residual;
  murm_linear_args a{};
  a.rows = M;
  a.in_features = static_cast<int32_t>(K);
  a.out_features = static_cast<int32_t>(N);
  a.dtype = dtype_code(x, "x");
  a.activation = static_cast<int32_t>(act);
  a.x = x.data_ptr();
  a.x_stride = row_stride(x);
  a.weight = weight.data_ptr();
  a.w_stride = row_stride(weight);
  if (bias_.defined()) {
    bias = bias_.contiguous();
    a.bias = bias.data_ptr();
  }
  if (residual_.defined()) {
    residual = rows_of(residual_);
    a.residual = residual.data_ptr();
    a.r_stride = row_stride(residual);
  }
  a.out = out.data_ptr();
  a.out_stride = N;
  if (slope.defined()) a.slope = slope.data_ptr();
  Tensor ws;
  check(g_lib.linear_workspace(&a, &a.workspace_bytes));
  if (a.workspace_bytes) {
    ws = bytes_on(x, a.workspace_bytes);
    a.workspace = ws.data_ptr();
  }
  check(g_lib.linear_fwd(&a, stream_of(x)));
  return {out, slope};
}

std::tuple<Tensor, Tensor, Tensor> linear_backward(const Tensor& go_, const Tensor& x_, const Tensor& weight_,
                                                   const Tensor& slope, int64_t act, bool need_x, bool need_w,
                                                   bool need_b) {
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = rows_of(x_), weight = rows_of(weight_), go = rows_of(go_.to(x_.scalar_type()));
  const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
  Tensor gx, gw, gb;
  murm_linear_bwd_args a{};
  a.rows = M;
  a.in_features = static_cast<int32_t>(K);
  a.out_features = static_cast<int32_t>(N);
  a.dtype = dtype_code(x, "x");
  a.activation = static_cast<int32_t>(act);
  a.x = x.data_ptr();
  a.x_stride = row_stride(x);
  a.weight = weight.data_ptr();
  a.w_stride = row_stride(weight);
  if (slope.defined()) a.slope = slope.data_ptr();
  a.grad_out = go.data_ptr();
  a.go_stride = row_stride(go);
  a.gx_stride = a.gw_stride = K;
  if (need_x) {
    gx = at::empty({M, K}, x.options());
    a.grad_x = M ? gx.data_ptr() : nullptr;
  }
  if (need_w) {
    gw = at::empty({N, K}, x.options());
    a.grad_weight = gw.data_ptr();
  }
  if (need_b) {
    gb = at::empty({N}, x.options());
    a.grad_bias = gb.data_ptr();
  }
  Tensor ws;
  check(g_lib.linear_bwd_workspace(&a, &a.workspace_bytes));
  if (a.workspace_bytes) {
    ws = bytes_on(x, a.workspace_bytes);
    a.workspace = ws.data_ptr();
  }
  check(g_lib.linear_bwd(&a, stream_of(x)));
  return {gx, gw, gb};
}

struct FusedLinearBackward : public Node {
  SavedVariable x, weight, slope;
  int64_t act = 0;

  variable_list apply(variable_list&& grads) override {
    variable_list res(4);
    const Tensor& go = grads[0];
    if (!go.defined()) return res;
    refuse_unseen("fused_linear's gradient", go);
    std::lock_guard<std::mutex> lock(mutex_);
    const bool nx = task_should_compute_output(0), nw = task_should_compute_output(1),
               nb = task_should_compute_output(2);
    if (nx || nw || nb)
      std::tie(res[0], res[1], res[2]) =
          linear_backward(go, x.unpack(), weight.unpack(), slope.unpack(), act, nx, nw, nb);
    res = once(std::move(res), "fused_linear");
    if (task_should_compute_output(3)) res[3] = go;
    return res;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    weight.reset_data();
    slope.reset_data();
  }
  std::string name() const override { return "FusedLinearBackward"; }
};

int64_t activation_code(const std::string& name) {
  static const char* const names[] = {"none", "relu", "silu", "gelu", "gelu_tanh"};
  for (int64_t i = 0; i < 5; ++i)
    if (name == names[i]) return i;
  TORCH_CHECK_VALUE(false, "activation must be one of none, relu, silu, gelu, gelu_tanh, got '", name, "'");
}

// The arguments of every entry, the registered operators' too: the kernels take pointers and x's and
// the weight's sizes. The residual's shape is the entry's to check.
void check_linear(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual) {
  dtype_code(x, "x");
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1),
              "x must be [..., K] and weight [N, K], got ", x.sizes(), " and ", weight.sizes());
  const int64_t N = weight.size(0), K = weight.size(1);
  TORCH_CHECK(N >= 1 && K >= 1, "weight must not be empty, got ", weight.sizes());
  TORCH_CHECK(N <= kMaxSize && K <= kMaxSize, "features must be below 2^31, got ", weight.sizes());
  like(weight, x, "weight");
  like(bias, x, "bias");
  like(residual, x, "residual");
  TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == N), "bias must be [N=", N, "], got ",
              bias.sizes());
}

Tensor fused_linear(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias_, const std::string& activation,
                    const optional<Tensor>& residual_) {
  const int64_t act = activation_code(activation);
  const Tensor bias = value(bias_);
  Tensor residual = value(residual_);
  check_linear(x, weight, bias, residual);
  refuse_unseen("fused_linear", x, weight, bias, residual);
  const int64_t N = weight.size(0), K = weight.size(1);
  const bool flat = x.dim() == 2;
  auto shape = x.sizes().vec();
  shape.back() = N;
  const Tensor x2 = flat ? x : x.reshape({-1, K});
  if (residual.defined()) {
    if (residual.sizes() != c10::IntArrayRef(shape)) {
      TORCH_CHECK(at::is_expandable_to(residual.sizes(), shape), "residual must broadcast to ", c10::IntArrayRef(shape),
                  ", got ", residual.sizes());
      residual = residual.expand(shape);
    }
    if (residual.dim() != 2) residual = residual.reshape({-1, N});
  }
  Tensor out, slope;
  if (at::GradMode::is_enabled() &&
      (wants_grad(x2) || wants_grad(weight) || wants_grad(bias) || wants_grad(residual))) {
    auto node = make_node<FusedLinearBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x2, weight, bias, residual));
    const bool save = wants_grad(x2) || wants_grad(weight) || wants_grad(bias);  // the residual's gradient needs none
    std::tie(out, slope) = linear_forward(x2, weight, bias, residual, act, save);
    node->act = act;
    node->x = SavedVariable(x2, false);
    node->weight = SavedVariable(weight, false);
    node->slope = SavedVariable(slope, false);
    torch::autograd::set_history(out, node);
  } else {
    out = linear_forward(x2, weight, bias, residual, act, false).first;
  }
  return flat ? out : out.view(shape);
}

// ---------------------------------------------------------------------------
// qk_norm_rope, rotary
// ---------------------------------------------------------------------------
// Everything about a rotation except its rows and gains.
struct Rotation {
  Tensor positions, freqs;
  murm_norm_rope_args args{};  // all but batch, tokens, dtype, rows and workspace
};

void check_rows(const Tensor& t, const char* name) {
  dtype_code(t, name);
  TORCH_CHECK(t.dim() == 4, name, " must be 4-D [B, H, N, head_dim], got shape ", t.sizes());
  for (const int64_t n : t.sizes()) TORCH_CHECK(n <= kMaxSize, name, "'s sizes must be below 2^31, got ", t.sizes());
}

Rotation make_rotation(const Tensor& x, const Tensor& positions, double base, optional<int64_t> rotary_dim,
                       bool interleaved, const optional<std::vector<int64_t>>& sections, const std::string& spectrum,
                       const optional<Tensor>& freqs, double eps) {
  Rotation r;
  auto& a = r.args;
  const int64_t B = x.size(0), N = x.size(2), d = x.size(3);
  const int64_t rd = rotary_dim.value_or(d);
  TORCH_CHECK(rd >= 0 && rd <= d && rd % 2 == 0, "rotary_dim must be even and in 0..", d, ", got ", rd);
  TORCH_CHECK_VALUE(spectrum == "shared" || spectrum == "own", "spectrum must be 'shared' or 'own', got '", spectrum,
                    "'");
  switch (positions.scalar_type()) {
    case at::kLong: a.position_type = MURM_POS_I64; break;
    case at::kInt: a.position_type = MURM_POS_I32; break;
    case at::kFloat: a.position_type = MURM_POS_F32; break;
    default: TORCH_CHECK_TYPE(false, "positions must be an int64, int32 or float32 tensor, got ", positions.scalar_type());
  }
  same_device(positions, x, "positions");
  a.axes = 1;
  int64_t inner = 0;  // axes, as the positions' last dimension
  if (sections.has_value()) {
    int64_t sum = 0;
    bool ok = sections->size() >= 1 && sections->size() <= 4;
    for (const int64_t s : *sections) {
      ok = ok && s >= 0;
      sum += s;
    }
    TORCH_CHECK(ok && sum == rd / 2, "sections must be 1 to 4 counts of pairs that add up to rotary_dim/2 = ", rd / 2,
                ", got ", c10::IntArrayRef(*sections));
    inner = a.axes = static_cast<int32_t>(sections->size());
    for (int i = 0; i < a.axes; ++i) a.sections[i] = static_cast<int32_t>((*sections)[i]);
  }
  const int64_t dims = 1 + (inner ? 1 : 0), got = positions.dim(), lead = got - dims;
  const bool fits = (lead == 0 || lead == 1) && positions.size(lead) == N && (!inner || positions.size(lead + 1) == inner) &&
                    (lead == 0 || positions.size(0) == B || positions.size(0) == 1);
  if (!fits) {
    std::vector<int64_t> want{N};
    if (inner) want.push_back(inner);
    std::vector<int64_t> batched(want);
    batched.insert(batched.begin(), B);
    TORCH_CHECK(false, "positions must be ", c10::IntArrayRef(want), " or ", c10::IntArrayRef(batched), ", got ",
                positions.sizes());
  }
  a.position_stride[0] = lead == 1 && positions.size(0) != 1 ? positions.stride(0) : 0;
  a.position_stride[1] = positions.stride(lead);
  a.position_stride[2] = inner ? positions.stride(lead + 1) : 0;
  r.positions = positions;
  if (defined(freqs)) {
    TORCH_CHECK(freqs->scalar_type() == at::kFloat && freqs->dim() == 1 && freqs->size(0) == rd / 2,
                "freqs must be a float32 tensor of rotary_dim/2 = ", rd / 2, " elements");
    same_device(*freqs, x, "freqs");
    r.freqs = freqs->contiguous();
  }
  a.head_dim = static_cast<int32_t>(d);
  a.rotary_dim = static_cast<int32_t>(rd);
  a.interleaved = interleaved;
  a.own_spectrum = spectrum == "own";
  a.base = base;
  a.eps = eps;
  return r;
}

Tensor gain(const optional<Tensor>& w, const Tensor& x, const char* name) {
  if (!defined(w)) return Tensor();
  dtype_code(*w, name);
  TORCH_CHECK_TYPE(w->scalar_type() == x.scalar_type() || w->scalar_type() == at::kFloat, name, " must be float32 or ",
                   x.scalar_type(), ", got ", w->scalar_type());
  TORCH_CHECK(w->dim() == 1 && w->size(0) == x.size(3), name, " must be [head_dim=", x.size(3), "], got ", w->sizes());
  same_device(*w, x, name);
  return w->contiguous();
}

// A result for t's rows, in their layout. Overlapping rows (a sliding window: token and element both of
// stride 1) have none to keep, and empty_like's guess may put the tokens innermost.
Tensor empty_rows(const Tensor& t) {
  Tensor out = at::empty_like(t);
  return out.stride(3) == 1 ? out : at::empty_like(t, at::MemoryFormat::Contiguous);
}
Tensor unit_rows(const Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); }
void set_strides(int64_t (&dst)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) dst[i] = t.stride(i);
}

murm_norm_rope_args call_args(const Rotation& r, const Tensor& x, bool normalize, bool inverse) {
  murm_norm_rope_args a = r.args;
  a.batch = static_cast<int32_t>(x.size(0));
  a.tokens = static_cast<int32_t>(x.size(2));
  a.dtype = dtype_code(x, "x");
  a.normalize = normalize;
  a.inverse = inverse;
  a.positions = r.positions.data_ptr();
  if (r.freqs.defined()) a.freqs = static_cast<const float*>(r.freqs.data_ptr());
  return a;
}
void set_rows(murm_head_rows& dst, const Tensor& x, const Tensor& out, const Tensor& weight) {
  dst.x = x.data_ptr();
  set_strides(dst.x_stride, x);
  dst.out = out.data_ptr();
  set_strides(dst.out_stride, out);
  dst.heads = static_cast<int32_t>(x.size(1));
  if (weight.defined()) {
    dst.weight = weight.data_ptr();
    dst.weight_dtype = dtype_code(weight, "weight");
  }
}

// The rotation alone of x's rows.
Tensor rotate(const Tensor& x_, const Rotation& r, bool inverse) {
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = unit_rows(x_);
  Tensor out = empty_rows(x);
  if (x.numel()) {
    murm_norm_rope_args a = call_args(r, x, false, inverse);
    set_rows(a.q, x, out, Tensor());
    check(g_lib.norm_rope_fwd(&a, stream_of(x)));
  }
  return out;
}

std::pair<Tensor, Tensor> norm_rope_forward(const Tensor& q_, const Tensor& k_, const Tensor& qw, const Tensor& kw,
                                            const Rotation& r) {
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(q_.device());
  const Tensor q = unit_rows(q_), k = k_.defined() ? unit_rows(k_) : k_;
  Tensor oq = empty_rows(q), ok = k.defined() ? empty_rows(k) : Tensor();
  if (q.numel() || (k.defined() && k.numel())) {
    murm_norm_rope_args a = call_args(r, q, true, false);
    set_rows(a.q, q, oq, qw);
    if (k.defined()) set_rows(a.k, k, ok, kw);
    check(g_lib.norm_rope_fwd(&a, stream_of(q)));
  }
  return {oq, ok};
}

// Gradients of q, k and the gains. need: q, k, q's gain, k's gain; a tensor of which neither is needed is
// left out, and so is the sum for a gain alone that is not.
variable_list norm_rope_backward(const Tensor (&x_)[2], const Tensor (&w)[2], const Tensor (&go_)[2],
                                 const std::array<bool, 4>& need, const Rotation& r) {
  at::NoGradGuard no_grad;
  const c10::cuda::CUDAGuard guard(x_[0].device());
  murm_norm_rope_args a = call_args(r, x_[0], true, false);
  murm_head_rows* rows[2] = {&a.q, &a.k};
  Tensor x[2], go[2], gx[2], gw[2];
  bool any = false, sums = false;
  for (int t = 0; t < 2; ++t) {
    const bool gain = w[t].defined() && need[2 + t];
    if (!x_[t].defined() || !(need[t] || gain)) continue;
    x[t] = unit_rows(x_[t]);
    gx[t] = empty_rows(x[t]);
    if (x[t].numel() == 0) {  // no rows: gain gradients are sums of nothing
      if (gain) gw[t] = at::zeros_like(w[t]);
      continue;
    }
    go[t] = unit_rows(go_[t].to(x[t].scalar_type()));
    set_rows(*rows[t], x[t], gx[t], w[t]);
    rows[t]->grad = go[t].data_ptr();
    set_strides(rows[t]->grad_stride, go[t]);
    if (gain) {
      gw[t] = at::empty_like(w[t]);
      rows[t]->grad_weight = gw[t].data_ptr();
      sums = true;
    }
    any = true;
  }
  Tensor ws;
  if (sums) {
    a.workspace_bytes = g_lib.norm_rope_workspace();
    ws = bytes_on(x_[0], a.workspace_bytes);
    a.workspace = ws.data_ptr();
  }
  if (any) check(g_lib.norm_rope_bwd(&a, stream_of(x_[0])));
  return {gx[0], gx[1], gw[0], gw[1]};
}

struct QkNormRopeBackward : public Node {
  SavedVariable q, k, qw, kw, positions, freqs;
  Rotation r;  // without its tensors

  variable_list apply(variable_list&& grads) override {
    for (const auto& go : grads) refuse_unseen("qk_norm_rope's gradient", go);
    std::lock_guard<std::mutex> lock(mutex_);
    Rotation now = r;
    now.positions = positions.unpack();
    now.freqs = freqs.unpack();
    const Tensor x[2] = {q.unpack(), k.unpack()}, w[2] = {qw.unpack(), kw.unpack()};
    const std::array<bool, 4> need{task_should_compute_output(0), task_should_compute_output(1),
                                   task_should_compute_output(2), task_should_compute_output(3)};
    Tensor go[2];
    for (int t = 0; t < 2; ++t)
      if (x[t].defined() && (need[t] || need[2 + t])) go[t] = grads[t].defined() ? grads[t] : at::zeros_like(x[t]);
    return once(norm_rope_backward(x, w, go, need, now), "qk_norm_rope");
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&q, &k, &qw, &kw, &positions, &freqs}) v->reset_data();
  }
  std::string name() const override { return "QkNormRopeBackward"; }
};

// q and k of every entry.
void check_qk(const Tensor& q, const Tensor& k) {
  check_rows(q, "q");
  if (!k.defined()) return;
  check_rows(k, "k");
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), "q and k must share a dtype, got ", q.scalar_type(), " and ",
                   k.scalar_type());
  same_device(k, q, "k");
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2) && k.size(3) == q.size(3), "k must be [B=", q.size(0),
              ", Hk, N=", q.size(2), ", d=", q.size(3), "], got ", k.sizes());
}

std::pair<Tensor, optional<Tensor>> qk_norm_rope(const Tensor& q, const optional<Tensor>& k_, const Tensor& positions,
                                                 const optional<Tensor>& q_weight, const optional<Tensor>& k_weight,
                                                 double eps, double base, optional<int64_t> rotary_dim, bool interleaved,
                                                 const optional<std::vector<int64_t>>& sections,
                                                 const std::string& spectrum, const optional<Tensor>& freqs) {
  const Tensor k = value(k_);
  check_qk(q, k);
  TORCH_CHECK(k.defined() || !defined(k_weight), "k_weight given without k");
  const Tensor qw = gain(q_weight, q, "q_weight"), kw = k.defined() ? gain(k_weight, k, "k_weight") : Tensor();
  refuse_unseen("qk_norm_rope", q, k, qw, kw);
  Rotation r = make_rotation(q, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, eps);
  auto [oq, ok] = norm_rope_forward(q, k, qw, kw, r);
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(qw) || wants_grad(kw))) {
    auto node = make_node<QkNormRopeBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, qw, kw));
    node->q = SavedVariable(q, false);
    node->k = SavedVariable(k, false);
    node->qw = SavedVariable(qw, false);
    node->kw = SavedVariable(kw, false);
    node->positions = SavedVariable(r.positions, false);
    node->freqs = SavedVariable(r.freqs, false);
    node->r.args = r.args;
    torch::autograd::set_history(oq, node);
    if (ok.defined()) torch::autograd::set_history(ok, node);
  }
  return {oq, ok.defined() ? optional<Tensor>(ok) : std::nullopt};
}

Tensor rotary_apply(const Tensor& x, const Rotation& r, bool inverse);

struct RotaryBackward : public Node {
  SavedVariable positions, freqs;
  Rotation r;
  bool inverse = false;

  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return {Tensor()};
    std::lock_guard<std::mutex> lock(mutex_);
    Rotation now = r;
    now.positions = positions.unpack();
    now.freqs = freqs.unpack();
    return {rotary_apply(grads[0], now, !inverse)};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    positions.reset_data();
    freqs.reset_data();
  }
  std::string name() const override { return "RotaryBackward"; }
};

Tensor rotary_apply(const Tensor& x, const Rotation& r, bool inverse) {
  refuse_unseen("rotary", x);
  Tensor out = rotate(x, r, inverse);
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    auto node = make_node<RotaryBackward>();
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->positions = SavedVariable(r.positions, false);
    node->freqs = SavedVariable(r.freqs, false);
    node->r.args = r.args;
    node->inverse = inverse;
    torch::autograd::set_history(out, node);
  }
  return out;
}

Tensor rotary(const Tensor& x, const Tensor& positions, double base, optional<int64_t> rotary_dim, bool interleaved,
              const optional<std::vector<int64_t>>& sections, const std::string& spectrum,
              const optional<Tensor>& freqs, bool inverse) {
  check_rows(x, "x");
  return rotary_apply(x, make_rotation(x, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, 0.0),
                      inverse);
}

// ---------------------------------------------------------------------------
// the passes without autograd, for the registered operators (torch_ops.py)
// ---------------------------------------------------------------------------
Tensor or_empty(const Tensor& t, const Tensor& like) { return t.defined() ? t : at::empty({0}, like.options()); }

void check_rows_2d(const Tensor& x) { TORCH_CHECK(x.dim() == 2, "x must be [M, K], got ", x.sizes()); }

std::tuple<Tensor, Tensor> linear_fwd(const Tensor& x, const Tensor& weight, const optional<Tensor>& bias,
                                      const std::string& activation, const optional<Tensor>& residual_, bool save) {
  const int64_t act = activation_code(activation);
  const Tensor residual = value(residual_);
  check_linear(x, weight, value(bias), residual);
  check_rows_2d(x);
  TORCH_CHECK(!residual.defined() || (residual.dim() == 2 && residual.size(0) == x.size(0) &&
                                      residual.size(1) == weight.size(0)),
              "residual must be [M=", x.size(0), ", N=", weight.size(0), "], got ", residual.sizes());
  auto [out, slope] = linear_forward(x, weight, value(bias), residual, act, save);
  return {out, or_empty(slope, x)};
}
std::tuple<Tensor, Tensor, Tensor> linear_bwd(const Tensor& go, const Tensor& x, const Tensor& weight,
                                              const Tensor& slope, const std::string& activation, bool need_x,
                                              bool need_weight, bool need_bias) {
  const int64_t act = activation_code(activation);
  check_linear(x, weight, Tensor(), go);
  check_rows_2d(x);
  const std::array<int64_t, 2> sizes{x.size(0), weight.size(0)};
  const c10::IntArrayRef shape(sizes);
  TORCH_CHECK(go.sizes() == shape, "grad_out must be ", shape, ", got ", go.sizes());
  if (act != MURM_ACT_NONE) {
    const at::ScalarType type = x.scalar_type() == at::kFloat ? at::kFloat : at::kShort;
    TORCH_CHECK_TYPE(slope.scalar_type() == type, "slope must be ", type, " beside ", x.scalar_type(), ", got ",
                     slope.scalar_type());
    same_device(slope, x, "slope");
    TORCH_CHECK(slope.sizes() == shape && slope.is_contiguous(), "slope must be contiguous and ", shape, ", got ",
                slope.sizes());
  }
  const auto [gx, gw, gb] =
      linear_backward(go, x, weight, act != MURM_ACT_NONE ? slope : Tensor(), act, need_x, need_weight, need_bias);
  return {or_empty(gx, x), or_empty(gw, x), or_empty(gb, x)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> qk_bwd(const Tensor& gq, const Tensor& gk, const Tensor& q,
                                                  const optional<Tensor>& k_, const Tensor& positions,
                                                  const optional<Tensor>& q_weight, const optional<Tensor>& k_weight,
                                                  double eps, double base, optional<int64_t> rotary_dim,
                                                  bool interleaved, const optional<std::vector<int64_t>>& sections,
                                                  const std::string& spectrum, const optional<Tensor>& freqs,
                                                  const std::array<bool, 4>& need) {
  const Tensor k = value(k_);
  check_qk(q, k);
  like(gq, q, "grad_q");
  TORCH_CHECK(gq.sizes() == q.sizes(), "grad_q must be ", q.sizes(), ", got ", gq.sizes());
  if (k.defined()) {
    like(gk, k, "grad_k");
    TORCH_CHECK(gk.sizes() == k.sizes(), "grad_k must be ", k.sizes(), ", got ", gk.sizes());
  }
  const Tensor x[2] = {q, k};
  const Tensor w[2] = {gain(q_weight, q, "q_weight"), k.defined() ? gain(k_weight, k, "k_weight") : Tensor()};
  const Tensor go[2] = {gq, gk};
  const auto res = norm_rope_backward(
      x, w, go, need, make_rotation(q, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, eps));
  return {or_empty(res[0], q), or_empty(res[1], q), or_empty(res[2], q), or_empty(res[3], q)};
}

}  // namespace

PYBIND11_MODULE(_murm_torch, m) {
  m.doc() = "torch binding of the block operators over the murm C ABI";
  m.def("bind", &bind);
  m.def("fused_linear", &fused_linear);
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("rotary", &rotary);
  m.def("linear_fwd", &linear_fwd, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("activation"),
        py::arg("residual"), py::arg("save") = true);
  m.def("linear_bwd", &linear_bwd, py::arg("grad_out"), py::arg("x"), py::arg("weight"), py::arg("slope"),
        py::arg("activation"), py::arg("need_x") = true, py::arg("need_weight") = true, py::arg("need_bias") = true);
  m.def("qk_bwd", &qk_bwd, py::arg("grad_q"), py::arg("grad_k"), py::arg("q"), py::arg("k"), py::arg("positions"),
        py::arg("q_weight"), py::arg("k_weight"), py::arg("eps"), py::arg("base"), py::arg("rotary_dim"),
        py::arg("interleaved"), py::arg("sections"), py::arg("spectrum"), py::arg("freqs"),
        py::arg("need") = std::array<bool, 4>{true, true, true, true});
}
