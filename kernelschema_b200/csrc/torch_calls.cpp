// The 8-bit operators and the token sorting as calls on torch tensors: checks of arguments, output tensors, device and stream, then one call
// of the C ABI (include/b200moe.h). In C++ because these calls are short (a token's norm takes 2 us on the device): the same checks
// and allocations take 12 us in Python and 3 us here. Nothing is computed here and nothing kept between calls.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "../../include/b200moe.h"

namespace py = pybind11;
using at::ScalarType;
using at::Tensor;
using Maybe = std::optional<Tensor>;

namespace {

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }

void check(int code, const char* what) {
  if (code == 0) return;
  const std::string text = b200moe_last_error();
  if (code >= 700 && code < 800) refuse(std::string(what) + ": " + text + " (code " + std::to_string(code) + ")");
  throw std::runtime_error(std::string(what) + " failed: " + text + " (code " + std::to_string(code) + ")");
}

int row_type(ScalarType t) {
  return t == at::kBFloat16 ? B200MOE_BF16 : t == at::kHalf ? B200MOE_FP16 : t == at::kFloat ? B200MOE_FP32 : -1;
}
int code_type(ScalarType t) { return t == at::kChar ? B200MOE_INT8 : t == at::kFloat8_e4m3fn ? B200MOE_E4M3 : -1; }

std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// The tensors of a call are on one CUDA device, which becomes the current one for its duration; its current stream takes the launches.
struct Here {
  c10::DeviceIndex index = -1;
  std::optional<c10::cuda::CUDAGuard> guard;
  void add(const Tensor& t) {
    if (!t.is_cuda()) refuse("libb200moe operates on CUDA tensors only");
    if (index < 0) index = t.device().index();
    if (t.device().index() != index) refuse("the tensors of a call must be on one device");
  }
  void add(const Maybe& t) {
    if (t) add(*t);
  }
  template <class... Ts>
  explicit Here(const Ts&... ts) {
    (add(ts), ...);
    guard.emplace(index);
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(index).stream(); }
};

template <class T = void>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <class T = void>
T* ptr(const Maybe& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

Tensor unit_rows(const Tensor& x) { return x.stride(1) == 1 || x.size(1) == 1 ? x : x.contiguous(); }
// Elements between rows; a single row has no next one, whatever its stride says.
int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }
int64_t row_stride(const Maybe& x) { return x ? row_stride(*x) : 0; }

Tensor fresh(at::IntArrayRef shape, ScalarType type, const Tensor& like) { return at::detail::empty_cuda(shape, type, like.device(), std::nullopt); }

// A caller's buffer for rows, or a vector with one value per row, checked; or a new one.
Tensor out_rows(const Maybe& out, int64_t rows, int64_t cols, ScalarType type, const char* name, const Tensor& like) {
  if (!out) return fresh({rows, cols}, type, like);
  if (out->scalar_type() != type || out->dim() != 2 || out->size(0) != rows || out->size(1) != cols || (cols > 1 && out->stride(1) != 1) ||
      (rows > 1 && out->stride(0) < cols))
    refuse(std::string(name) + " must be " + c10::toString(type) + " [" + std::to_string(rows) + ", " + std::to_string(cols) +
           "] with unit inner stride and rows that do not overlap");
  return *out;
}
Tensor out_values(const Maybe& out, int64_t n, const char* name, const Tensor& like) {
  if (!out) return fresh({n}, at::kFloat, like);
  if (out->scalar_type() != at::kFloat || out->dim() != 1 || out->size(0) != n || !out->is_contiguous())
    refuse(std::string(name) + " must be contiguous float32 [" + std::to_string(n) + "]");
  return *out;
}

bool wants_gradient(const Tensor& t) { return t.requires_grad(); }
bool wants_gradient(const Maybe& t) { return t && t->requires_grad(); }
// Whether t carries a tangent that forward-mode differentiation asks for. A dual tensor does not require a gradient, and the kernels read its
// primal part alone.
bool has_tangent(const Tensor& t) { return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined(); }
bool has_tangent(const Maybe& t) { return t && has_tangent(*t); }

// The 8-bit operators have no derivative: tensors that ask for one are refused, their results would come without it.
template <class... Ts>
void no_derivative(const char* what, const Ts&... ts) {
  if (at::GradMode::is_enabled() && (wants_gradient(ts) || ...))
    refuse(std::string(what) + " has no gradient: pass detached tensors, or call it under torch.no_grad()");
  if ((has_tangent(ts) || ...)) refuse(std::string(what) + " has no forward-mode derivative");
}

int wanted_codes(ScalarType dtype) {
  const int code = code_type(dtype);
  if (code < 0) refuse("dtype must be torch.int8 or torch.float8_e4m3fn");
  return code;
}

std::tuple<Tensor, Tensor, Tensor, Maybe> rmsnorm_quantize(const Tensor& x_in, const Tensor& weight_in, const Maybe& residual_in, double eps, ScalarType dtype,
                                                           bool normed, const Maybe& q_out, const Maybe& scale_out, const Maybe& hidden_out,
                                                           const Maybe& norm_out) {
  const int rows = row_type(x_in.scalar_type());
  if (x_in.dim() != 2 || rows < 0 || (residual_in && (residual_in->scalar_type() != x_in.scalar_type() || residual_in->sizes() != x_in.sizes())))
    refuse("rmsnorm_quantize expects bf16, fp16 or fp32 [T, H] and a residual like it");
  const int64_t t = x_in.size(0), h = x_in.size(1);
  if (weight_in.dim() != 1 || weight_in.size(0) != h || (weight_in.scalar_type() != x_in.scalar_type() && weight_in.scalar_type() != at::kFloat))
    refuse("weight must be [" + std::to_string(h) + "] in x's type or float32");
  const int code = wanted_codes(dtype);
  no_derivative("rmsnorm_quantize", x_in, weight_in, residual_in, q_out, scale_out, hidden_out, norm_out);
  const Here here(x_in, weight_in, residual_in, q_out, scale_out, hidden_out, norm_out);
  const Tensor x = unit_rows(x_in), weight = weight_in.contiguous();
  const Maybe residual = residual_in ? Maybe(unit_rows(*residual_in)) : Maybe();
  const Tensor q = out_rows(q_out, t, h, dtype, "q", x), scale = out_values(scale_out, t, "scale", x);
  Maybe hidden, norm;
  if (residual || hidden_out) hidden = out_rows(hidden_out, t, h, x.scalar_type(), "hidden", x);
  if (normed || norm_out) norm = out_rows(norm_out, t, h, x.scalar_type(), "normed", x);
  check(b200moe_rmsnorm_quantize(ptr(x), row_stride(x), ptr(residual), row_stride(residual), ptr(weight), row_type(weight.scalar_type()), t, h, (float)eps, rows,
                                 code, ptr(q), row_stride(q), ptr<float>(scale), ptr(hidden), row_stride(hidden), ptr(norm), row_stride(norm), here.stream()),
        "b200moe_rmsnorm_quantize");
  return {q, scale, hidden ? *hidden : x_in, norm};
}

std::tuple<Tensor, Tensor> swiglu_quantize(const Tensor& x_in, ScalarType dtype, const Maybe& q_out, const Maybe& scale_out) {
  const int rows = row_type(x_in.scalar_type());
  if (x_in.dim() != 2 || rows < 0 || x_in.size(1) % 2 || !x_in.size(1)) refuse("swiglu_quantize expects bf16, fp16 or fp32 [T, 2I]");
  const int code = wanted_codes(dtype);
  no_derivative("swiglu_quantize", x_in, q_out, scale_out);
  const Here here(x_in, q_out, scale_out);
  const Tensor x = unit_rows(x_in);
  const int64_t t = x.size(0), i = x.size(1) / 2;
  const Tensor q = out_rows(q_out, t, i, dtype, "q", x), scale = out_values(scale_out, t, "scale", x);
  check(b200moe_swiglu_quantize(ptr(x), row_stride(x), t, i, rows, code, ptr(q), row_stride(q), ptr<float>(scale), here.stream()), "b200moe_swiglu_quantize");
  return {q, scale};
}

// offsets: null for one product, else segments of rows with a weight matrix each.
Tensor mm_8bit(const Tensor& a_in, const Tensor& a_scale_in, const Tensor& b, const Tensor& b_scale_in, const Maybe& offsets_in, const Maybe& out_in,
               ScalarType out_dtype, const Maybe& status) {
  const int code = code_type(a_in.scalar_type());
  const int64_t lead = offsets_in ? 1 : 0;
  if (a_in.dim() != 2 || b.dim() != 2 + lead || code < 0 || b.scalar_type() != a_in.scalar_type())
    refuse(lead ? "a [M, K] and b [E, N, K] must both be int8 or both float8_e4m3fn" : "a [M, K] and b [N, K] must both be int8 or both float8_e4m3fn");
  const int64_t m = a_in.size(0), k = a_in.size(1), n = b.size(lead), experts = lead ? b.size(0) : 0;
  if (b.size(lead + 1) != k || k % 16 || !k || !n) refuse("a " + shape_of(a_in) + " and b " + shape_of(b) + " must share K, a multiple of 16");
  if (offsets_in && (offsets_in->scalar_type() != at::kInt || offsets_in->dim() != 1 || offsets_in->size(0) != experts + 1))
    refuse("offsets must be int32 [E + 1]");
  if (a_scale_in.scalar_type() != at::kFloat || a_scale_in.numel() != m || b_scale_in.scalar_type() != at::kFloat || b_scale_in.numel() != b.numel() / k)
    refuse("a_scale must hold one fp32 value per row of a, b_scale one per row of b");
  if (out_in) out_dtype = out_in->scalar_type();
  const int out_type = row_type(out_dtype);
  if (out_type < 0) refuse("the output must be bfloat16, float16 or float32");
  if (status && (status->scalar_type() != at::kInt || !status->numel())) refuse("status must be an int32 tensor");
  no_derivative(lead ? "mm_8bit_grouped" : "mm_8bit", a_in, a_scale_in, b, b_scale_in, out_in);
  const Here here(a_in, a_scale_in, b, b_scale_in, offsets_in, out_in, status);
  Tensor a = unit_rows(a_in);
  if (row_stride(a) < k || row_stride(a) % 16 || (uintptr_t)a.data_ptr() % 16) a = a.clone(at::MemoryFormat::Contiguous);
  if (!b.is_contiguous() || (uintptr_t)b.data_ptr() % 16) refuse("b must be contiguous and 16-byte aligned");
  const Tensor a_scale = a_scale_in.contiguous(), b_scale = b_scale_in.contiguous(), out = out_rows(out_in, m, n, out_dtype, "out", a);
  if (!offsets_in) {
    check(b200moe_gemm_8bit(ptr(a), row_stride(a), ptr<float>(a_scale), ptr(b), ptr<float>(b_scale), ptr(out), m, n, k, row_stride(out), code, out_type,
                            ptr<int32_t>(status), here.stream()),
          "b200moe_gemm_8bit");
  } else {
    const Tensor offsets = offsets_in->contiguous();
    check(b200moe_gemm_8bit_grouped(ptr(a), row_stride(a), ptr<float>(a_scale), ptr(b), ptr<float>(b_scale), ptr<int32_t>(offsets), (int32_t)experts, ptr(out), m,
                                    n, k, row_stride(out), code, out_type, !out_in, ptr<int32_t>(status), here.stream()),
          "b200moe_gemm_8bit_grouped");
  }
  return out;
}

std::tuple<Tensor, Tensor, Tensor> route_sort(const Tensor& ids_in, int64_t num_experts) {
  if (ids_in.dim() != 2 || ids_in.scalar_type() != at::kInt || !ids_in.size(1)) refuse("ids must be int32 [T, top_k]");
  if (num_experts <= 0 || num_experts > 1024) refuse("num_experts must be in 1..1024");
  const Here here(ids_in);
  const Tensor ids = unit_rows(ids_in);
  const int64_t t = ids.size(0), k = ids.size(1), n = t * k;
  const int64_t need = b200moe_route_sort_workspace_bytes(t, (int32_t)k, (int32_t)num_experts);
  if (need < 0) refuse(std::string("route_sort: ") + b200moe_last_error());
  const Tensor offsets = fresh({num_experts + 1}, at::kInt, ids), row_of = fresh({t, k}, at::kInt, ids);
  // The workspace lies behind route_of_row: a graph that was not captured by torch has no pool that would keep a buffer of this call alone.
  const Tensor last = fresh({n + need / 4}, at::kInt, ids), route_of_row = need ? last.narrow(0, 0, n) : last;
  check(b200moe_route_sort(ptr<int32_t>(ids), row_stride(ids), t, (int32_t)k, (int32_t)num_experts, ptr<int32_t>(offsets), ptr<int32_t>(row_of),
                           ptr<int32_t>(route_of_row), need ? ptr<int32_t>(last) + n : nullptr, need, here.stream()),
        "b200moe_route_sort");
  return {offsets, row_of, route_of_row};
}

// Tables of a sorted order that fits `tokens` tokens, or `rows` rows (-1: not asked).
void check_order(const Tensor& offsets, const Tensor& row_of, int64_t tokens, int64_t rows) {
  if (row_of.dim() != 2 || row_of.scalar_type() != at::kInt || offsets.scalar_type() != at::kInt || offsets.dim() != 1 || !offsets.size(0) ||
      !row_of.is_contiguous() || !offsets.is_contiguous() || !row_of.size(1))
    refuse("order must come from route_sort");
  if ((tokens >= 0 && row_of.size(0) != tokens) || (rows >= 0 && row_of.numel() != rows))
    refuse("the order is of " + std::to_string(row_of.size(0)) + " tokens and " + std::to_string(row_of.numel()) + " rows, the tensor has " +
           std::to_string(tokens >= 0 ? tokens : rows));
}
const int32_t* valid_rows(const Tensor& offsets) { return ptr<int32_t>(offsets) + offsets.size(0) - 1; }

Tensor sort_rows(const Tensor& x_in, const Tensor& offsets, const Tensor& row_of) {
  if ((x_in.dim() != 1 && x_in.dim() != 2) || x_in.element_size() > 4 || x_in.is_complex() || (x_in.dim() == 2 && !x_in.size(1)))
    refuse("sort_tokens expects [T, H] or [T] of a 1-, 2- or 4-byte type");
  check_order(offsets, row_of, x_in.size(0), -1);
  const Here here(x_in, offsets, row_of);
  const Tensor x = unit_rows(x_in.dim() == 1 ? x_in.unsqueeze(1) : x_in);
  const int64_t t = row_of.size(0), k = row_of.size(1), size = x.element_size();
  const Tensor rows = x_in.dim() == 1 ? fresh({t * k}, x.scalar_type(), x) : fresh({t * k, x.size(1)}, x.scalar_type(), x);
  check(b200moe_sort_rows(ptr(x), row_stride(x) * size, t, x.size(1) * size, ptr<int32_t>(row_of), (int32_t)k, valid_rows(offsets), ptr(rows), here.stream()),
        "b200moe_sort_rows");
  return rows;
}

void check_rows(const Tensor& rows, const Tensor& offsets, const Tensor& row_of, const Maybe& weights) {
  if (rows.dim() != 2 || row_type(rows.scalar_type()) < 0 || !rows.size(1)) refuse("unsort_tokens expects bf16, fp16 or fp32 [T * top_k, H]");
  check_order(offsets, row_of, -1, rows.size(0));
  if (weights && (weights->scalar_type() != at::kFloat || weights->sizes() != row_of.sizes())) refuse("weights must be float32 " + shape_of(row_of));
}

Tensor unsort_rows(const Tensor& rows_in, const Tensor& offsets, const Tensor& row_of, const Maybe& weights_in) {
  check_rows(rows_in, offsets, row_of, weights_in);
  const Here here(rows_in, offsets, row_of, weights_in);
  const Tensor rows = unit_rows(rows_in);
  const Maybe weights = weights_in ? Maybe(weights_in->contiguous()) : Maybe();
  const int64_t t = row_of.size(0), k = row_of.size(1), h = rows.size(1);
  const Tensor y = fresh({t, h}, rows.scalar_type(), rows);
  check(b200moe_unsort_rows(ptr(rows), row_stride(rows), rows.size(0), ptr<int32_t>(row_of), ptr<float>(weights), t, (int32_t)k, h, row_type(rows.scalar_type()),
                            ptr(y), h, here.stream()),
        "b200moe_unsort_rows");
  return y;
}

// The gradient of the rows reads the weights (none: 1), the gradient of the weights the rows: where `rows` is given, it is asked for.
std::tuple<Maybe, Maybe> unsort_rows_backward(const Tensor& grad_in, const Maybe& rows_in, const Tensor& offsets, const Tensor& row_of, const Maybe& weights_in,
                                              bool want_rows) {
  const int type = row_type(grad_in.scalar_type());
  check_order(offsets, row_of, grad_in.dim() == 2 ? grad_in.size(0) : -1, -1);
  if (grad_in.dim() != 2 || type < 0) refuse("the gradient must be like the output of unsort_tokens");
  if (rows_in) {
    check_rows(*rows_in, offsets, row_of, weights_in);
    if (grad_in.scalar_type() != rows_in->scalar_type() || grad_in.size(1) != rows_in->size(1)) refuse("the gradient must be like the output of unsort_tokens");
  }
  const Here here(grad_in, rows_in, offsets, row_of, weights_in);
  const Tensor grad = unit_rows(grad_in);
  const Maybe rows = rows_in ? Maybe(unit_rows(*rows_in)) : Maybe(), weights = weights_in ? Maybe(weights_in->contiguous()) : Maybe();
  const int64_t t = row_of.size(0), k = row_of.size(1), h = grad.size(1);
  Maybe grad_rows, grad_weights;
  if (want_rows) grad_rows = fresh({t * k, h}, grad.scalar_type(), grad);
  if (rows) grad_weights = fresh({t, k}, at::kFloat, grad);
  check(b200moe_unsort_rows_backward(ptr(grad), row_stride(grad), ptr(rows), row_stride(rows), ptr<int32_t>(row_of), ptr<float>(weights), t, (int32_t)k, h, type,
                                     valid_rows(offsets), ptr(grad_rows), ptr<float>(grad_weights), here.stream()),
        "b200moe_unsort_rows_backward");
  return {grad_rows, grad_weights};
}

// ---- gradients of the token sorting
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool is_default(cudaStream_t stream) { return !stream || stream == cudaStreamLegacy; }
// The capture that a stream takes part in: 0 none (the default stream never does).
unsigned long long capture_of(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  return !is_default(stream) && cudaStreamGetCaptureInfo(stream, &status, &id) == cudaSuccess && status == cudaStreamCaptureStatusActive ? id : 0;
}

// A graph that was built outside a capture and is still alive keeps the gradient node of its leaf on the stream it was built on, and a backward pass
// runs it there. A stream of its own joins the capture through the events that autograd records; the default stream cannot, nor can one that
// another capture has, and the attempt ends the process inside autograd's worker thread. So the call is refused while it can be: where a
// node that t's gradient will reach, its leaves' among them, is on such a stream.
void check_capture(const Tensor& t) {
  if (!t.is_cuda() || !t.requires_grad()) return;
  const unsigned long long capture = capture_of(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
  if (!capture) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> open{t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!open.empty()) {
    const auto node = open.back();
    open.pop_back();
    if (!node || !seen.insert(node.get()).second) continue;
    if (const auto stream = node->stream()) {
      const cudaStream_t handle = c10::cuda::CUDAStream(*stream).stream();
      const unsigned long long other = capture_of(handle);
      if (is_default(handle) || (other && other != capture))
        refuse("a graph of this leaf from outside the capture is still alive: let it go, or capture with x.detach().requires_grad_()");
    }
    for (const auto& edge : node->next_edges()) open.push_back(edge.function);
  }
}

// Gradients that have none themselves, as torch's once_differentiable makes them.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  return torch::autograd::DelayedError("the gradients of sort_tokens and unsort_tokens are not differentiable", (int64_t)grads.size())
      .apply(std::move(grads));
}

void refuse_tangents(bool any) {
  if (any) refuse("sort_tokens and unsort_tokens have no forward-mode derivative");
}

struct SortTokens : torch::autograd::Function<SortTokens> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& offsets, const Tensor& row_of) {
    ctx->save_for_backward({offsets, row_of});
    return sort_rows(x, offsets, row_of);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_tangents(has_tangent(grads[0]));                  // forward mode over this pass: the inputs need not carry any
    const variable_list saved = ctx->get_saved_variables();
    const Tensor grad = grads[0].detach();
    const Tensor dx = grad.dim() == 1 ? unsort_rows(grad.unsqueeze(1), saved[0], saved[1], {}).squeeze(1) : unsort_rows(grad, saved[0], saved[1], {});
    return once({dx, Tensor(), Tensor()});
  }
};

// What is saved is what a gradient that is asked for reads: the rows, the largest tensor here, only where the weights have one.
struct UnsortTokens : torch::autograd::Function<UnsortTokens> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Maybe& weights, const Tensor& offsets, const Tensor& row_of) {
    ctx->save_for_backward({weights && weights->requires_grad() ? rows : Tensor(), weights && rows.requires_grad() ? *weights : Tensor(), offsets, row_of});
    return unsort_rows(rows, offsets, row_of, weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_tangents(has_tangent(grads[0]));
    const variable_list saved = ctx->get_saved_variables();
    const auto given = [](const Tensor& t) { return t.defined() ? Maybe(t.detach()) : Maybe(); };
    const bool want_weights = saved[0].defined() && ctx->needs_input_grad(1);
    auto [grad_rows, grad_weights] = unsort_rows_backward(grads[0].detach(), want_weights ? given(saved[0]) : Maybe(), saved[2], saved[3], given(saved[1]),
                                                          ctx->needs_input_grad(0));
    return once({grad_rows ? *grad_rows : Tensor(), grad_weights ? *grad_weights : Tensor(), Tensor(), Tensor()});
  }
};

Tensor sort_tokens(const Tensor& x, const Tensor& offsets, const Tensor& row_of) {
  refuse_tangents(has_tangent(x));
  if (!at::GradMode::is_enabled() || !x.requires_grad()) return sort_rows(x, offsets, row_of);
  if (row_type(x.scalar_type()) < 0) refuse("sort_tokens has a gradient for bf16, fp16 and fp32 rows");
  check_capture(x);
  return SortTokens::apply(x, offsets, row_of);
}

Tensor unsort_tokens(const Tensor& rows, const Tensor& offsets, const Tensor& row_of, const Maybe& weights) {
  refuse_tangents(has_tangent(rows) || has_tangent(weights));
  if (!at::GradMode::is_enabled() || !(rows.requires_grad() || (weights && weights->requires_grad()))) return unsort_rows(rows, offsets, row_of, weights);
  check_capture(rows);
  if (weights) check_capture(*weights);
  return UnsortTokens::apply(rows, weights, offsets, row_of);
}

}  // namespace

PYBIND11_MODULE(_b200moe_torch, m) {
  m.doc() = "libb200moe's 8-bit operators and token sorting on torch tensors";
  m.def("abi_version", &b200moe_abi_version);
  m.def("rmsnorm_quantize", &rmsnorm_quantize);
  m.def("swiglu_quantize", &swiglu_quantize);
  m.def("mm_8bit", &mm_8bit);
  m.def("route_sort", &route_sort);
  m.def("sort_tokens", &sort_tokens);
  m.def("unsort_tokens", &unsort_tokens);
}
