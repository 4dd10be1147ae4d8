// Layer norm entry points: argument checks, outputs and workspace for
// layer_norm_kernels.hip.

#include <hip/hip_runtime.h>

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>

#include "call_checks.h"

extern "C" {
void sgp_layer_norm_fwd(int dtype, const void* x, int64_t xs,
                        const void* res, int64_t rs, const void* w,
                        const void* b, bool w32, void* y, float* mean,
                        float* rstd, float eps, int64_t M, int C, bool relu,
                        hipStream_t s);
int sgp_layer_norm_partials(int dtype, int64_t M, int C);
void sgp_layer_norm_bwd(int dtype, const void* dy, int64_t ds, const void* x,
                        int64_t xs, const void* y, const void* w, bool w32,
                        const float* mean, const float* rstd, void* dx,
                        void* dres, float* partials, int P, void* dw,
                        void* db, bool g32, int64_t M, int C, hipStream_t s);
}

namespace {

using torch::autograd::variable_list;
typedef torch::optional<torch::Tensor> OptTensor;

int dtype_code(const torch::Tensor& x) {
  switch (x.scalar_type()) {
    case torch::kFloat32: return 0;
    case torch::kBFloat16: return 1;
    case torch::kFloat16: return 2;
    default:
      TORCH_CHECK(false, "layer_norm: x must be fp32, bf16 or fp16, got ",
                  x.scalar_type());
  }
}

// a [M, C] matrix whose rows are contiguous; their distance is free
void check_rows(const torch::Tensor& t, const char* name,
                const torch::Tensor& x) {
  TORCH_CHECK(t.is_cuda(), "layer_norm: ", name, " must be a device tensor");
  TORCH_CHECK(t.device() == x.device(), "layer_norm: ", name,
              " is on another device than x");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), "layer_norm: ", name,
              " must have x's dtype");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == x.size(0)
              && t.size(1) == x.size(1),
              "layer_norm: ", name, " must have x's shape");
  TORCH_CHECK(t.numel() == 0 || t.size(1) == 1 || t.stride(1) == 1,
              "layer_norm: ", name,
              " must have contiguous rows");
  check_memory("layer_norm", t);
}

void check_vector(const torch::Tensor& t, const char* name,
                  const torch::Tensor& x) {
  TORCH_CHECK(t.is_cuda() && t.device() == x.device(), "layer_norm: ", name,
              " must be on x's device");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == x.size(1) && t.is_contiguous(),
              "layer_norm: ", name, " must be a contiguous [", x.size(1),
              "] vector");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32
              || t.scalar_type() == x.scalar_type(),
              "layer_norm: ", name, " must be fp32 or have x's dtype");
  check_memory("layer_norm", t);
}

const void* ptr(const OptTensor& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

bool is_fp32(const OptTensor& w, const OptTensor& b) {
  if (w.has_value() && b.has_value())
    TORCH_CHECK(w->scalar_type() == b->scalar_type(),
                "layer_norm: weight and bias must have one dtype");
  return (w.has_value() && w->scalar_type() == torch::kFloat32)
         || (b.has_value() && b->scalar_type() == torch::kFloat32);
}

void check_size(const torch::Tensor& x) {
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= (int64_t(1) << 30),
              "layer_norm: the last dimension must be 1 to 2^30 long");
}

// x: [M, C] -> (y, mean [M], rstd [M]); the statistics only if asked for.  y
// is made with the sizes that the caller shows: a view of it, made where
// autograd does not look, could not be changed in place.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> forward_rows(
    const torch::Tensor& x, const OptTensor& weight, const OptTensor& bias,
    const OptTensor& res, double eps, bool relu, bool statistics,
    at::IntArrayRef sizes) {
  check_rows(x, "x", x);
  const int dtype = dtype_code(x);
  check_size(x);
  if (weight.has_value()) check_vector(*weight, "weight", x);
  if (bias.has_value()) check_vector(*bias, "bias", x);
  if (res.has_value()) check_rows(*res, "residual", x);
  const bool w32 = is_fp32(weight, bias);
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0);
  torch::Tensor y = torch::empty(sizes, x.options());
  check_memory("layer_norm", y);  // under a mode that makes such tensors
  torch::Tensor mean, rstd;
  if (statistics) {
    mean = torch::empty({M}, x.options().dtype(torch::kFloat32));
    rstd = torch::empty_like(mean);
  }
  if (M > 0) {
    sgp_layer_norm_fwd(
        dtype, x.data_ptr(), x.stride(0), ptr(res),
        res.has_value() ? res->stride(0) : 0, ptr(weight), ptr(bias), w32,
        y.data_ptr(), statistics ? mean.data_ptr<float>() : nullptr,
        statistics ? rstd.data_ptr<float>() : nullptr, (float)eps, M,
        (int)x.size(1), relu,
        c10::hip::getCurrentHIPStream(x.device().index()).stream());
    C10_HIP_CHECK(hipGetLastError());
  }
  return {y, mean, rstd};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> layer_norm_fwd(
    const torch::Tensor& x, const OptTensor& weight, const OptTensor& bias,
    const OptTensor& res, double eps, bool relu, bool statistics) {
  return forward_rows(x, weight, bias, res, eps, relu, statistics, x.sizes());
}

// -> (dx, dres, dw, db), each only if asked for.  `y`: the output, if there
// was a ReLU.  dw and db have `weight`'s dtype, or `vector_dtype` without.
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor>
layer_norm_bwd(const torch::Tensor& dy, const torch::Tensor& x,
               const OptTensor& y, const OptTensor& weight,
               const torch::Tensor& mean, const torch::Tensor& rstd,
               bool vectors_fp32, bool need_dx, bool need_dres, bool need_dw,
               bool need_db) {
  check_rows(x, "x", x);
  const int dtype = dtype_code(x);
  check_size(x);
  check_rows(dy, "dy", x);
  if (y.has_value()) {
    check_rows(*y, "y", x);
    TORCH_CHECK(y->is_contiguous(), "layer_norm: y must be contiguous");
  }
  if (weight.has_value()) check_vector(*weight, "weight", x);
  const int64_t M = x.size(0), C = x.size(1);
  for (const torch::Tensor& t : {mean, rstd}) {
    TORCH_CHECK(t.is_cuda() && t.device() == x.device() && t.is_contiguous()
                && t.scalar_type() == torch::kFloat32 && t.numel() == M,
                "layer_norm: the statistics must be fp32 [M] on x's device");
    check_memory("layer_norm", t);
  }
  const c10::DeviceGuard guard(x.device());
  const bool g32 = vectors_fp32 || dtype == 0;
  const auto vec = g32 ? x.options().dtype(torch::kFloat32) : x.options();
  torch::Tensor dx, dres, dw, db, partials;
  if (need_dx) dx = torch::empty({M, C}, x.options());
  if (need_dres) dres = torch::empty({M, C}, x.options());
  if (M == 0) {
    if (need_dw) dw = torch::zeros({C}, vec);
    if (need_db) db = torch::zeros({C}, vec);
    return {dx, dres, dw, db};
  }
  if (need_dw) dw = torch::empty({C}, vec);
  if (need_db) db = torch::empty({C}, vec);
  // the grid, and with it the rows of partial sums: asked for once
  const int P = sgp_layer_norm_partials(dtype, M, (int)C);
  if (need_dw || need_db)
    partials = torch::empty({(int64_t)P * 2 * C},
                            x.options().dtype(torch::kFloat32));
  for (const torch::Tensor& t : {dx, dres, dw, db, partials})
    if (t.defined()) check_memory("layer_norm", t);
  sgp_layer_norm_bwd(
      dtype, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), ptr(y),
      ptr(weight),
      weight.has_value() && weight->scalar_type() == torch::kFloat32,
      mean.data_ptr<float>(), rstd.data_ptr<float>(),
      need_dx ? dx.data_ptr() : nullptr,
      need_dres ? dres.data_ptr() : nullptr,
      partials.defined() ? partials.data_ptr<float>() : nullptr, P,
      need_dw ? dw.data_ptr() : nullptr, need_db ? db.data_ptr() : nullptr,
      g32, M, (int)C,
      c10::hip::getCurrentHIPStream(x.device().index()).stream());
  C10_HIP_CHECK(hipGetLastError());
  return {dx, dres, dw, db};
}

// ------------------------------------------------------------- autograd
// In C++: the way through the Python layer costs more than the kernels do on
// ordinary activations.

// t as a matrix of its last dimension's rows: a view where they are
// contiguous and evenly spaced, a copy elsewhere
torch::Tensor rows(const torch::Tensor& t) {
  torch::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

OptTensor rows(const OptTensor& t) {
  return t.has_value() ? OptTensor(rows(*t)) : t;
}

class LayerNorm : public torch::autograd::Function<LayerNorm> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx,
                               const torch::Tensor& x,
                               const OptTensor& weight, const OptTensor& bias,
                               const OptTensor& res, double eps, bool relu) {
    auto [y, mean, rstd] = forward_rows(rows(x), weight, bias, rows(res),
                                        eps, relu, true, x.sizes());
    ctx->save_for_backward({x, weight.value_or(torch::Tensor()), mean, rstd,
                            relu ? y : torch::Tensor()});
    const OptTensor& vector = weight.has_value() ? weight : bias;
    int64_t flags = relu ? 1 : 0;
    if (vector.has_value() && vector->scalar_type() == torch::kFloat32)
      flags |= 2;
    if (weight.has_value()) flags |= 4;
    if (bias.has_value()) flags |= 8;
    if (res.has_value()) flags |= 16;
    ctx->saved_data["flags"] = flags;
    return y;
  }

  static variable_list backward(torch::autograd::AutogradContext* ctx,
                                variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const torch::Tensor &x = saved[0], &weight = saved[1], &mean = saved[2],
                        &rstd = saved[3], &y = saved[4];
    const torch::Tensor& dy = grads[0];
    check_untraced("layer_norm");
    check_tangent("layer_norm", dy);
    const int64_t flags = ctx->saved_data["flags"].toInt();
    // numbered over the tensors that there are
    size_t edge = 0;
    auto needs = [&](bool given) {
      return given && ctx->needs_input_grad(edge++);
    };
    const bool need_dx = needs(true), need_dw = needs(flags & 4),
               need_db = needs(flags & 8), need_dres = needs(flags & 16);
    // without a ReLU the residual's gradient is dy itself
    const bool masked = need_dres && (flags & 1);
    torch::Tensor dx, dw, db, dres;
    if (need_dx || need_dw || need_db || masked) {
      const at::AutoGradMode no_grad(false);
      std::tie(dx, dres, dw, db) = layer_norm_bwd(
          rows(dy), rows(x), y.defined() ? OptTensor(rows(y)) : OptTensor(),
          weight.defined() ? OptTensor(weight) : OptTensor(), mean, rstd,
          flags & 2, need_dx, masked, need_dw, need_db);
      if (need_dx) dx = dx.view(x.sizes());
      if (masked) dres = dres.view(x.sizes());
    }
    if (need_dres && !masked) dres = dy;
    variable_list out = {dx, dw, db, dres, torch::Tensor(), torch::Tensor()};
    if (!torch::GradMode::is_enabled()) return out;
    // create_graph: these have no graph of their own, and say so when asked
    variable_list given;
    for (const torch::Tensor& t : out)
      if (t.defined()) given.push_back(t.detach().requires_grad_(true));
    if (given.empty()) return out;
    const auto error = std::make_shared<torch::autograd::DelayedError>(
        "layer_norm is differentiable once", (int64_t)given.size());
    given = (*error)(std::move(given));
    size_t k = 0;
    for (torch::Tensor& t : out)
      if (t.defined()) t = given[k++];
    return out;
  }
};

torch::Tensor layer_norm(const torch::Tensor& x, const OptTensor& weight,
                         const OptTensor& bias, double eps,
                         const OptTensor& res, bool relu) {
  check_untraced("layer_norm");
  check_tangent("layer_norm", x);
  for (const OptTensor* t : {&weight, &bias, &res})
    if (t->has_value()) check_tangent("layer_norm", **t);
  auto wants = [](const OptTensor& t) {
    return t.has_value() && t->requires_grad();
  };
  if (torch::GradMode::is_enabled()
      && (x.requires_grad() || wants(weight) || wants(bias) || wants(res)))
    return LayerNorm::apply(x, weight, bias, res, eps, relu);
  return std::get<0>(forward_rows(rows(x), weight, bias, rows(res), eps,
                                  relu, false, x.sizes()));
}

}  // namespace

void init_layer_norm(py::module_& m) {
  m.def("layer_norm", &layer_norm,
        "layer norm over the last dimension, differentiable");
  m.def("layer_norm_fwd", &layer_norm_fwd,
        "row-wise layer norm (+residual)(+ReLU) -> (y, mean, rstd)");
  m.def("layer_norm_bwd", &layer_norm_bwd,
        "layer norm gradients -> (dx, dres, dw, db)");
}
