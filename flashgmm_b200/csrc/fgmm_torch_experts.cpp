// pybind11 bindings of the expert operators over the C ABI (include/flashgmm_b200.h), part of the
// module of fgmm_torch.cpp: CUDA tensors only, every argument's dtype, shape and device checked,
// launches on the current stream of the tensors' device, scratch from torch's caching allocator.
// Rows that are not contiguous are copied; a score matrix is read through its row stride.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include "../../include/flashgmm_b200.h"

namespace {

using torch::Tensor;

void check_rc(int rc, const char *op) {
  TORCH_CHECK(rc == FGMM_OK, op, ": flashgmm_b200 error ", rc, ": ", fgmm_last_error());
}

// Only tensors that own their memory and whose derivatives autograd records are read through their pointers: a forward-mode tangent
// would be dropped, and the pointer of a traced, batched or wrapped tensor is none (that of a traced tensor's slice is not null).
void check_plain(const Tensor &t, const char *name) {
  constexpr c10::DispatchKeySet kOthers({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                         c10::DispatchKey::Functionalize, c10::DispatchKey::ZeroTensor});
  TORCH_CHECK(t.defined() && t.layout() == torch::kStrided && !t.key_set().has_any(kOthers), name,
              " must be a plain strided tensor (not a traced, batched, sparse or wrapped one)");
  TORCH_CHECK(!t._fw_grad(0).defined(), name, " has a forward-mode tangent: flashgmm_b200 has no forward-mode derivatives");
}

void check_cuda(const Tensor &t, const char *name, int dim, const torch::Device *dev) {
  check_plain(t, name);
  TORCH_CHECK(t.dim() == dim, name, " must be ", dim, "D");
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (flashgmm_b200 has no CPU path)");
  if (dev) TORCH_CHECK(t.device() == *dev, name, " is on ", t.device(), ", expected ", *dev);
}

int dtype_of(const Tensor &t, const char *name) {
  if (t.scalar_type() == torch::kFloat32) return FGMM_F32;
  if (t.scalar_type() == torch::kBFloat16) return FGMM_BF16;
  TORCH_CHECK(t.scalar_type() == torch::kFloat16, name, " must be float32, bfloat16 or float16");
  return FGMM_F16;
}

void check_type(const Tensor &t, const char *name, torch::ScalarType type) {
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type);
}

void check_shape(const Tensor &t, const char *name, std::initializer_list<int64_t> want) {
  TORCH_CHECK(t.sizes() == torch::IntArrayRef(want), "shape mismatch: ", name, t.sizes(), ", expected ",
              torch::IntArrayRef(want));
}

// Contiguous, with the values in memory (a view may hold them negated).
Tensor dense(const Tensor &t) { return t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }

// Rows contiguous; the row stride stays (an expanded or sliced matrix is not copied).
Tensor with_rows(const Tensor &t) {
  return !t.is_neg() && (t.size(1) <= 1 || t.stride(1) == 1) ? t : dense(t);
}
int64_t row_stride(const Tensor &t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// Contiguous and on a 16-byte boundary, as the products read their matrices.
Tensor for_products(const Tensor &t) {
  Tensor c = dense(t);
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}

// A result or scratch of torch's caching allocator, past the dispatcher (a microsecond of a small call).
Tensor fresh(torch::IntArrayRef sizes, torch::ScalarType type, const torch::Device &dev) {
  return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

Tensor scratch(size_t bytes, const torch::Device &dev) {
  return fresh({(int64_t)std::max<size_t>(bytes, 256)}, torch::kUInt8, dev);
}

void *stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int narrow(int64_t v, const char *name) {
  TORCH_CHECK(v >= INT32_MIN && v <= INT32_MAX, name, " is out of range: ", v);
  return (int)v;
}

int score_func(const std::string &name) {
  if (name == "softmax") return FGMM_SCORE_SOFTMAX;
  if (name == "sigmoid") return FGMM_SCORE_SIGMOID;
  TORCH_CHECK(name == "given", "score_func must be 'softmax', 'sigmoid' or 'given', got '", name, "'");
  return FGMM_SCORE_GIVEN;
}

std::tuple<Tensor, Tensor> route_experts(const Tensor &scores, int64_t top_k, const std::string &func,
                                         const c10::optional<Tensor> &bias, int64_t n_groups,
                                         const c10::optional<int64_t> &top_groups, bool renormalize, double scale) {
  const int dtype = dtype_of(scores, "scores"), f = score_func(func);
  check_cuda(scores, "scores", 2, nullptr);
  const torch::Device dev = scores.device();
  const int64_t N = scores.size(0), K = scores.size(1);
  Tensor b;
  if (bias) {
    check_type(*bias, "bias", torch::kFloat32);
    check_cuda(*bias, "bias", 1, &dev);
    check_shape(*bias, "bias", {K});
    b = dense(*bias);
  }
  TORCH_CHECK(top_k >= 1 && top_k <= K && top_k <= FGMM_MAX_TOP_K, "top_k must be in [1, min(K, ", FGMM_MAX_TOP_K, ")], got ", top_k);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor z = with_rows(scores);
  Tensor w = fresh({N, top_k}, torch::kFloat32, dev);
  Tensor idx = fresh({N, top_k}, torch::kInt32, dev);
  check_rc(fgmm_route_experts(z.data_ptr(), dtype, N, narrow(K, "K"), row_stride(z), bias ? b.data_ptr<float>() : nullptr,
                              (int)top_k, f, narrow(n_groups, "n_groups"), narrow(top_groups.value_or(n_groups), "top_groups"),
                              renormalize, (float)scale, w.data_ptr<float>(), idx.data_ptr<int32_t>(), stream()),
           "route_experts");
  return {w, idx};
}

Tensor route_experts_backward(const Tensor &d_weights, const Tensor &scores, const Tensor &indices,
                              const std::string &func, bool renormalize, double scale) {
  const int dtype = dtype_of(scores, "scores"), f = score_func(func);
  check_cuda(scores, "scores", 2, nullptr);
  const torch::Device dev = scores.device();
  const int64_t N = scores.size(0), K = scores.size(1);
  check_type(d_weights, "d_weights", torch::kFloat32);
  check_cuda(d_weights, "d_weights", 2, &dev);
  check_type(indices, "indices", torch::kInt32);
  check_cuda(indices, "indices", 2, &dev);
  const int64_t top_k = indices.size(1);
  check_shape(indices, "indices", {N, top_k});
  check_shape(d_weights, "d_weights", {N, top_k});
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor z = with_rows(scores), dw = dense(d_weights), idx = dense(indices);
  Tensor dz = fresh({N, K}, z.scalar_type(), dev);
  check_rc(fgmm_route_experts_backward(dw.data_ptr<float>(), z.data_ptr(), dtype, N, narrow(K, "K"), row_stride(z),
                                       idx.data_ptr<int32_t>(), narrow(top_k, "top_k"), f, renormalize, (float)scale,
                                       dz.data_ptr(), stream()),
           "route_experts_backward");
  return dz;
}

std::tuple<Tensor, Tensor, Tensor> group_routes(const Tensor &indices, int64_t K) {
  check_type(indices, "indices", torch::kInt32);
  check_cuda(indices, "indices", 2, nullptr);
  TORCH_CHECK(indices.size(1) >= 1, "indices must have at least one column");
  TORCH_CHECK(K >= 1 && K <= FGMM_MAX_EXPERTS, "K must be in [1, ", FGMM_MAX_EXPERTS, "], got ", K);
  const int64_t R = indices.numel();
  TORCH_CHECK(R <= INT32_MAX - 1024, "indices has more than 2^31 - 1025 routes");
  const torch::Device dev = indices.device();
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor idx = dense(indices);
  Tensor order = fresh({R}, torch::kInt32, dev), offsets = fresh({K + 1}, torch::kInt32, dev);
  Tensor position = fresh(indices.sizes(), torch::kInt32, dev);
  Tensor ws = scratch(fgmm_group_routes_workspace_bytes(R, (int)K), dev);
  check_rc(fgmm_group_routes(idx.data_ptr<int32_t>(), R, (int)K, order.data_ptr<int32_t>(), offsets.data_ptr<int32_t>(),
                             position.data_ptr<int32_t>(), ws.data_ptr(), ws.numel(), stream()),
           "group_routes");
  return {order, offsets, position};
}

// The plan of group_routes as its users check it.
struct Plan {
  Tensor order, offsets, position;
  int64_t R, N;
  int K, top_k;
};

Plan plan_of(const Tensor &order, const Tensor &offsets, const Tensor &position, const torch::Device &dev) {
  check_type(order, "order", torch::kInt32);
  check_cuda(order, "order", 1, &dev);
  check_type(offsets, "offsets", torch::kInt32);
  check_cuda(offsets, "offsets", 1, &dev);
  check_type(position, "position", torch::kInt32);
  check_cuda(position, "position", 2, &dev);
  TORCH_CHECK(position.size(1) >= 1, "position must have at least one column");
  check_shape(order, "order", {position.numel()});
  TORCH_CHECK(offsets.size(0) >= 2 && offsets.size(0) <= FGMM_MAX_EXPERTS + 1, "offsets must have K + 1 entries, K in [1, ",
              FGMM_MAX_EXPERTS, "]");
  TORCH_CHECK(order.numel() <= INT32_MAX - 1024, "the plan has more than 2^31 - 1025 routes");
  return {dense(order), dense(offsets), dense(position), order.size(0), position.size(0),
          (int)offsets.size(0) - 1, (int)position.size(1)};
}

Tensor expert_products(const Tensor &x, const Tensor &weight, const Tensor &order, const Tensor &offsets, const Tensor &position) {
  const int dtype = dtype_of(x, "x");
  check_cuda(x, "x", 2, nullptr);
  const torch::Device dev = x.device();
  check_type(weight, "weight", x.scalar_type());
  check_cuda(weight, "weight", 3, &dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Plan p = plan_of(order, offsets, position, dev);
  const int64_t d_in = x.size(1), d_out = weight.size(1);
  check_shape(x, "x", {p.N, d_in});
  check_shape(weight, "weight", {p.K, d_out, d_in});
  TORCH_CHECK(d_in >= 1 && d_out >= 1, "x and weight must have at least one column");
  const Tensor xc = for_products(x), wc = for_products(weight);
  Tensor y = fresh({p.R, d_out}, x.scalar_type(), dev);
  const int di = narrow(d_in, "d_in"), dn = narrow(d_out, "d_out");
  const size_t nb = fgmm_expert_products_workspace_bytes(dtype, p.N, p.K, di, dn, p.top_k);
  TORCH_CHECK(nb > 0, "expert_products: ", fgmm_last_error());
  Tensor ws = scratch(nb, dev);
  check_rc(fgmm_expert_products(xc.data_ptr(), dtype, p.N, di, wc.data_ptr(), p.K, dn, p.order.data_ptr<int32_t>(),
                                p.offsets.data_ptr<int32_t>(), p.top_k, y.data_ptr(), ws.data_ptr(), ws.numel(), stream()),
           "expert_products");
  return y;
}

std::tuple<c10::optional<Tensor>, c10::optional<Tensor>> expert_products_backward(
    const Tensor &dy, const Tensor &x, const Tensor &weight, const Tensor &order, const Tensor &offsets,
    const Tensor &position, bool need_dx, bool need_dweight) {
  const int dtype = dtype_of(x, "x");
  check_cuda(x, "x", 2, nullptr);
  const torch::Device dev = x.device();
  check_type(weight, "weight", x.scalar_type());
  check_cuda(weight, "weight", 3, &dev);
  check_type(dy, "dy", x.scalar_type());
  check_cuda(dy, "dy", 2, &dev);
  const c10::cuda::CUDAGuard guard(dev);
  const Plan p = plan_of(order, offsets, position, dev);
  const int64_t d_in = x.size(1), d_out = weight.size(1);
  check_shape(x, "x", {p.N, d_in});
  check_shape(weight, "weight", {p.K, d_out, d_in});
  check_shape(dy, "dy", {p.R, d_out});
  TORCH_CHECK(d_in >= 1 && d_out >= 1, "x and weight must have at least one column");
  const Tensor xc = for_products(x), wc = for_products(weight), gc = for_products(dy);
  c10::optional<Tensor> dx, dw;
  if (need_dx) dx = fresh({p.N, d_in}, x.scalar_type(), dev);
  if (need_dweight) dw = fresh({p.K, d_out, d_in}, x.scalar_type(), dev);
  if (!need_dx && !need_dweight) return {dx, dw};
  const int di = narrow(d_in, "d_in"), dn = narrow(d_out, "d_out");
  const size_t nb = fgmm_expert_products_backward_workspace_bytes(dtype, p.N, p.K, di, dn, p.top_k);
  TORCH_CHECK(nb > 0, "expert_products_backward: ", fgmm_last_error());
  Tensor ws = scratch(nb, dev);
  check_rc(fgmm_expert_products_backward(gc.data_ptr(), xc.data_ptr(), dtype, p.N, di, wc.data_ptr(), p.K, dn,
                                         p.order.data_ptr<int32_t>(), p.offsets.data_ptr<int32_t>(),
                                         p.position.data_ptr<int32_t>(), p.top_k, dx ? dx->data_ptr() : nullptr,
                                         dw ? dw->data_ptr() : nullptr, ws.data_ptr(), ws.numel(), stream()),
           "expert_products_backward");
  return {dx, dw};
}

Tensor combine_experts(const Tensor &y, const Tensor &weights, const Tensor &order, const Tensor &offsets, const Tensor &position) {
  const int dtype = dtype_of(y, "y");
  check_cuda(y, "y", 2, nullptr);
  const torch::Device dev = y.device();
  const c10::cuda::CUDAGuard guard(dev);
  const Plan p = plan_of(order, offsets, position, dev);
  const int64_t d = y.size(1);
  check_shape(y, "y", {p.R, d});
  check_type(weights, "weights", torch::kFloat32);
  check_cuda(weights, "weights", 2, &dev);
  check_shape(weights, "weights", {p.N, p.top_k});
  TORCH_CHECK(d >= 1, "y must have at least one column");
  const Tensor yc = dense(y), w = dense(weights);
  Tensor out = fresh({p.N, d}, y.scalar_type(), dev);
  check_rc(fgmm_combine_experts(yc.data_ptr(), dtype, p.N, narrow(d, "d"), w.data_ptr<float>(), p.position.data_ptr<int32_t>(),
                                p.top_k, out.data_ptr(), stream()),
           "combine_experts");
  return out;
}

std::tuple<Tensor, Tensor> combine_experts_backward(const Tensor &d_out, const Tensor &y, const Tensor &weights,
                                                    const Tensor &order, const Tensor &offsets, const Tensor &position) {
  const int dtype = dtype_of(y, "y");
  check_cuda(y, "y", 2, nullptr);
  const torch::Device dev = y.device();
  const c10::cuda::CUDAGuard guard(dev);
  const Plan p = plan_of(order, offsets, position, dev);
  const int64_t d = y.size(1);
  check_shape(y, "y", {p.R, d});
  check_type(weights, "weights", torch::kFloat32);
  check_cuda(weights, "weights", 2, &dev);
  check_shape(weights, "weights", {p.N, p.top_k});
  check_type(d_out, "d_out", y.scalar_type());
  check_cuda(d_out, "d_out", 2, &dev);
  check_shape(d_out, "d_out", {p.N, d});
  TORCH_CHECK(d >= 1, "y must have at least one column");
  const Tensor yc = dense(y), gc = dense(d_out), w = dense(weights);
  Tensor dy = fresh({p.R, d}, y.scalar_type(), dev), dw = fresh({p.N, p.top_k}, torch::kFloat32, dev);
  check_rc(fgmm_combine_experts_backward_placed(gc.data_ptr(), yc.data_ptr(), dtype, p.N, narrow(d, "d"), w.data_ptr<float>(),
                                                p.order.data_ptr<int32_t>(), p.offsets.data_ptr<int32_t>(),
                                                p.position.data_ptr<int32_t>(), p.K, p.top_k, dy.data_ptr(),
                                                dw.data_ptr<float>(), stream()),
           "combine_experts_backward");
  return {dy, dw};
}

}  // namespace

void bind_experts(pybind11::module_ &m) {
  namespace py = pybind11;
  m.def("route_experts", &route_experts, py::arg("scores"), py::arg("top_k"), py::arg("score_func"), py::arg("bias"),
        py::arg("n_groups"), py::arg("top_groups"), py::arg("renormalize"), py::arg("scale"));
  m.def("route_experts_backward", &route_experts_backward, py::arg("d_weights"), py::arg("scores"), py::arg("indices"),
        py::arg("score_func"), py::arg("renormalize"), py::arg("scale"));
  m.def("group_routes", &group_routes, py::arg("indices"), py::arg("K"));
  m.def("expert_products", &expert_products, py::arg("x"), py::arg("weight"), py::arg("order"), py::arg("offsets"),
        py::arg("position"));
  m.def("expert_products_backward", &expert_products_backward, py::arg("dy"), py::arg("x"), py::arg("weight"),
        py::arg("order"), py::arg("offsets"), py::arg("position"), py::arg("need_dx"), py::arg("need_dweight"));
  m.def("combine_experts", &combine_experts, py::arg("y"), py::arg("weights"), py::arg("order"), py::arg("offsets"),
        py::arg("position"));
  m.def("combine_experts_backward", &combine_experts_backward, py::arg("d_out"), py::arg("y"), py::arg("weights"),
        py::arg("order"), py::arg("offsets"), py::arg("position"));
}
