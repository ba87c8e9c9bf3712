// extern "C" entry points of the expert operators: checks of arguments, workspaces, launches.
#include <cmath>

#include "fgmm_experts.cuh"

namespace fgmm {
namespace {

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int check_experts(int dtype, int64_t N, int K, int top_k) {
  if (dtype != FGMM_F32 && dtype != FGMM_BF16 && dtype != FGMM_F16)
    return fail(FGMM_ERR_INVALID, "dtype must be FGMM_F32, FGMM_BF16 or FGMM_F16");
  if (N < 0 || K < 1 || top_k < 1)
    return fail(FGMM_ERR_INVALID, "N must be >= 0, K and top_k >= 1 (got N=" + std::to_string(N) + " K=" + std::to_string(K) +
                                      " top_k=" + std::to_string(top_k) + ")");
  if (K > FGMM_MAX_EXPERTS) return fail(FGMM_ERR_UNSUPPORTED, "K > " + std::to_string(FGMM_MAX_EXPERTS) + " is not supported");
  // (row numbers a tile behind the last one stay in 32 bits)
  if (N > (INT32_MAX - 1024) / top_k) return fail(FGMM_ERR_UNSUPPORTED, "N top_k must be at most 2^31 - 1025");
  return FGMM_OK;
}

int check_widths(int d_in, int d_out) {
  if (d_in < 1 || d_out < 1) return fail(FGMM_ERR_INVALID, "d_in and d_out must be >= 1");
  if (d_in > (1 << 20) || d_out > (1 << 20)) return fail(FGMM_ERR_UNSUPPORTED, "d_in and d_out must be <= 2^20");
  return FGMM_OK;
}

// Which products run on the tensor cores.  The CUDA-core products read float32 weights, and 16-bit ones with rows of no multiple of
// 16 bytes, as they are, and write the gradients of experts without a row straight.
// Rows an expert, on average, up to which they are faster; us at 64 experts of 512 x 1,024, CUDA cores / tensor cores:
//   rows          0.25      1         2          4          8           16
//   y  float32    9 / 77    16 / 89   28 / 90    43 / 102   66 / 104    103 / 115
//   dx float32    19 / 89   28 / 89   49 / 91    82 / 113   128 / 114
//   dW float32    25 / 51   29 / 53   35 / 54    44 / 60    66 / 62
//   dW bf16       15 / 26   19 / 27   27 / 27    28 / 27
// and at 16 rows of 509 x 1,024 bf16: y 154 / 55, dx 196 / 54, dW 112 / 101.
// The host knows the mean only.  dW gives an expert's rows to one column of blocks there, one row after the other, and a popular
// expert is slow; us with the rows spread evenly / half of them on one expert / all on one:
//   24,576 rows, 4,096 experts of 64 x 64 float32   55 / 6,010 / 11,560
//   384 rows, 64 experts of 512 x 1,024 float32     63 / 402 / 846
//   4,096 rows, 4,096 experts of 64 x 64 bf16       27 / 820 / 1,640
// y and dx give windows of rows to the blocks and gain by it (108 / 92 / 79 and 91 / 64 / 50 at the first).
TcParts on_tensor_cores(int dtype, int64_t R, int K, int d_in, int d_out) {
  const bool f32 = dtype == FGMM_F32, in_copied = f32 || d_in % 8 != 0, out_copied = in_copied || d_out % 8 != 0;
  const auto few = [&](int rows) { return R <= (int64_t)rows * K; };
  return {!(in_copied && few(f32 ? 16 : 4)), !(out_copied && few(f32 ? 6 : 4)), !few(out_copied ? 6 : 1)};
}

// dx_rows: one matrix, or the parts of the CUDA-core product.
size_t dx_rows_bytes(const TcParts &tc, int64_t R, int K, int d_in, int d_out) {
  return align_up((size_t)R * d_in * sizeof(float) * (tc.inputs ? 1 : few_dx_parts(R, K, d_in, d_out)), 256);
}

int check_route(int dtype, int64_t N, int K, int64_t row_stride, int top_k, int func) {
  int rc = check_experts(dtype, N, K, top_k);
  if (rc) return rc;
  if (top_k > K || top_k > FGMM_MAX_TOP_K)
    return fail(FGMM_ERR_INVALID, "top_k must be <= K and <= " + std::to_string(FGMM_MAX_TOP_K));
  if (func != FGMM_SCORE_SOFTMAX && func != FGMM_SCORE_SIGMOID && func != FGMM_SCORE_GIVEN)
    return fail(FGMM_ERR_INVALID, "unknown score function");
  if (row_stride < 0) return fail(FGMM_ERR_INVALID, "row_stride must be >= 0");
  return FGMM_OK;
}

}  // namespace
}  // namespace fgmm

using namespace fgmm;

extern "C" {

int fgmm_route_experts(const void *scores, int32_t dtype, int64_t N, int32_t K, int64_t row_stride,
                       const float *bias, int32_t top_k, int32_t score_func, int32_t n_groups,
                       int32_t top_groups, int32_t renormalize, float scale, float *weights,
                       int32_t *indices, void *stream) {
  int rc = check_route(dtype, N, K, row_stride, top_k, score_func);
  if (rc) return rc;
  if (n_groups < 1 || n_groups > FGMM_MAX_SCORE_GROUPS || K % n_groups != 0)
    return fail(FGMM_ERR_INVALID, "n_groups must divide K and be in [1, " + std::to_string(FGMM_MAX_SCORE_GROUPS) + "]");
  if (top_groups < 1 || top_groups > n_groups) return fail(FGMM_ERR_INVALID, "top_groups must be in [1, n_groups]");
  if (N == 0) return FGMM_OK;
  if (!scores || !weights || !indices) return fail(FGMM_ERR_INVALID, "null pointer argument");
  if (!aligned(scores, elem_size(dtype))) return fail(FGMM_ERR_INVALID, "scores must be aligned to their elements");
  // one group, or all of them kept, is no restriction
  if (top_groups == n_groups) n_groups = top_groups = 1;
  return route_forward(scores, dtype, N, K, row_stride, bias, top_k, score_func, n_groups, top_groups,
                       renormalize != 0, scale, weights, indices, (cudaStream_t)stream);
}

int fgmm_route_experts_backward(const float *d_weights, const void *scores, int32_t dtype, int64_t N,
                                int32_t K, int64_t row_stride, const int32_t *indices, int32_t top_k,
                                int32_t score_func, int32_t renormalize, float scale, void *d_scores,
                                void *stream) {
  int rc = check_route(dtype, N, K, row_stride, top_k, score_func);
  if (rc) return rc;
  if (N == 0) return FGMM_OK;
  if (!d_weights || !scores || !indices || !d_scores) return fail(FGMM_ERR_INVALID, "null pointer argument");
  if (!aligned(scores, elem_size(dtype)) || !aligned(d_scores, elem_size(dtype)))
    return fail(FGMM_ERR_INVALID, "scores and d_scores must be aligned to their elements");
  return route_backward(d_weights, scores, dtype, N, K, row_stride, indices, top_k, score_func,
                        renormalize != 0, scale, d_scores, (cudaStream_t)stream);
}

size_t fgmm_group_routes_workspace_bytes(int64_t R, int32_t K) {
  if (R < 0 || R > INT32_MAX - 1024 || K < 1 || K > FGMM_MAX_EXPERTS) return 0;
  return group_workspace_bytes(R, K);
}

int fgmm_group_routes(const int32_t *indices, int64_t R, int32_t K, int32_t *order, int32_t *offsets,
                      int32_t *position, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = check_experts(FGMM_F32, R, K, 1);
  if (rc) return rc;
  if (!offsets) return fail(FGMM_ERR_INVALID, "null pointer argument");
  if (R == 0) {
    FGMM_CUDA_TRY(cudaMemsetAsync(offsets, 0, (size_t)(K + 1) * sizeof(int32_t), (cudaStream_t)stream));
    return FGMM_OK;
  }
  if (!indices || !order || !position || !workspace) return fail(FGMM_ERR_INVALID, "null pointer argument");
  if (!aligned(workspace, 256)) return fail(FGMM_ERR_INVALID, "workspace must be 256-byte aligned");
  if (workspace_bytes < group_workspace_bytes(R, K)) return fail(FGMM_ERR_WORKSPACE, "workspace too small");
  return group_routes(indices, R, K, order, offsets, position, workspace, (cudaStream_t)stream);
}

size_t fgmm_expert_products_workspace_bytes(int32_t dtype, int64_t N, int32_t K, int32_t d_in,
                                            int32_t d_out, int32_t top_k) {
  if (check_experts(dtype, N, K, top_k) || check_widths(d_in, d_out)) return 0;
  const TcParts tc = on_tensor_cores(dtype, N * top_k, K, d_in, d_out);
  return tc.forward ? products_tc_workspace(dtype, N, K, d_in, d_out, top_k, {true, false, false}) : 256;
}

int fgmm_expert_products(const void *x, int32_t dtype, int64_t N, int32_t d_in, const void *weight,
                         int32_t K, int32_t d_out, const int32_t *order, const int32_t *offsets,
                         int32_t top_k, void *y, void *workspace, size_t workspace_bytes, void *stream) {
  int rc = check_experts(dtype, N, K, top_k);
  if (!rc) rc = check_widths(d_in, d_out);
  if (rc || N == 0) return rc;
  if (!x || !weight || !order || !offsets || !y || !workspace) return fail(FGMM_ERR_INVALID, "null pointer argument");
  const size_t es = elem_size(dtype);
  if (!aligned(x, 16) || !aligned(weight, 16) || !aligned(y, es) || !aligned(workspace, 256))
    return fail(FGMM_ERR_INVALID, "x and weight must be 16-byte aligned, y to its elements, the workspace to 256 bytes");
  if (workspace_bytes < fgmm_expert_products_workspace_bytes(dtype, N, K, d_in, d_out, top_k))
    return fail(FGMM_ERR_WORKSPACE, "workspace too small");
  if ((rc = take_failure((cudaStream_t)stream))) return rc;
  const RoutePlan plan{order, offsets, N * top_k, K, top_k};
  if (!on_tensor_cores(dtype, plan.R, K, d_in, d_out).forward)
    return products_few(x, weight, dtype, N, d_in, d_out, plan, y, (cudaStream_t)stream);
  return products_tc(x, weight, dtype, N, d_in, d_out, plan, y, workspace, (cudaStream_t)stream);
}

size_t fgmm_expert_products_backward_workspace_bytes(int32_t dtype, int64_t N, int32_t K, int32_t d_in,
                                                     int32_t d_out, int32_t top_k) {
  if (check_experts(dtype, N, K, top_k) || check_widths(d_in, d_out)) return 0;
  TcParts tc = on_tensor_cores(dtype, N * top_k, K, d_in, d_out);
  tc.forward = false;
  return products_tc_workspace(dtype, N, K, d_in, d_out, top_k, tc) + dx_rows_bytes(tc, N * top_k, K, d_in, d_out);
}

int fgmm_expert_products_backward(const void *dy, const void *x, int32_t dtype, int64_t N, int32_t d_in,
                                  const void *weight, int32_t K, int32_t d_out, const int32_t *order,
                                  const int32_t *offsets, const int32_t *position, int32_t top_k,
                                  void *dx, void *d_weight, void *workspace, size_t workspace_bytes,
                                  void *stream) {
  int rc = check_experts(dtype, N, K, top_k);
  if (!rc) rc = check_widths(d_in, d_out);
  if (rc) return rc;
  const size_t es = elem_size(dtype);
  cudaStream_t st = (cudaStream_t)stream;
  if (N == 0) {
    if (d_weight) FGMM_CUDA_TRY(cudaMemsetAsync(d_weight, 0, (size_t)K * d_out * d_in * es, st));
    return FGMM_OK;
  }
  if (!dy || !order || !offsets || !workspace || (dx && (!weight || !position)) || (d_weight && !x))
    return fail(FGMM_ERR_INVALID, "null pointer argument");
  if (!aligned(dy, 16) || !aligned(x, 16) || !aligned(weight, 16) || !aligned(dx, es) || !aligned(d_weight, es) ||
      !aligned(workspace, 256))
    return fail(FGMM_ERR_INVALID, "dy, x and weight must be 16-byte aligned, the results to their elements, the workspace to 256 bytes");
  if (workspace_bytes < fgmm_expert_products_backward_workspace_bytes(dtype, N, K, d_in, d_out, top_k))
    return fail(FGMM_ERR_WORKSPACE, "workspace too small");
  if ((rc = take_failure(st))) return rc;
  const RoutePlan plan{order, offsets, N * top_k, K, top_k};
  // the rows of dx first, in fp32: their sum over a point's slots rounds once
  TcParts tc = on_tensor_cores(dtype, plan.R, K, d_in, d_out);
  tc.forward = false;
  float *dx_rows = static_cast<float *>(workspace);
  void *rest = static_cast<char *>(workspace) + dx_rows_bytes(tc, plan.R, K, d_in, d_out);
  const int parts = tc.inputs ? 1 : few_dx_parts(plan.R, K, d_in, d_out);
  if (dx && !tc.inputs) rc = products_few_dx(dy, weight, dtype, d_in, d_out, plan, dx_rows, st);
  if (!rc && d_weight && !tc.weights) rc = products_few_dw(dy, x, dtype, N, d_in, d_out, plan, d_weight, st);
  tc.inputs = tc.inputs && dx;
  tc.weights = tc.weights && d_weight;
  if (!rc && (tc.inputs || tc.weights))
    rc = products_tc_backward(dy, x, weight, dtype, N, d_in, d_out, plan, dx_rows, d_weight, tc, rest, st);
  if (rc || !dx) return rc;
  return sum_rows(dx_rows, parts, dtype, d_in, plan, position, N, dx, st);
}

const volatile int32_t *fgmm_expert_error_word(void) { return experts_error_word(); }

int fgmm_combine_experts(const void *y, int32_t dtype, int64_t N, int32_t d, const float *weights,
                         const int32_t *position, int32_t top_k, void *out, void *stream) {
  int rc = check_experts(dtype, N, 1, top_k);
  if (!rc) rc = check_widths(d, d);
  if (rc || N == 0) return rc;
  if (!y || !weights || !position || !out) return fail(FGMM_ERR_INVALID, "null pointer argument");
  if (!aligned(y, elem_size(dtype)) || !aligned(out, elem_size(dtype)))
    return fail(FGMM_ERR_INVALID, "y and out must be aligned to their elements");
  return combine_forward(y, dtype, N * top_k, d, weights, position, N, top_k, out, (cudaStream_t)stream);
}

int fgmm_combine_experts_backward(const void *d_out, const void *y, int32_t dtype, int64_t N, int32_t d,
                                  const float *weights, const int32_t *order, const int32_t *offsets,
                                  int32_t K, int32_t top_k, void *dy, float *d_weights, void *stream) {
  return fgmm_combine_experts_backward_placed(d_out, y, dtype, N, d, weights, order, offsets, nullptr, K, top_k, dy, d_weights, stream);
}

int fgmm_combine_experts_backward_placed(const void *d_out, const void *y, int32_t dtype, int64_t N, int32_t d,
                                         const float *weights, const int32_t *order, const int32_t *offsets,
                                         const int32_t *position, int32_t K, int32_t top_k, void *dy,
                                         float *d_weights, void *stream) {
  int rc = check_experts(dtype, N, K, top_k);
  if (!rc) rc = check_widths(d, d);
  if (rc || N == 0) return rc;
  if (!d_out || !y || !weights || !order || !offsets || !dy || !d_weights)
    return fail(FGMM_ERR_INVALID, "null pointer argument");
  if (!aligned(d_out, elem_size(dtype)) || !aligned(y, elem_size(dtype)) || !aligned(dy, elem_size(dtype)))
    return fail(FGMM_ERR_INVALID, "d_out, y and dy must be aligned to their elements");
  const RoutePlan plan{order, offsets, N * top_k, K, top_k};
  return combine_backward(d_out, y, dtype, d, weights, plan, position, dy, d_weights, (cudaStream_t)stream);
}

}  // extern "C"
