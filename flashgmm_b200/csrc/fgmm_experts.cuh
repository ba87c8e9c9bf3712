// Shared by the expert operators (fgmm_experts.cu, fgmm_experts_route.cu, fgmm_experts_tc.cu):
// element types, the grouped rows' plan, and the launchers behind the C ABI.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fgmm_common.cuh"

namespace fgmm {

constexpr int kMaxExperts = FGMM_MAX_EXPERTS;  // a block keeps a count per expert in shared memory

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

inline int elem_size(int dtype) { return dtype == FGMM_F32 ? 4 : 2; }

// The routes grouped by expert.  Grouped row r (0 <= r < offsets[K]) belongs to the expert e with
// offsets[e] <= r < offsets[e + 1] and to route order[r], which is slot order[r] % top_k of point
// order[r] / top_k; the rows behind offsets[K] belong to routes without an expert.
struct RoutePlan {
  const int32_t *order;    // [R]
  const int32_t *offsets;  // [K + 1]
  int64_t R;
  int32_t K, top_k;
};

// Rows of expert e, whatever `offsets` holds: 0 <= lo <= hi <= R, and no row below the last expert's end
// is left out (the first expert begins at row 0).
__device__ __forceinline__ void expert_rows(const int32_t *offsets, int e, int R, int &lo, int &hi) {
  lo = e == 0 ? 0 : min(max(__ldg(offsets + e), 0), R);
  hi = min(max(__ldg(offsets + e + 1), lo), R);
}

// Point of grouped row r, -1 where `order` holds no route.
__device__ __forceinline__ int row_point(const int32_t *order, int r, int R, int top_k) {
  const int id = __ldg(order + r);
  return id >= 0 && id < R ? id / top_k : -1;
}

// ---- fgmm_experts_route.cu ----
int route_forward(const void *scores, int dtype, int64_t N, int K, int64_t stride, const float *bias,
                  int top_k, int func, int n_groups, int top_groups, bool renorm, float scale,
                  float *weights, int32_t *indices, cudaStream_t st);
int route_backward(const float *dw, const void *scores, int dtype, int64_t N, int K, int64_t stride,
                   const int32_t *indices, int top_k, int func, bool renorm, float scale, void *dz,
                   cudaStream_t st);

// ---- fgmm_experts.cu ----
size_t group_workspace_bytes(int64_t R, int K);
int group_routes(const int32_t *indices, int64_t R, int K, int32_t *order, int32_t *offsets,
                 int32_t *position, void *ws, cudaStream_t st);
// out[n] = sum_j w[n][j] y[position[n][j]], positions outside [0, R) skipped.
int combine_forward(const void *y, int dtype, int64_t R, int d, const float *weights,
                    const int32_t *position, int64_t N, int top_k, void *out, cudaStream_t st);
// The same of fp32 rows[parts][R][d] with weights 1, summed over the parts; rows behind offsets[K], which no kernel wrote, are
// skipped whatever position says.
int sum_rows(const float *rows, int parts, int dtype, int d, const RoutePlan &plan, const int32_t *position, int64_t N, void *out,
             cudaStream_t st);
// Without position (which may be null) a launch more sets the gradients of slots that order leaves out.
int combine_backward(const void *d_out, const void *y, int dtype, int d, const float *weights,
                     const RoutePlan &plan, const int32_t *position, void *dy, float *d_weights, cudaStream_t st);

// ---- fgmm_experts_few.cu: CUDA-core products for a few rows an expert ----
int products_few(const void *x, const void *weight, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, void *y, cudaStream_t st);
int few_dx_parts(int64_t R, int K, int d_in, int d_out);  // dx_rows there: [parts][R][d_in]
int products_few_dx(const void *dy, const void *weight, int dtype, int d_in, int d_out, const RoutePlan &p, float *dx_rows, cudaStream_t st);
int products_few_dw(const void *dy, const void *x, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, void *d_weight, cudaStream_t st);

// ---- fgmm_experts_tc.cu: tensor-core products ----
int take_failure(cudaStream_t st);  // the error of an earlier product whose wait ran out, once
int *experts_error_word();
// Which of the three products run there; the others cost no workspace.
struct TcParts {
  bool forward, inputs, weights;
};
size_t products_tc_workspace(int dtype, int64_t N, int K, int d_in, int d_out, int top_k, const TcParts &parts);
int products_tc(const void *x, const void *weight, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, void *y,
                void *ws, cudaStream_t st);
// dx_rows[R][d_in] and d_weight, as parts says.
int products_tc_backward(const void *dy, const void *x, const void *weight, int dtype, int64_t N, int d_in, int d_out,
                         const RoutePlan &p, float *dx_rows, void *d_weight, const TcParts &parts, void *ws, cudaStream_t st);

}  // namespace fgmm
