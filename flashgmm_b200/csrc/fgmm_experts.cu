// The grouping of routes by expert, and the weighted join of their results.
#include <algorithm>

#include "fgmm_experts.cuh"

namespace fgmm {
namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// ----------------------------------------------------------------------------- grouping
//
// A stable counting sort of the R routes by expert (routes without one last): every block counts its
// 2048 routes per key, the counts are summed over the blocks in order, and the same blocks place them.
// A warp takes 256 routes in their order, 32 at a time; lanes with the same key find each other with one
// match instruction.
constexpr int kSortWarps = 8, kSortRounds = 8, kSortItems = kSortWarps * kSortRounds * 32;

__device__ __forceinline__ int route_key(const int32_t *indices, int64_t i, int K) {
  const int e = __ldg(indices + i);
  return e >= 0 && e < K ? e : K;
}

// Counts this block's routes per key into s_count[warp][key]; rank[r] is a route's place among those
// of its key in its warp.
__device__ __forceinline__ void count_keys(const int32_t *indices, int64_t R, int K, uint16_t *s_count,
                                           int (&key)[kSortRounds], int (&rank)[kSortRounds]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, keys = K + 1;
  uint16_t *mine = s_count + warp * keys;
  for (int i = threadIdx.x; i < kSortWarps * keys; i += blockDim.x) s_count[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortItems + warp * kSortRounds * 32 + lane;
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) key[r] = base + r * 32 < R ? route_key(indices, base + r * 32, K) : -1;
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    const unsigned same = __match_any_sync(kFull, key[r]);
    const int below = __popc(same & ((1u << lane) - 1u));
    const int seen = key[r] >= 0 ? mine[key[r]] : 0;
    __syncwarp();
    if (key[r] >= 0 && below == 0) mine[key[r]] = (uint16_t)(seen + __popc(same));
    __syncwarp();
    rank[r] = seen + below;
  }
  __syncthreads();
}

// counts[key][block]
__global__ void __launch_bounds__(kSortWarps * 32) group_count_kernel(const int32_t *__restrict__ indices, int64_t R, int K,
                                                                      int blocks, int32_t *__restrict__ counts) {
  extern __shared__ uint16_t s_count[];
  int key[kSortRounds], rank[kSortRounds];
  count_keys(indices, R, K, s_count, key, rank);
  for (int e = threadIdx.x; e <= K; e += blockDim.x) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) n += s_count[w * (K + 1) + e];
    counts[(int64_t)e * blocks + blockIdx.x] = n;
  }
}

// A warp per key: exclusive sums over the blocks in place, and the key's total.
__global__ void __launch_bounds__(128) group_scan_kernel(int32_t *__restrict__ counts, int K, int blocks,
                                                         int32_t *__restrict__ totals) {
  const int e = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e > K) return;
  int32_t *c = counts + (int64_t)e * blocks;
  int run = 0;
  for (int b0 = 0; b0 < blocks; b0 += 32) {
    const int n = b0 + lane < blocks ? c[b0 + lane] : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, sum, o);
      if (lane >= o) sum += v;
    }
    if (b0 + lane < blocks) c[b0 + lane] = run + sum - n;
    run += __shfl_sync(kFull, sum, 31);
  }
  if (lane == 0) totals[e] = run;
}

__global__ void __launch_bounds__(kSortWarps * 32) group_place_kernel(const int32_t *__restrict__ indices, int64_t R, int K,
                                                                      int blocks, const int32_t *__restrict__ counts,
                                                                      const int32_t *__restrict__ totals,
                                                                      int32_t *__restrict__ order, int32_t *__restrict__ offsets,
                                                                      int32_t *__restrict__ position) {
  extern __shared__ uint16_t s_count[];
  const int keys = K + 1;
  int32_t *s_start = reinterpret_cast<int32_t *>(s_count + kSortWarps * keys);  // [keys]
  __shared__ int s_warp[kSortWarps];
  __shared__ int s_run;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int key[kSortRounds], rank[kSortRounds];
  count_keys(indices, R, K, s_count, key, rank);
  // where each key's routes begin: exclusive sums of the totals
  if (threadIdx.x == 0) s_run = 0;
  __syncthreads();
  for (int e0 = 0; e0 < keys; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    const int n = e < keys ? __ldg(totals + e) : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) s_warp[warp] = sum;
    __syncthreads();
    int start = s_run + sum - n;
    for (int w = 0; w < warp; ++w) start += s_warp[w];
    if (e < keys) {
      if (blockIdx.x == 0) offsets[e] = start;
      s_start[e] = start + __ldg(counts + (int64_t)e * blocks + blockIdx.x);
    }
    __syncthreads();
    if (threadIdx.x == blockDim.x - 1) s_run = start + n;
    __syncthreads();
  }
  // the warps before this one
  for (int e = threadIdx.x; e < keys; e += blockDim.x) {
    int run = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int n = s_count[w * keys + e];
      s_count[w * keys + e] = (uint16_t)run;
      run += n;
    }
  }
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortItems + warp * kSortRounds * 32 + lane;
#pragma unroll
  for (int r = 0; r < kSortRounds; ++r) {
    if (key[r] < 0) continue;
    const int at = s_start[key[r]] + s_count[warp * keys + key[r]] + rank[r];
    order[at] = (int32_t)(base + r * 32);
    position[base + r * 32] = key[r] < K ? at : -1;
  }
}

// ----------------------------------------------------------------------------- the join

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T *p, float (&f)[V]) {
  T raw[V];
  if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
    for (int i = 0; i < V * (int)sizeof(T) / 16; ++i)
      reinterpret_cast<uint4 *>(raw)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
  } else {
    raw[0] = __ldg(p);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f32(raw[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const float (&f)[V]) {
  T raw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) raw[i] = from_f32<T>(f[i]);
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(raw);
  else p[0] = raw[0];
}

// tpr threads share a point; each owns packs of columns.
template <typename TY, typename T, int V>
__global__ void __launch_bounds__(256) combine_kernel(const TY *__restrict__ y, int64_t R, int d, const float *__restrict__ weights,
                                                      const int32_t *__restrict__ position, int64_t N, int top_k, int tpr,
                                                      T *__restrict__ out) {
  const int64_t n = (int64_t)blockIdx.x * (256 / tpr) + threadIdx.x / tpr;
  if (n >= N) return;
  for (int c = (threadIdx.x % tpr) * V; c < d; c += tpr * V) {
    float acc[V] = {};
    for (int j = 0; j < top_k; ++j) {
      const int p = __ldg(position + n * top_k + j);
      if (p < 0 || p >= R) continue;
      const float w = weights ? __ldg(weights + n * top_k + j) : 1.0f;
      float f[V];
      load_pack<TY, V>(y + (int64_t)p * d + c, f);
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(w, f[i], acc[i]);
    }
    store_pack<T, V>(out + n * d + c, acc);
  }
}

// A warp per grouped row r of route order[r]: dy[r] = w dout[point], dw = <dout[point], y[r]>.
template <typename T, int V>
__global__ void __launch_bounds__(128) combine_backward_kernel(const T *__restrict__ d_out, const T *__restrict__ y, int d,
                                                               const float *__restrict__ weights, RoutePlan p,
                                                               T *__restrict__ dy, float *__restrict__ d_weights) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= p.R) return;
  const int id = __ldg(p.order + r);
  const bool known = id >= 0 && id < p.R, live = known && r < __ldg(p.offsets + p.K);
  const float w = live ? __ldg(weights + id) : 0.0f;
  const T *g = d_out + (int64_t)(live ? id / p.top_k : 0) * d, *yr = y + r * d;
  float dot = 0.0f;
  for (int c = lane * V; c < d; c += 32 * V) {
    float f[V] = {}, o[V];
    if (live) {
      float u[V];
      load_pack<T, V>(g + c, f);
      load_pack<T, V>(yr + c, u);
#pragma unroll
      for (int i = 0; i < V; ++i) dot = fmaf(f[i], u[i], dot);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = live ? w * f[i] : 0.0f;
    store_pack<T, V>(dy + r * d + c, o);
  }
  dot = warp_sum(dot);
  if (lane == 0 && known) d_weights[id] = dot;
}

template <typename TY, typename T>
int combine_forward_t(const TY *y, int64_t R, int d, const float *w, const int32_t *pos, int64_t N, int top_k, T *out, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = d % V == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  int tpr = 1;
  while (tpr < 256 && tpr * (vec ? V : 1) < d) tpr *= 2;
  const unsigned grid = (unsigned)cdiv(N, 256 / tpr);
  if (vec) combine_kernel<TY, T, V><<<grid, 256, 0, st>>>(y, R, d, w, pos, N, top_k, tpr, out);
  else combine_kernel<TY, T, 1><<<grid, 256, 0, st>>>(y, R, d, w, pos, N, top_k, tpr, out);
  FGMM_LAUNCH_CHECK("combine_kernel");
  return FGMM_OK;
}

template <typename T>
int combine_backward_t(const T *g, const T *y, int d, const float *w, const RoutePlan &p, T *dy, float *dw, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = d % V == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(dy) % 16 == 0;
  const unsigned grid = (unsigned)cdiv(p.R, 4);
  if (vec) combine_backward_kernel<T, V><<<grid, 128, 0, st>>>(g, y, d, w, p, dy, dw);
  else combine_backward_kernel<T, 1><<<grid, 128, 0, st>>>(g, y, d, w, p, dy, dw);
  FGMM_LAUNCH_CHECK("combine_backward_kernel");
  return FGMM_OK;
}

}  // namespace

static int sort_blocks(int64_t R) { return (int)std::max<int64_t>(1, cdiv(R, kSortItems)); }

size_t group_workspace_bytes(int64_t R, int K) {
  Carve c(nullptr);
  c.take<int32_t>((size_t)(K + 1) * sort_blocks(R));
  c.take<int32_t>(K + 1);
  return c.bytes();
}

int group_routes(const int32_t *indices, int64_t R, int K, int32_t *order, int32_t *offsets,
                 int32_t *position, void *ws, cudaStream_t st) {
  const int blocks = sort_blocks(R), keys = K + 1;
  Carve c(ws);
  int32_t *counts = c.take<int32_t>((size_t)keys * blocks), *totals = c.take<int32_t>(keys);
  const size_t smem = (size_t)kSortWarps * keys * sizeof(uint16_t), smem_place = smem + (size_t)keys * sizeof(int32_t);
  std::atomic<bool> &once = device_once_flag(8);
  if (!once.load(std::memory_order_acquire)) {
    const int most = (kMaxExperts + 1) * (kSortWarps * 2 + 4);
    FGMM_CUDA_TRY(cudaFuncSetAttribute(group_count_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    FGMM_CUDA_TRY(cudaFuncSetAttribute(group_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    once.store(true, std::memory_order_release);
  }
  group_count_kernel<<<blocks, kSortWarps * 32, smem, st>>>(indices, R, K, blocks, counts);
  FGMM_LAUNCH_CHECK("group_count_kernel");
  group_scan_kernel<<<(unsigned)cdiv(keys, 4), 128, 0, st>>>(counts, K, blocks, totals);
  FGMM_LAUNCH_CHECK("group_scan_kernel");
  group_place_kernel<<<blocks, kSortWarps * 32, smem_place, st>>>(indices, R, K, blocks, counts, totals, order, offsets, position);
  FGMM_LAUNCH_CHECK("group_place_kernel");
  return FGMM_OK;
}

int combine_forward(const void *y, int dtype, int64_t R, int d, const float *weights,
                    const int32_t *position, int64_t N, int top_k, void *out, cudaStream_t st) {
  if (dtype == FGMM_F32) return combine_forward_t((const float *)y, R, d, weights, position, N, top_k, (float *)out, st);
  if (dtype == FGMM_BF16) return combine_forward_t((const __nv_bfloat16 *)y, R, d, weights, position, N, top_k, (__nv_bfloat16 *)out, st);
  return combine_forward_t((const __half *)y, R, d, weights, position, N, top_k, (__half *)out, st);
}

int sum_rows(const float *rows, int dtype, int64_t R, int d, const int32_t *position, int64_t N, int top_k, void *out,
             cudaStream_t st) {
  if (dtype == FGMM_F32) return combine_forward_t(rows, R, d, nullptr, position, N, top_k, (float *)out, st);
  if (dtype == FGMM_BF16) return combine_forward_t(rows, R, d, nullptr, position, N, top_k, (__nv_bfloat16 *)out, st);
  return combine_forward_t(rows, R, d, nullptr, position, N, top_k, (__half *)out, st);
}

int combine_backward(const void *d_out, const void *y, int dtype, int d, const float *weights,
                     const RoutePlan &plan, void *dy, float *d_weights, cudaStream_t st) {
  if (dtype == FGMM_F32) return combine_backward_t((const float *)d_out, (const float *)y, d, weights, plan, (float *)dy, d_weights, st);
  if (dtype == FGMM_BF16) return combine_backward_t((const __nv_bfloat16 *)d_out, (const __nv_bfloat16 *)y, d, weights, plan, (__nv_bfloat16 *)dy, d_weights, st);
  return combine_backward_t((const __half *)d_out, (const __half *)y, d, weights, plan, (__half *)dy, d_weights, st);
}

}  // namespace fgmm
