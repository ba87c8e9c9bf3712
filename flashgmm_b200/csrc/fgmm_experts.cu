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
// A stable counting sort of the R routes by expert (routes without one last): every block counts its routes per key, the counts
// are summed over the blocks in order, and the same blocks place them.  Up to 4,096 routes are one block's work and one
// launch.  A warp takes its routes in their order, 32 at a time (ROUNDS times); lanes with the same key find each other with one
// match instruction.  Latency, not bytes, bounds it: 524,288 routes over 1,024 experts take 16 us with four rounds a warp
// and 21 us with eight, 2,097,152 routes over 256 (whose blocks' counts are a long column) 45 and 33 us.
constexpr int kSortWarps = 16, kSortThreads = kSortWarps * 32;
constexpr int sort_items(int rounds) { return kSortThreads * rounds; }

__device__ __forceinline__ int route_key(const int32_t *indices, int64_t i, int K) {
  const int e = __ldg(indices + i);
  return e >= 0 && e < K ? e : K;
}

// counts[block][key]
template <int ROUNDS>
__global__ void __launch_bounds__(kSortThreads) group_count_kernel(const int32_t *__restrict__ indices, int64_t R, int K,
                                                                   int32_t *__restrict__ counts) {
  extern __shared__ int s_hist[];
  const int keys = K + 1;
  for (int e = threadIdx.x; e < keys; e += kSortThreads) s_hist[e] = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch();  // after the wait: the place kernel reads the indices before its own
  const int64_t base = (int64_t)blockIdx.x * sort_items(ROUNDS) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i)
    if (base + i * kSortThreads < R) atomicAdd(s_hist + route_key(indices, base + i * kSortThreads, K), 1);
  __syncthreads();
  for (int e = threadIdx.x; e < keys; e += kSortThreads) counts[(int64_t)blockIdx.x * keys + e] = s_hist[e];
}

// Exclusive sums over the blocks in place, and the keys' totals: 32 keys a block, 16 threads share a key's column.
constexpr int kScanParts = 16;
__global__ void __launch_bounds__(32 * kScanParts) group_scan_kernel(int32_t *__restrict__ counts, int K, int blocks,
                                                                     int32_t *__restrict__ totals) {
  __shared__ int s_part[kScanParts][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, keys = K + 1, e = blockIdx.x * 32 + lane;
  const int per = (blocks + kScanParts - 1) / kScanParts, b0 = part * per, b1 = min(blocks, b0 + per);
  griddep_wait();
  griddep_launch();
  int sum = 0;
  if (e < keys) {
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += counts[(int64_t)b * keys + e];
  }
  s_part[part][lane] = sum;
  __syncthreads();
  if (e >= keys) return;
  int run = 0, total = 0;
#pragma unroll
  for (int q = 0; q < kScanParts; ++q) {
    if (q < part) run += s_part[q][lane];
    total += s_part[q][lane];
  }
  if (part == 0) totals[e] = total;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) {
    int32_t *c = counts + (int64_t)b * keys + e;
    const int n = *c;
    *c = run;
    run += n;
  }
}

// Places this block's routes; with ONE it is the only block and its own counts are the totals.
template <bool ONE, int ROUNDS>
__global__ void __launch_bounds__(kSortThreads) group_place_kernel(const int32_t *__restrict__ indices, int64_t R, int K,
                                                                   const int32_t *__restrict__ counts, const int32_t *__restrict__ totals,
                                                                   int32_t *__restrict__ order, int32_t *__restrict__ offsets,
                                                                   int32_t *__restrict__ position) {
  extern __shared__ uint16_t s_count[];  // [warp][keys]: routes of a key in the warps before, then places
  const int keys = K + 1;
  int32_t *s_start = reinterpret_cast<int32_t *>(s_count + kSortWarps * keys);  // [keys]
  __shared__ int s_warp[kSortWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t *mine = s_count + warp * keys;
  for (int i = threadIdx.x; i < kSortWarps * keys / 2; i += kSortThreads) reinterpret_cast<uint32_t *>(s_count)[i] = 0u;
  if (ONE) griddep_wait();
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * sort_items(ROUNDS) + warp * ROUNDS * 32 + lane;
  int key[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) key[r] = base + r * 32 < R ? route_key(indices, base + r * 32, K) : -1;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const unsigned same = __match_any_sync(kFull, key[r]);
    const int below = __popc(same & ((1u << lane) - 1u));
    const int seen = key[r] >= 0 ? mine[key[r]] : 0;
    __syncwarp();
    if (key[r] >= 0 && below == 0) mine[key[r]] = (uint16_t)(seen + __popc(same));
    __syncwarp();
    rank[r] = seen + below;
  }
  __syncthreads();
  // per key: the warps before each, and (ONE) the total
  for (int e = threadIdx.x; e < keys; e += kSortThreads) {
    int run = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const int n = s_count[w * keys + e];
      s_count[w * keys + e] = (uint16_t)run;
      run += n;
    }
    if (ONE) s_start[e] = run;
  }
  if (ONE) __syncthreads();
  else griddep_wait();
  griddep_launch();
  // where each key's routes begin: exclusive sums of the totals, a run of neighbouring keys a thread
  const int per = (keys + kSortThreads - 1) / kSortThreads, e0 = min(keys, (int)threadIdx.x * per), e1 = min(keys, e0 + per);
  int sum = 0;
  for (int e = e0; e < e1; ++e) sum += ONE ? s_start[e] : __ldg(totals + e);
  int end = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(kFull, end, o);
    if (lane >= o) end += v;
  }
  if (lane == 31) s_warp[warp] = end;
  __syncthreads();
  int start = end - sum;
  for (int w = 0; w < warp; ++w) start += s_warp[w];
  for (int e = e0; e < e1; ++e) {
    const int n = ONE ? s_start[e] : __ldg(totals + e);
    if (blockIdx.x == 0) offsets[e] = start;
    s_start[e] = start;
    start += n;
  }
  __syncthreads();
  if (!ONE) {
    for (int e = threadIdx.x; e < keys; e += kSortThreads) s_start[e] += __ldg(counts + (int64_t)blockIdx.x * keys + e);
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    if (key[r] < 0) continue;
    const int at = s_start[key[r]] + mine[key[r]] + rank[r];
    order[at] = (int32_t)(base + r * 32);
    position[base + r * 32] = key[r] < K ? at : -1;
  }
}

// ----------------------------------------------------------------------------- the join

// V consecutive elements as they are in memory (16 bytes, or 32 of fp32 rows that become a 16-bit type; 1 element unaligned).
template <typename T, int V> struct alignas(V * sizeof(T) >= 16 ? 16 : sizeof(T)) Pack {
  T v[V];
};
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_raw(const T *p) {
  Pack<T, V> r;
  if constexpr (V * sizeof(T) >= 16) {
#pragma unroll
    for (int i = 0; i < V * (int)sizeof(T) / 16; ++i)
      reinterpret_cast<uint4 *>(&r)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
  } else {
    r.v[0] = __ldg(p);
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const float (&f)[V]) {
  T raw[V];
#pragma unroll
  for (int i = 0; i < V; ++i) raw[i] = from_f32<T>(f[i]);
  if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(raw);
  else p[0] = raw[0];
}

// tpr threads share a point; each owns packs of columns and adds the rows of J slots at a time, whose places are fetched a
// point ahead and whose packs are on their way together.  ENDS: places from *rows_end on are skipped.  Memory bounds it: 8,192 points of 4 rows of 2,048 bf16 (168 MB)
// 32 us, 5.2 TB/s; 16,411 points of 2 rows of 1,000 fp32 (197 MB) 39 us.  PARTS: the rows are sums of `parts` matrices.
template <typename TY, typename T, int V, int J, bool PARTS, bool ENDS>
__global__ void __launch_bounds__(256) combine_kernel(const TY *__restrict__ y, int64_t R, int d, const float *__restrict__ weights,
                                                      const int32_t *__restrict__ position, int64_t N, int top_k, int tpr,
                                                      int parts, const int32_t *__restrict__ rows_end, T *__restrict__ out) {
  griddep_wait();
  griddep_launch();
  const int64_t end = ENDS ? min((int64_t)max(__ldg(rows_end), 0), R) : R;
  const int64_t stride = (int64_t)gridDim.x * (256 / tpr);
  int64_t n = (int64_t)blockIdx.x * (256 / tpr) + threadIdx.x / tpr;
  int p[J], ahead[J];
  float w[J], w_ahead[J];
  auto places = [&](int64_t n, int j0, int (&p)[J], float (&w)[J]) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const bool slot = n < N && j0 + j < top_k;
      p[j] = slot ? __ldg(position + n * top_k + j0 + j) : -1;
      w[j] = slot && weights ? __ldg(weights + n * top_k + j0 + j) : 1.0f;
    }
  };
  places(n, 0, ahead, w_ahead);
  for (; n < N; n += stride) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      p[j] = ahead[j];
      w[j] = w_ahead[j];
    }
    places(n + stride, 0, ahead, w_ahead);
    for (int c = (threadIdx.x % tpr) * V; c < d; c += tpr * V) {
      float acc[V] = {};
      for (int j0 = 0; j0 < top_k; j0 += J) {
        if (top_k > J && (j0 > 0 || c >= tpr * V)) places(n, j0, p, w);
        Pack<TY, V> f[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {  // (a slot without an expert reads row 0 and leaves it)
          if (p[j] >= end) p[j] = -1;
          f[j] = load_raw<TY, V>(y + (int64_t)max(p[j], 0) * d + c);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = p[j] >= 0 ? fmaf(w[j], to_f32(f[j].v[i]), acc[i]) : acc[i];
          if constexpr (PARTS) {
            for (int q = 1; q < parts && p[j] >= 0; ++q) {
              const Pack<TY, V> u = load_raw<TY, V>(y + (q * R + p[j]) * d + c);
#pragma unroll
              for (int i = 0; i < V; ++i) acc[i] = fmaf(w[j], to_f32(u.v[i]), acc[i]);
            }
          }
        }
      }
      store_pack<T, V>(out + n * d + c, acc);
    }
  }
}

// d_weights of the slots that `order` leaves out (a plan of a part of the experts) stay 0; not needed where position is at hand.
__global__ void __launch_bounds__(256) zero_weights_kernel(float *__restrict__ d_weights, int64_t R) {
  griddep_wait();
  griddep_launch();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < R; i += (int64_t)gridDim.x * 256) d_weights[i] = 0.0f;
}

// A warp per grouped row r of route order[r]: dy[r] = w dout[point], dw = <dout[point], y[r]>; U packs of both rows
// are on their way at once.  16,411 points of 2 rows of 1,000 fp32 (328 MB) 56 us, 5.9 TB/s.
template <typename T, int V, int U>
__global__ void __launch_bounds__(128) combine_backward_kernel(const T *__restrict__ d_out, const T *__restrict__ y, int d,
                                                               const float *__restrict__ weights, RoutePlan p,
                                                               const int32_t *__restrict__ position, T *__restrict__ dy,
                                                               float *__restrict__ d_weights) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= p.R) return;
  const int id = __ldg(p.order + r);
  const bool known = id >= 0 && id < p.R, live = known && r < __ldg(p.offsets + p.K);
  if (position && lane == 1) {  // slot r: 0 where its place does not lead back to it
    const int at = __ldg(position + r);
    if (at < 0 || at >= p.R || __ldg(p.order + at) != r) d_weights[r] = 0.0f;
  }
  const bool placed = known && (!position || __ldg(position + id) == r);
  T *to = dy + r * d;
  float dot = 0.0f;
  if (live) {
    const float w = __ldg(weights + id);
    const T *g = d_out + (int64_t)(id / p.top_k) * d, *yr = y + r * d;
    for (int c0 = lane * V; c0 < d; c0 += U * 32 * V) {
      Pack<T, V> f[U], u[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {  // (behind the row: its first pack again, left unused)
        const int c = c0 + q * 32 * V < d ? c0 + q * 32 * V : c0;
        f[q] = load_raw<T, V>(g + c);
        u[q] = load_raw<T, V>(yr + c);
      }
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int c = c0 + q * 32 * V;
        if (c < d) {
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            o[i] = to_f32(f[q].v[i]);
            dot = fmaf(o[i], to_f32(u[q].v[i]), dot);
            o[i] *= w;
          }
          store_pack<T, V>(to + c, o);
        }
      }
    }
    dot = warp_sum(dot);
  } else {
    const float zeros[V] = {};
    for (int c = lane * V; c < d; c += 32 * V) store_pack<T, V>(to + c, zeros);
  }
  if (lane == 0 && placed) d_weights[id] = dot;
}

template <bool ENDS, typename TY, typename T>
int combine_forward_t(const TY *y, int64_t R, int d, const float *w, const int32_t *pos, int64_t N, int top_k, T *out, cudaStream_t st, int parts = 1,
                      const int32_t *rows_end = nullptr) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = d % V == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  int tpr = 1;
  while (tpr < 256 && tpr * (vec ? V : 1) < d) tpr *= 2;
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(N, 256 / tpr), 8 * num_sms());
  auto run = [&](auto v, auto j, auto several) {
    return launch_pdl(combine_kernel<TY, T, v(), j(), several(), ENDS>, dim3(grid), dim3(256), 0, st, y, R, d, w, pos, N, top_k, tpr, parts, rows_end,
                      out);
  };
  auto by_slots = [&](auto v, auto several) {
    // (elements one by one are bound by instructions, not by loads on their way: one slot after the other)
    if (top_k == 1 || v() == 1) return run(v, std::integral_constant<int, 1>{}, several);
    if (top_k == 2) return run(v, std::integral_constant<int, 2>{}, several);
    return run(v, std::integral_constant<int, 4>{}, several);
  };
  auto by_parts = [&](auto v) {
    if constexpr (ENDS)
      if (parts > 1) return by_slots(v, std::true_type{});
    return by_slots(v, std::false_type{});
  };
  FGMM_CUDA_TRY(vec ? by_parts(std::integral_constant<int, V>{}) : by_parts(std::integral_constant<int, 1>{}));
  return FGMM_OK;
}

template <typename T>
int combine_backward_t(const T *g, const T *y, int d, const float *w, const RoutePlan &p, const int32_t *position, T *dy, float *dw, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = d % V == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0 && reinterpret_cast<uintptr_t>(g) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(dy) % 16 == 0;
  const unsigned grid = (unsigned)cdiv(p.R, 4);
  if (!position)
    FGMM_CUDA_TRY(launch_pdl(zero_weights_kernel, dim3((unsigned)std::min<int64_t>(cdiv(p.R, 256), 8 * num_sms())), dim3(256), 0, st, dw, p.R));
  auto *kernel = !vec ? combine_backward_kernel<T, 1, 4>
                 : d <= 32 * V ? combine_backward_kernel<T, V, 1>
                 : d <= 64 * V ? combine_backward_kernel<T, V, 2> : combine_backward_kernel<T, V, 4>;
  FGMM_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(128), 0, st, g, y, d, w, p, position, dy, dw));
  return FGMM_OK;
}

}  // namespace

static int sort_rounds(int64_t R) { return R <= sort_items(8) || R > (1 << 20) ? 8 : 4; }
static int sort_blocks(int64_t R) { return (int)std::max<int64_t>(1, cdiv(R, sort_items(sort_rounds(R)))); }

size_t group_workspace_bytes(int64_t R, int K) {
  Carve c(nullptr);
  c.take<int32_t>(sort_blocks(R) > 1 ? (size_t)(K + 1) * sort_blocks(R) : 0);
  c.take<int32_t>(K + 1);
  return c.bytes();
}

int group_routes(const int32_t *indices, int64_t R, int K, int32_t *order, int32_t *offsets,
                 int32_t *position, void *ws, cudaStream_t st) {
  const int blocks = sort_blocks(R), keys = K + 1;
  Carve c(ws);
  int32_t *counts = c.take<int32_t>(blocks > 1 ? (size_t)keys * blocks : 0), *totals = c.take<int32_t>(keys);
  auto place_smem = [](int n) { return align_up((size_t)kSortWarps * n * sizeof(uint16_t), 4) + (size_t)n * sizeof(int32_t); };
  std::atomic<bool> &once = device_once_flag(8);
  if (!once.load(std::memory_order_acquire)) {
    const int most = (int)place_smem(kMaxExperts + 1);
    FGMM_CUDA_TRY(cudaFuncSetAttribute(group_place_kernel<true, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    FGMM_CUDA_TRY(cudaFuncSetAttribute(group_place_kernel<false, 8>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    FGMM_CUDA_TRY(cudaFuncSetAttribute(group_place_kernel<false, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    once.store(true, std::memory_order_release);
  }
  if (blocks == 1) {
    FGMM_CUDA_TRY(launch_pdl(group_place_kernel<true, 8>, dim3(1), dim3(kSortThreads), place_smem(keys), st, indices, R, K,
                             (const int32_t *)nullptr, (const int32_t *)nullptr, order, offsets, position));
    return FGMM_OK;
  }
  const bool eight = sort_rounds(R) == 8;
  FGMM_CUDA_TRY(launch_pdl(eight ? group_count_kernel<8> : group_count_kernel<4>, dim3(blocks), dim3(kSortThreads), keys * sizeof(int), st,
                           indices, R, K, counts));
  FGMM_CUDA_TRY(launch_pdl(group_scan_kernel, dim3((unsigned)cdiv(keys, 32)), dim3(32 * kScanParts), 0, st, counts, K, blocks, totals));
  FGMM_CUDA_TRY(launch_pdl(eight ? group_place_kernel<false, 8> : group_place_kernel<false, 4>, dim3(blocks), dim3(kSortThreads), place_smem(keys),
                           st, indices, R, K, counts, totals, order, offsets, position));
  return FGMM_OK;
}

int combine_forward(const void *y, int dtype, int64_t R, int d, const float *weights,
                    const int32_t *position, int64_t N, int top_k, void *out, cudaStream_t st) {
  if (dtype == FGMM_F32) return combine_forward_t<false>((const float *)y, R, d, weights, position, N, top_k, (float *)out, st);
  if (dtype == FGMM_BF16) return combine_forward_t<false>((const __nv_bfloat16 *)y, R, d, weights, position, N, top_k, (__nv_bfloat16 *)out, st);
  return combine_forward_t<false>((const __half *)y, R, d, weights, position, N, top_k, (__half *)out, st);
}

int sum_rows(const float *rows, int parts, int dtype, int d, const RoutePlan &p, const int32_t *position, int64_t N, void *out, cudaStream_t st) {
  const int32_t *end = p.offsets + p.K;
  if (dtype == FGMM_F32) return combine_forward_t<true>(rows, p.R, d, nullptr, position, N, p.top_k, (float *)out, st, parts, end);
  if (dtype == FGMM_BF16) return combine_forward_t<true>(rows, p.R, d, nullptr, position, N, p.top_k, (__nv_bfloat16 *)out, st, parts, end);
  return combine_forward_t<true>(rows, p.R, d, nullptr, position, N, p.top_k, (__half *)out, st, parts, end);
}

int combine_backward(const void *d_out, const void *y, int dtype, int d, const float *weights,
                     const RoutePlan &plan, const int32_t *position, void *dy, float *d_weights, cudaStream_t st) {
  if (dtype == FGMM_F32) return combine_backward_t((const float *)d_out, (const float *)y, d, weights, plan, position, (float *)dy, d_weights, st);
  if (dtype == FGMM_BF16) return combine_backward_t((const __nv_bfloat16 *)d_out, (const __nv_bfloat16 *)y, d, weights, plan, position, (__nv_bfloat16 *)dy, d_weights, st);
  return combine_backward_t((const __half *)d_out, (const __half *)y, d, weights, plan, position, (__half *)dy, d_weights, st);
}

}  // namespace fgmm
