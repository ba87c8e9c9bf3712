// Products of experts on the CUDA cores, for every size and type: one tiled kernel in fp32.
//
//   rows x weight   Y[r, o]  = sum_i X[point(r), i] W[e(r), o, i]
//   rows x weight^T DX[r, i] = sum_o DY[r, o] W[e(r), o, i]
//   sums over rows  DW[e, o, i] = sum_{r of e} DY[r, o] X[point(r), i]
#include <algorithm>

#include "fgmm_experts.cuh"

namespace fgmm {
namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

enum { kForward = 0, kInputs = 1, kWeights = 2 };

// A block's tile of 64 grouped rows: the expert and the rows [r0, r1).  Tiles are numbered expert
// by expert; the rows that belong to no expert follow as expert K.  False past the last tile.
__device__ bool find_tile(const RoutePlan &p, int tile, int *s_scan, int &e, int &r0, int &r1) {
  __shared__ int s_hit[3], s_base;
  const int tid = threadIdx.x, R = (int)p.R;
  if (tid == 0) { s_hit[0] = -1; s_base = 0; }
  __syncthreads();
  for (int e0 = 0; e0 <= p.K; e0 += kThreads) {
    const int c = e0 + tid;
    int lo = 0, hi = 0;
    if (c < p.K) {
      expert_rows(p.offsets, c, R, lo, hi);
    } else if (c == p.K) {
      lo = min(max(__ldg(p.offsets + p.K), 0), R);
      hi = R;
    }
    const int n = (hi - lo + kTile - 1) / kTile;
    s_scan[tid] = n;
    __syncthreads();
    for (int o = 1; o < kThreads; o <<= 1) {
      const int v = tid >= o ? s_scan[tid - o] : 0;
      __syncthreads();
      s_scan[tid] += v;
      __syncthreads();
    }
    const int end = s_base + s_scan[tid], first = end - n;
    if (c <= p.K && tile >= first && tile < end) {
      s_hit[0] = c;
      s_hit[1] = lo + (tile - first) * kTile;
      s_hit[2] = min(hi, lo + (tile - first + 1) * kTile);
    }
    __syncthreads();
    if (tid == 0) s_base += s_scan[kThreads - 1];
    __syncthreads();
    if (s_hit[0] >= 0) break;
  }
  e = s_hit[0]; r0 = s_hit[1]; r1 = s_hit[2];
  return e >= 0;
}

// C[m, n] = sum_k A[m, k] B[k, n] over a 64 x 64 tile, 4 x 4 results a thread.
template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads)
products_simt_kernel(const T *__restrict__ a, const T *__restrict__ b, int64_t N, int d_in, int d_out,
                     RoutePlan p, T *__restrict__ c) {
  __shared__ int s_scan[kThreads];
  __shared__ float s_a[kDepth][kTile + 4], s_b[kDepth][kTile + 4];
  __shared__ int s_row[kTile];  // source row of A (or, for the weights, of B) per tile row, -1: none
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int R = (int)p.R;
  int e, r0, r1;
  if (MODE == kWeights) {
    e = blockIdx.z;
    expert_rows(p.offsets, e, R, r0, r1);
  } else if (!find_tile(p, blockIdx.x, s_scan, e, r0, r1)) {
    return;
  }
  const int n0 = blockIdx.y * kTile;                        // first column of C
  const int m0 = MODE == kWeights ? blockIdx.x * kTile : 0;  // first row of C (weights only)
  const int width = MODE == kForward ? d_out : d_in;
  if (MODE != kWeights && e == p.K) {  // rows of no expert
    for (int i = tid; i < (r1 - r0) * kTile; i += kThreads) {
      const int n = n0 + i % kTile;
      if (n < width) c[(int64_t)(r0 + i / kTile) * width + n] = from_f32<T>(0.0f);
    }
    return;
  }
  const int depth = MODE == kForward ? d_in : MODE == kInputs ? d_out : r1 - r0;
  if (MODE != kWeights) {
    if (tid < kTile) {
      const int r = r0 + tid;
      int src = -1;
      if (r < r1) {
        src = MODE == kForward ? row_point(p.order, r, R, p.top_k) : r;
        if (MODE == kForward && src >= N) src = -1;
      }
      s_row[tid] = src;
    }
    __syncthreads();
  }
  const T *w = b + (MODE == kWeights ? 0 : (int64_t)e * d_out * d_in);
  float acc[4][4] = {};
  for (int k0 = 0; k0 < depth; k0 += kDepth) {
    if (MODE == kWeights) {
      if (tid < kDepth) {
        const int r = r0 + k0 + tid;
        int src = r < r1 ? row_point(p.order, r, R, p.top_k) : -1;
        s_row[tid] = src < N ? src : -1;
      }
      __syncthreads();
      for (int i = tid; i < kDepth * kTile; i += kThreads) {
        const int k = i / kTile, j = i % kTile, r = r0 + k0 + k;
        const bool live = r < r1 && s_row[k] >= 0;
        s_a[k][j] = live && m0 + j < d_out ? to_f32(a[(int64_t)r * d_out + m0 + j]) : 0.0f;
        s_b[k][j] = live && n0 + j < d_in ? to_f32(b[(int64_t)s_row[k] * d_in + n0 + j]) : 0.0f;
      }
    } else {
      for (int i = tid; i < kDepth * kTile; i += kThreads) {
        const int k = i % kDepth, m = i / kDepth, src = s_row[m];
        s_a[k][m] = src >= 0 && k0 + k < depth ? to_f32(a[(int64_t)src * depth + k0 + k]) : 0.0f;
        if (MODE == kForward) {
          s_b[k][m] = n0 + m < width && k0 + k < depth ? to_f32(w[(int64_t)(n0 + m) * d_in + k0 + k]) : 0.0f;
        } else {
          const int kb = i / kTile, n = i % kTile;
          s_b[kb][n] = n0 + n < width && k0 + kb < depth ? to_f32(w[(int64_t)(k0 + kb) * d_in + n0 + n]) : 0.0f;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      const float4 av = *reinterpret_cast<const float4 *>(&s_a[k][ty * 4]);
      const float4 bv = *reinterpret_cast<const float4 *>(&s_b[k][tx * 4]);
      const float am[4] = {av.x, av.y, av.z, av.w}, bn[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(am[i], bn[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = ty * 4 + i;
    const bool live = MODE == kWeights ? m0 + m < d_out : r0 + m < r1;
    const int64_t row = MODE == kWeights ? (int64_t)e * d_out + m0 + m : r0 + m;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (live && n < width) c[row * width + n] = from_f32<T>(acc[i][j]);
    }
  }
}

template <int MODE>
int launch(const void *a, const void *b, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p,
           void *c, cudaStream_t st) {
  const int width = MODE == kForward ? d_out : d_in;
  dim3 grid;
  if (MODE == kWeights) {
    grid = dim3((unsigned)cdiv(d_out, kTile), (unsigned)cdiv(d_in, kTile), p.K);
  } else {
    grid = dim3((unsigned)(cdiv(p.R, kTile) + std::min<int64_t>(p.K + 1, p.R)), (unsigned)cdiv(width, kTile));
  }
  if (dtype == FGMM_F32)
    products_simt_kernel<float, MODE><<<grid, kThreads, 0, st>>>((const float *)a, (const float *)b, N, d_in, d_out, p, (float *)c);
  else if (dtype == FGMM_BF16)
    products_simt_kernel<__nv_bfloat16, MODE><<<grid, kThreads, 0, st>>>((const __nv_bfloat16 *)a, (const __nv_bfloat16 *)b, N, d_in, d_out, p, (__nv_bfloat16 *)c);
  else
    products_simt_kernel<__half, MODE><<<grid, kThreads, 0, st>>>((const __half *)a, (const __half *)b, N, d_in, d_out, p, (__half *)c);
  FGMM_LAUNCH_CHECK("products_simt_kernel");
  return FGMM_OK;
}

}  // namespace

int products_simt(const void *x, const void *weight, int dtype, int64_t N, int d_in, int d_out,
                  const RoutePlan &plan, void *y, cudaStream_t st) {
  return launch<kForward>(x, weight, dtype, N, d_in, d_out, plan, y, st);
}
int products_simt_dx(const void *dy, const void *weight, int dtype, int d_in, int d_out,
                     const RoutePlan &plan, void *dx_rows, cudaStream_t st) {
  return launch<kInputs>(dy, weight, dtype, 0, d_in, d_out, plan, dx_rows, st);
}
int products_simt_dw(const void *dy, const void *x, int dtype, int64_t N, int d_in, int d_out,
                     const RoutePlan &plan, void *dweight, cudaStream_t st) {
  return launch<kWeights>(dy, x, dtype, N, d_in, d_out, plan, dweight, st);
}

}  // namespace fgmm
