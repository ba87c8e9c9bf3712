// Products of experts that have a few rows each, on the CUDA cores.
//
// What bounds them is reading each expert's weights once (Y, DX) or writing every expert's gradient once (DW).  float32
// weights, and 16-bit ones whose rows TMA cannot read, are taken as they are: the tensor-core path would first copy all
// of them, also those of experts without a row.  A block owns a window of neighbouring grouped rows and a tile of columns; the
// rows of one expert in the window share each weight that is read.  64 experts of 512 x 1,024 float32 with one row each on
// average (some 40 of them met, 85 MB: 13 us): y 16 us, dx 28, dW 29 (134 MB written: 21 us); the rule that chooses them
// stands with more figures beside their launches.
#include <algorithm>

#include "fgmm_experts.cuh"

namespace fgmm {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256, kWarps = kThreads / 32;

// Expert of grouped row r and the end of its rows, K where r belongs to none; all lanes of a warp together (32 probes a round).
__device__ __forceinline__ int expert_of(const RoutePlan &p, int r, int &end) {
  const int lane = threadIdx.x & 31, R = (int)p.R;
  int lo = 0, n = p.K;
  while (n > 1) {
    const int step = (n + 31) / 32, i = lane * step;
    const unsigned before = __ballot_sync(kFull, i < n && (lo + i == 0 || __ldg(p.offsets + lo + i) <= r));
    const int j = before ? 31 - __clz(before) : 0;
    lo += j * step;
    n = min(step, n - j * step);
  }
  int first;
  expert_rows(p.offsets, lo, R, first, end);
  if (r >= first && r < end) return lo;
  end = R;
  return p.K;
}

// Four consecutive values, zeros from `n` on.
template <typename T, bool VEC>
__device__ __forceinline__ float4 load4(const T *p, int n) {
  if constexpr (VEC) {
    if (n <= 0) return make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (sizeof(T) == 4) return __ldg(reinterpret_cast<const float4 *>(p));
    alignas(8) T h[4];
    *reinterpret_cast<uint2 *>(h) = __ldg(reinterpret_cast<const uint2 *>(p));
    return make_float4(to_f32(h[0]), to_f32(h[1]), to_f32(h[2]), to_f32(h[3]));
  }
  return make_float4(n > 0 ? to_f32(p[0]) : 0.f, n > 1 ? to_f32(p[1]) : 0.f, n > 2 ? to_f32(p[2]) : 0.f, n > 3 ? to_f32(p[3]) : 0.f);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T *p, const float (&v)[4], int n) {
  if constexpr (VEC) {
    if (n <= 0) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      alignas(8) T h[4] = {from_f32<T>(v[0]), from_f32<T>(v[1]), from_f32<T>(v[2]), from_f32<T>(v[3])};
      *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(h);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = from_f32<T>(v[i]);
}

__device__ __forceinline__ float dot4(const float4 &a, const float4 &b, float acc) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, acc))));
}

// Y: a warp takes four outputs, its lanes four inputs each; the window's rows wait in shared memory.
constexpr int kOuts = 4, kDepth = 512;  // outputs of a warp; inputs staged at a time
template <typename T, bool VEC, int RW>
__global__ void __launch_bounds__(kThreads) few_forward_kernel(const T *__restrict__ x, const T *__restrict__ w, int64_t N, int d_in,
                                                               int d_out, RoutePlan p, T *__restrict__ y) {
  __shared__ float4 s_x[RW][kDepth / 4];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = (int)p.R;
  const int r0 = blockIdx.x * RW, r1 = min(R, r0 + RW), o0 = (blockIdx.y * kWarps + warp) * kOuts;
  for (int r = r0; r < r1;) {
    int end;
    const int e = expert_of(p, r, end);  // (every warp finds the same)
    const int n = min(end, r1) - r;
    float acc[RW][kOuts] = {};
    if (e < p.K) {
      const T *we = w + (int64_t)e * d_out * d_in;
      for (int k0 = 0; k0 < d_in; k0 += kDepth) {
        const int depth = min(kDepth, d_in - k0);
        __syncthreads();
        for (int i = threadIdx.x; i < n * (kDepth / 4); i += kThreads) {
          const int row = i / (kDepth / 4), c = i % (kDepth / 4) * 4, pt = row_point(p.order, r + row, R, p.top_k);
          s_x[row][c / 4] = load4<T, VEC>(x + (int64_t)max(pt, 0) * d_in + k0 + c, pt >= 0 && pt < N ? depth - c : 0);
        }
        __syncthreads();
#pragma unroll 2
        for (int c = lane * 4; c < depth; c += 128) {
          float4 wv[kOuts];
#pragma unroll
          for (int q = 0; q < kOuts; ++q) wv[q] = load4<T, VEC>(we + (int64_t)min(o0 + q, d_out - 1) * d_in + k0 + c, depth - c);
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            if (i >= n) break;
            const float4 xv = s_x[i][c / 4];
#pragma unroll
            for (int q = 0; q < kOuts; ++q) acc[i][q] = dot4(wv[q], xv, acc[i][q]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
      if (i >= n) break;
#pragma unroll
      for (int q = 0; q < kOuts; ++q) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[i][q] += __shfl_xor_sync(kFull, acc[i][q], o);
        if (lane == q && o0 + q < d_out) y[(int64_t)(r + i) * d_out + o0 + q] = from_f32<T>(acc[i][q]);
      }
    }
    r += n;
  }
}

// DX: a lane takes four inputs, the warps every eighth output of the block's part of them (blockIdx.z); the warps' sums meet in
// shared memory, the parts' (each [R][d_in]) in the sum over a point's slots.
template <typename T, bool VEC, int RW>
__global__ void __launch_bounds__(kThreads) few_inputs_kernel(const T *__restrict__ dy, const T *__restrict__ w, int d_in, int d_out,
                                                              RoutePlan p, int part, float *__restrict__ dx) {
  __shared__ float s_g[RW][kDepth];
  __shared__ float4 s_sum[kWarps][32];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = (int)p.R;
  const int r0 = blockIdx.x * RW, r1 = min(R, r0 + RW), c = (blockIdx.y * 32 + lane) * 4, left = d_in - c;
  const int k_begin = blockIdx.z * part, k_end = min(d_out, k_begin + part);
  dx += (int64_t)blockIdx.z * p.R * d_in;
  for (int r = r0; r < r1;) {
    int end;
    const int e = expert_of(p, r, end);
    const int n = min(end, r1) - r;
    float acc[RW][4] = {};
    if (e < p.K) {
      const T *we = w + (int64_t)e * d_out * d_in + c;
      for (int k0 = k_begin; k0 < k_end; k0 += kDepth) {
        const int depth = min(kDepth, k_end - k0);
        __syncthreads();
        for (int i = threadIdx.x; i < n * kDepth; i += kThreads) {
          const int k = i % kDepth;
          s_g[i / kDepth][k] = k < depth ? to_f32(dy[(int64_t)(r + i / kDepth) * d_out + k0 + k]) : 0.0f;
        }
        __syncthreads();
#pragma unroll 8
        for (int k = warp; k < depth; k += kWarps) {
          const float4 wv = load4<T, VEC>(we + (int64_t)(k0 + k) * d_in, left);
#pragma unroll
          for (int i = 0; i < RW; ++i) {
            if (i >= n) break;
            const float g = s_g[i][k];
            acc[i][0] = fmaf(g, wv.x, acc[i][0]);
            acc[i][1] = fmaf(g, wv.y, acc[i][1]);
            acc[i][2] = fmaf(g, wv.z, acc[i][2]);
            acc[i][3] = fmaf(g, wv.w, acc[i][3]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < RW; ++i) {
        if (i >= n) break;
        __syncthreads();
        s_sum[warp][lane] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
        __syncthreads();
        if (warp == 0) {
          float4 s = s_sum[0][lane];
#pragma unroll
          for (int q = 1; q < kWarps; ++q) {
            const float4 u = s_sum[q][lane];
            s.x += u.x; s.y += u.y; s.z += u.z; s.w += u.w;
          }
          const float v[4] = {s.x, s.y, s.z, s.w};
          if (VEC) store4<float, VEC>(dx + (int64_t)(r + i) * d_in + c, v, left);
          else store4<float, false>(dx + (int64_t)(r + i) * d_in + c, v, left);
        }
      }
    }
    if (e == p.K && warp == 0) {  // rows of no expert are read afterwards below offsets[K] only (where offsets do not ascend): zeros
      const int known = min(max(__ldg(p.offsets + p.K), 0), R);
      for (int i = 0; i < n && r + i < known; ++i) {
        const float zeros[4] = {};
        store4<float, VEC>(dx + (int64_t)(r + i) * d_in + c, zeros, left);
      }
    }
    r += n;
  }
}

// DW: a block has 32 outputs of one expert and kSpan x 128 inputs; a warp takes four outputs, a lane four inputs at a time.  The
// plan's entries of the expert's first rows are read once for the block.
constexpr int kSpan = 8, kPoints = 64;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) few_weights_kernel(const T *__restrict__ dy, const T *__restrict__ x, int64_t N, int d_in,
                                                               int d_out, RoutePlan p, int spans, T *__restrict__ dw) {
  __shared__ int s_point[kPoints];
  __shared__ __align__(16) float s_g[kPoints][32];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = (int)p.R;
  const int e = blockIdx.y, o_tile = blockIdx.x / spans * 32, o0 = o_tile + warp * kOuts, c0 = blockIdx.x % spans * kSpan * 128;
  int lo, hi;
  expert_rows(p.offsets, e, R, lo, hi);
  const int kept = min(hi - lo, kPoints);
  for (int i = threadIdx.x; i < kept; i += kThreads) {
    const int pt = row_point(p.order, lo + i, R, p.top_k);
    s_point[i] = pt < N ? pt : -1;
  }
  for (int i = threadIdx.x; i < kept * 32; i += kThreads) {
    const int o = o_tile + i % 32;
    s_g[i / 32][i % 32] = o < d_out ? to_f32(dy[(int64_t)(lo + i / 32) * d_out + o]) : 0.0f;
  }
  if (kept > 0) __syncthreads();
  for (int c = c0 + lane * 4; c < min(d_in, c0 + kSpan * 128); c += 128) {
    const int left = d_in - c;
    float acc[kOuts][4] = {};
    auto add = [&](int pt, float g0, float g1, float g2, float g3) {
      const float4 xv = load4<T, VEC>(x + (int64_t)max(pt, 0) * d_in + c, pt >= 0 ? left : 0);
      const float g[4] = {g0, g1, g2, g3}, v[4] = {xv.x, xv.y, xv.z, xv.w};
      if (pt < 0) return;  // (its dy is not looked at)
#pragma unroll
      for (int q = 0; q < kOuts; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[q][k] = fmaf(g[q], v[k], acc[q][k]);
    };
    static_assert(kOuts == 4, "one 16-byte read of s_g");
#pragma unroll 4
    for (int i = 0; i < kept; ++i) {
      const float4 g = *reinterpret_cast<const float4 *>(&s_g[i][warp * kOuts]);
      add(s_point[i], g.x, g.y, g.z, g.w);
    }
    for (int r = lo + kept; r < hi; ++r) {
      const int pt = row_point(p.order, r, R, p.top_k);
      float g[4];
#pragma unroll
      for (int q = 0; q < kOuts; ++q) g[q] = to_f32(dy[(int64_t)r * d_out + min(o0 + q, d_out - 1)]);
      add(pt < N ? pt : -1, g[0], g[1], g[2], g[3]);
    }
#pragma unroll
    for (int q = 0; q < kOuts; ++q)
      if (o0 + q < d_out) store4<T, VEC>(dw + ((int64_t)e * d_out + o0 + q) * d_in + c, acc[q], left);
  }
}

// Rows of a window: with two rows an expert and more, neighbours share the weights that are read.
int window_rows(int64_t R, int K) { return R >= 2 * (int64_t)K ? 8 : 2; }

template <typename T, bool VEC>
int forward_t(const T *x, const T *w, int64_t N, int d_in, int d_out, const RoutePlan &p, T *y, cudaStream_t st) {
  const int rows = window_rows(p.R, p.K);
  const dim3 grid((unsigned)cdiv(p.R, rows), (unsigned)cdiv(d_out, kWarps * kOuts));
  if (rows == 8) FGMM_CUDA_TRY(launch_pdl(few_forward_kernel<T, VEC, 8>, grid, dim3(kThreads), 0, st, x, w, N, d_in, d_out, p, y));
  else FGMM_CUDA_TRY(launch_pdl(few_forward_kernel<T, VEC, 2>, grid, dim3(kThreads), 0, st, x, w, N, d_in, d_out, p, y));
  return FGMM_OK;
}

template <typename T, bool VEC>
int inputs_t(const T *dy, const T *w, int d_in, int d_out, const RoutePlan &p, int parts, float *dx, cudaStream_t st) {
  const int part = (int)cdiv(d_out, parts), rows = window_rows(p.R, p.K);
  const dim3 grid((unsigned)cdiv(p.R, rows), (unsigned)cdiv(d_in, 128), parts);
  if (rows == 8) FGMM_CUDA_TRY(launch_pdl(few_inputs_kernel<T, VEC, 8>, grid, dim3(kThreads), 0, st, dy, w, d_in, d_out, p, part, dx));
  else FGMM_CUDA_TRY(launch_pdl(few_inputs_kernel<T, VEC, 2>, grid, dim3(kThreads), 0, st, dy, w, d_in, d_out, p, part, dx));
  return FGMM_OK;
}

template <typename T, bool VEC>
int weights_t(const T *dy, const T *x, int64_t N, int d_in, int d_out, const RoutePlan &p, T *dw, cudaStream_t st) {
  const int spans = (int)cdiv(d_in, kSpan * 128);
  FGMM_CUDA_TRY(launch_pdl(few_weights_kernel<T, VEC>, dim3((unsigned)(cdiv(d_out, 32) * spans), p.K), dim3(kThreads), 0, st, dy, x, N, d_in, d_out, p, spans, dw));
  return FGMM_OK;
}

// Calls f with a null pointer of the element type and whether rows of d_in elements can be read four at a time.
template <typename F> int by_type(int dtype, int d_in, const void *result, F f) {
  const bool vec = d_in % 4 == 0 && reinterpret_cast<uintptr_t>(result) % 16 == 0;
  auto go = [&](auto *t) { return vec ? f(t, std::true_type{}) : f(t, std::false_type{}); };
  if (dtype == FGMM_F32) return go((float *)nullptr);
  if (dtype == FGMM_BF16) return go((__nv_bfloat16 *)nullptr);
  return go((__half *)nullptr);
}

}  // namespace

int products_few(const void *x, const void *weight, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, void *y, cudaStream_t st) {
  return by_type(dtype, d_in, nullptr, [&](auto *t, auto vec) {
    using T = std::remove_pointer_t<decltype(t)>;
    return forward_t<T, vec()>((const T *)x, (const T *)weight, N, d_in, d_out, p, (T *)y, st);
  });
}

// Parts of the outputs: enough blocks for eight on every SM, 64 outputs a part at least.
int few_dx_parts(int64_t R, int K, int d_in, int d_out) {
  const int64_t blocks = std::max<int64_t>(1, cdiv(R, window_rows(R, K))) * cdiv(d_in, 128);
  return (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(8 * num_sms(), blocks), d_out / 64));
}

int products_few_dx(const void *dy, const void *weight, int dtype, int d_in, int d_out, const RoutePlan &p, float *dx_rows, cudaStream_t st) {
  const int parts = few_dx_parts(p.R, p.K, d_in, d_out);
  return by_type(dtype, d_in, dx_rows, [&](auto *t, auto vec) {
    using T = std::remove_pointer_t<decltype(t)>;
    return inputs_t<T, vec()>((const T *)dy, (const T *)weight, d_in, d_out, p, parts, dx_rows, st);
  });
}

int products_few_dw(const void *dy, const void *x, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, void *d_weight, cudaStream_t st) {
  return by_type(dtype, d_in, d_weight, [&](auto *t, auto vec) {
    using T = std::remove_pointer_t<decltype(t)>;
    return weights_t<T, vec()>((const T *)dy, (const T *)x, N, d_in, d_out, p, (T *)d_weight, st);
  });
}

}  // namespace fgmm
