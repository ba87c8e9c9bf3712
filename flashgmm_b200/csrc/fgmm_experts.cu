// Routing to experts, the grouping of routes by expert, and the weighted join.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fgmm_experts.cuh"

namespace fgmm {
namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// ------------------------------------------------------------------------------ routing
//
// s = softmax(z), sigmoid(z) or z; c = s + bias; the top_groups groups with the largest sums of
// their two best c stay; the top_k experts by c, ties to the lowest index; w = s, divided by the
// chosen ones' sum where asked, times the scale.  Without bias and groups the order of c is that of z,
// and z itself is compared.  A score of -inf or NaN is masked; +inf counts as the largest finite value.
//
// A warp owns a row and keeps c in registers as unsigned keys in the order of the floats (0: masked or
// taken), so the largest key of a warp is one redux instruction.  c is fp32 there; the order is defined
// on 64-bit values, so a row where two deciding values lie closer than the fp32 error allows (and are
// not the same score and bias) is decided again in fp64, from its scores, by route_row64.

// Unsigned order of floats; 0 is below every float.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 and 0 are equal
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// A score as it counts: masked ones as -inf.
__device__ __forceinline__ float clean(float z) { return z > -INFINITY ? fminf(z, FLT_MAX) : -INFINITY; }

struct RouteArgs {
  int64_t N, stride;
  int K, top_k, func, n_groups, top_groups;
  const float *bias;
  bool renorm;
  float scale;
};

template <typename T> __device__ __forceinline__ float score_at(const T *row, int c) { return clean(to_f32(row[c])); }

// The value c that the 64-bit order compares; m and inv_total are the softmax's.
__device__ __forceinline__ double value64(float z, int func, double m, double total, const float *bias, int c) {
  if (!(z > -INFINITY)) return -INFINITY;
  double s = (double)z;
  if (func == FGMM_SCORE_SOFTMAX) s = exp((double)z - m) / total;
  else if (func == FGMM_SCORE_SIGMOID) s = 1.0 / (1.0 + exp(-(double)z));
  if (bias) s += (double)__ldg(bias + c);
  return isnan(s) ? -INFINITY : s;
}

// (v, i) comes before (w, j): a larger value, or an equal one of a lower index.
__device__ __forceinline__ bool before(double v, int i, double w, int j) { return v > w || (v == w && i < j); }

// Decides one row in 64 bits, scanning its scores again for every choice: the next one is the first
// behind the last in (value descending, index ascending).  Lane j returns slot j's expert.
template <typename T>
__device__ __noinline__ int route_row64(const T *row, const RouteArgs &a) {
  const int lane = threadIdx.x & 31, per = a.K / a.n_groups;
  double m = -INFINITY, total = 0.0;
  if (a.func == FGMM_SCORE_SOFTMAX) {
    for (int c = lane; c < a.K; c += 32) m = fmax(m, (double)score_at(row, c));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(kFull, m, o));
    for (int c = lane; c < a.K; c += 32) {
      const float z = score_at(row, c);
      if (z > -INFINITY) total += exp((double)z - m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
  }
  unsigned kept = kFull;
  if (a.n_groups > 1) {
    double mine = -INFINITY;  // lane g: group g's sum
    for (int g = 0; g < a.n_groups; ++g) {
      double b1 = -INFINITY, b2 = -INFINITY;
      for (int c = g * per + lane; c < (g + 1) * per; c += 32) {
        const double v = value64(score_at(row, c), a.func, m, total, a.bias, c);
        if (v > b1) { b2 = b1; b1 = v; } else if (v > b2) b2 = v;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
        b2 = fmax(fmin(b1, o1), fmax(b2, o2));
        b1 = fmax(b1, o1);
      }
      if (lane == g) mine = b2 > -INFINITY ? b1 + b2 : b1;
    }
    int rank = 0;
    for (int g = 0; g < a.n_groups; ++g) {
      const double v = __shfl_sync(kFull, mine, g);
      if (before(v, g, mine, lane)) ++rank;
    }
    kept = __ballot_sync(kFull, lane < a.n_groups && rank < a.top_groups);
  }
  int chosen = -1, last = -1;
  double lv = INFINITY;
  for (int j = 0; j < a.top_k; ++j) {
    double bv = -INFINITY;
    int bi = a.K;
    for (int c = lane; c < a.K; c += 32) {
      if (a.n_groups > 1 && !((kept >> (c / per)) & 1u)) continue;
      const double v = value64(score_at(row, c), a.func, m, total, a.bias, c);
      if (v > -INFINITY && before(lv, last, v, c) && before(v, c, bv, bi)) { bv = v; bi = c; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(kFull, bv, o);
      const int oi = __shfl_xor_sync(kFull, bi, o);
      if (before(ov, oi, bv, bi)) { bv = ov; bi = oi; }
    }
    if (bi >= a.K) break;
    if (lane == j) chosen = bi;
    lv = bv;
    last = bi;
  }
  return chosen;
}

// Loads one row: value i * V + v of a lane is column (i * 32 + lane) * V + v, masked past K.
template <typename T, int VPT, int V>
__device__ __forceinline__ void load_row(const T *row, int K, int lane, float (&z)[VPT]) {
#pragma unroll
  for (int i = 0; i < VPT / V; ++i) {
    const int c = (i * 32 + lane) * V;
    if (V > 1 && c + V <= K) {
      T raw[V];
      if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(raw) = __ldg(reinterpret_cast<const uint4 *>(row + c));
      else if constexpr (V * sizeof(T) == 8) *reinterpret_cast<uint2 *>(raw) = __ldg(reinterpret_cast<const uint2 *>(row + c));
      else raw[0] = row[c];
#pragma unroll
      for (int v = 0; v < V; ++v) z[i * V + v] = clean(to_f32(raw[v]));
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) z[i * V + v] = c + v < K ? score_at(row, c + v) : -INFINITY;
    }
  }
}

template <int VPT>
__device__ __forceinline__ void softmax_terms(const float (&z)[VPT], float &m, float &total) {
  m = -INFINITY;
#pragma unroll
  for (int i = 0; i < VPT; ++i) m = fmaxf(m, z[i]);
  m = of_key(__reduce_max_sync(kFull, key_of(m)));
  if (m == -INFINITY) m = 0.0f;
  total = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) total += z[i] > -INFINITY ? expf(z[i] - m) : 0.0f;
  total = warp_sum(total);
}

// The chosen scores' shares of their sum (lane j: slot j), from the scores themselves, so that a ratio
// of values that both underflow is still their ratio; `sum` is the sum before the division.
__device__ __forceinline__ float chosen_share(float z, bool live, int func, float &sum) {
  float t = 0.0f;
  if (func == FGMM_SCORE_GIVEN) {
    t = live ? z : 0.0f;
  } else {
    float m = of_key(__reduce_max_sync(kFull, key_of(live ? z : -INFINITY)));
    if (m == -INFINITY) m = 0.0f;
    if (func == FGMM_SCORE_SOFTMAX) t = live ? expf(z - m) : 0.0f;
    else t = live ? expf(fminf(z, 0.0f) - fminf(m, 0.0f)) / (1.0f + expf(-fabsf(z))) : 0.0f;
  }
  sum = warp_sum(t);
  return sum == 0.0f ? 0.0f : t / sum;
}

template <typename T, int VPT, int V>
__global__ void __launch_bounds__(128) route_kernel(const T *__restrict__ scores, RouteArgs a,
                                                    float *__restrict__ weights, int32_t *__restrict__ indices) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  const T *row = scores + n * a.stride;
  const bool by_value = a.bias != nullptr || a.n_groups > 1;
  uint32_t key[VPT];
  float m = 0.0f, total = 1.0f, bmax = 0.0f;
  {
    float z[VPT];
    load_row<T, VPT, V>(row, a.K, lane, z);
    if (a.func == FGMM_SCORE_SOFTMAX && (by_value || !a.renorm)) softmax_terms(z, m, total);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float c = z[i];
      bool live = c > -INFINITY;
      if (by_value && live) {
        if (a.func == FGMM_SCORE_SOFTMAX) c = expf(c - m) / total;
        else if (a.func == FGMM_SCORE_SIGMOID) c = 1.0f / (1.0f + expf(-c));
        if (a.bias) {
          const float b = __ldg(a.bias + (i / V * 32 + lane) * V + i % V);
          if (b > -INFINITY) bmax = fmaxf(bmax, fabsf(b));
          c += b;
          live = c > -INFINITY;  // false for NaN
        }
      }
      key[i] = live ? key_of(c) : 0u;
    }
    if (a.bias) bmax = __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(bmax)));
  }
  // The fp32 values are off by at most a few 2^-23 of |s| and |bias|, so two of them further apart
  // than this are in the right order.
  constexpr float kTol = 1.0f / (1 << 20);
  bool sure = true;
  if (a.n_groups > 1) {
    const int per = a.K / a.n_groups;
    float mine = -INFINITY, size = 0.0f;
    for (int g = 0; g < a.n_groups; ++g) {
      uint32_t k1 = 0u, k2 = 0u;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = (i / V * 32 + lane) * V + i % V;
        const uint32_t k = c >= g * per && c < (g + 1) * per ? key[i] : 0u;
        k2 = max(k2, min(k1, k));
        k1 = max(k1, k);
      }
      const uint32_t best = __reduce_max_sync(kFull, k1);
      const unsigned holders = __ballot_sync(kFull, k1 == best);
      const uint32_t next = __reduce_max_sync(kFull, lane == __ffs(holders) - 1 ? k2 : k1);
      if (lane == g && best) {
        mine = of_key(best) + (next ? of_key(next) : 0.0f);
        size = fabsf(of_key(best)) + (next ? fabsf(of_key(next)) : 0.0f) + 2.0f * bmax;
      }
    }
    int rank = 0;
    for (int g = 0; g < a.n_groups; ++g) {
      const float v = __shfl_sync(kFull, mine, g);
      if (v > mine || (v == mine && g < lane)) ++rank;
    }
    const bool in = lane < a.n_groups && rank < a.top_groups;
    const unsigned kept = __ballot_sync(kFull, in);
    // the smallest sum that stays against the largest that goes, both live
    const bool alive = lane < a.n_groups && mine > -INFINITY;
    const uint32_t low = __reduce_min_sync(kFull, alive && in ? key_of(mine) : kFull);
    const uint32_t high = __reduce_max_sync(kFull, alive && !in ? key_of(mine) : 0u);
    size = __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(alive ? size : 0.0f)));
    if (high != 0u && low != kFull && !(of_key(low) - of_key(high) > 2.0f * kTol * size)) sure = false;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i / V * 32 + lane) * V + i % V;
      if (c < a.K && !((kept >> (c / per)) & 1u)) key[i] = 0u;
    }
  }
  int chosen = -1;
  float value = 0.0f;
  uint32_t top = 0u;  // the largest key left in this lane, and its first place
  int place = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (key[i] > top) { top = key[i]; place = i; }
  // one choice more than asked, where its distance from the last one is looked at
  const int rounds = by_value ? a.top_k + 1 : a.top_k;
  for (int j = 0; j < rounds; ++j) {
    const uint32_t best = __reduce_max_sync(kFull, top);
    if (best == 0u) break;
    const int col = (place / V * 32 + lane) * V + place % V;
    const int first = (int)__reduce_min_sync(kFull, top == best ? (unsigned)col : kFull);
    if (lane == (j & 31) && j < 32) { chosen = first; value = of_key(best); }
    if (top == best && col == first) {
      top = 0u;
      const int gone = place;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (i == gone) key[i] = 0u;
        if (key[i] > top) { top = key[i]; place = i; }
      }
    }
  }
  if (by_value && sure) {
    const float z = chosen >= 0 ? score_at(row, chosen) : 0.0f;
    const float b = chosen >= 0 && a.bias ? __ldg(a.bias + chosen) : 0.0f;
    const int prev = __shfl_up_sync(kFull, chosen, 1);
    const float pv = __shfl_up_sync(kFull, value, 1), pz = __shfl_up_sync(kFull, z, 1), pb = __shfl_up_sync(kFull, b, 1);
    bool near = false;
    if (lane > 0 && chosen >= 0 && prev >= 0 && !(pz == z && pb == b))
      near = !(pv - value > kTol * (fabsf(pv) + fabsf(value) + 2.0f * bmax));
    if (__any_sync(kFull, near) || a.top_k == 32) sure = false;  // 32 slots leave no lane for the next value
  }
  if (!sure) chosen = route_row64(row, a);
  if (lane >= a.top_k) chosen = -1;
  const bool live = chosen >= 0;
  const float z = live ? score_at(row, chosen) : 0.0f;
  float w;
  if (a.renorm) {
    float sum;
    w = chosen_share(z, live, a.func, sum);
  } else if (a.func == FGMM_SCORE_SOFTMAX) {
    w = expf(z - m) / total;
  } else {
    w = a.func == FGMM_SCORE_SIGMOID ? 1.0f / (1.0f + expf(-z)) : z;
  }
  if (lane < a.top_k) {
    weights[n * a.top_k + lane] = live ? w * a.scale : 0.0f;
    indices[n * a.top_k + lane] = chosen;
  }
}

// d z from d w.  With p the shares and g = scale dw: renormalised, the chosen get
// p (g - sum p g), times 1 - s for the sigmoid, or (g - sum p g) / sum for given values, and all
// others nothing; else the softmax gives s (g [chosen] - sum of g s over the chosen) to every score, and
// sigmoid and given values pass g s (1 - s) and g on.  One warp a row; the row of d z is written once.
template <typename T, int VPT, int V>
__global__ void __launch_bounds__(128) route_backward_kernel(const float *__restrict__ dw, const T *__restrict__ scores,
                                                             const int32_t *__restrict__ indices, RouteArgs a,
                                                             T *__restrict__ dz) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  const T *row = scores + n * a.stride;
  int chosen = lane < a.top_k ? __ldg(indices + n * a.top_k + lane) : -1;
  if (chosen >= a.K) chosen = -1;
  bool live = chosen >= 0;
  const float z = live ? score_at(row, chosen) : 0.0f;
  live = live && z > -INFINITY;  // a masked score gets no gradient
  const float g = live ? __ldg(dw + n * a.top_k + lane) * a.scale : 0.0f;
  const bool dense = a.func == FGMM_SCORE_SOFTMAX && !a.renorm;
  float zr[VPT], m = 0.0f, total = 1.0f, all = 0.0f, d;
  if (dense) {
    load_row<T, VPT, V>(row, a.K, lane, zr);
    softmax_terms(zr, m, total);
    const float s = live ? expf(z - m) / total : 0.0f;
    d = s * g;
    all = warp_sum(d);
  } else if (a.renorm) {
    float sum;
    const float p = chosen_share(z, live, a.func, sum);
    d = g - warp_sum(p * g);
    if (a.func == FGMM_SCORE_GIVEN) d = sum == 0.0f ? 0.0f : d / sum;
    else d *= a.func == FGMM_SCORE_SIGMOID ? p / (1.0f + expf(z)) : p;
  } else {
    d = g;
    if (a.func == FGMM_SCORE_SIGMOID) {
      const float e = expf(-fabsf(z));
      d = g * e / ((1.0f + e) * (1.0f + e));
    }
  }
  if (!live) { d = 0.0f; chosen = -1; }
  float out[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) out[i] = dense && zr[i] > -INFINITY ? -(expf(zr[i] - m) / total) * all : 0.0f;
  for (int j = 0; j < a.top_k; ++j) {
    const int cj = __shfl_sync(kFull, chosen, j);
    const float dj = __shfl_sync(kFull, d, j);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if ((i / V * 32 + lane) * V + i % V == cj) out[i] += dj;
  }
  T *to = dz + n * a.K;
#pragma unroll
  for (int i = 0; i < VPT / V; ++i) {
    const int c = (i * 32 + lane) * V;
    if (V > 1 && c + V <= a.K) {
      T raw[V];
#pragma unroll
      for (int v = 0; v < V; ++v) raw[v] = from_f32<T>(out[i * V + v]);
      if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(to + c) = *reinterpret_cast<uint4 *>(raw);
      else if constexpr (V * sizeof(T) == 8) *reinterpret_cast<uint2 *>(to + c) = *reinterpret_cast<uint2 *>(raw);
      else to[c] = raw[0];
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (c + v < a.K) to[c + v] = from_f32<T>(out[i * V + v]);
    }
  }
}

template <typename F> int by_row_width(int K, bool vec, F f) {
  // values a lane holds: K over 32 lanes, in vectors of four where the rows are aligned for them
#define FGMM_WIDTH(n) \
  if (K <= 32 * n) return vec && n >= 4 ? f(std::integral_constant<int, n>{}, std::integral_constant<int, (n >= 4 ? 4 : 1)>{}) \
                                        : f(std::integral_constant<int, n>{}, std::integral_constant<int, 1>{});
  FGMM_WIDTH(1) FGMM_WIDTH(2) FGMM_WIDTH(4) FGMM_WIDTH(8) FGMM_WIDTH(16) FGMM_WIDTH(32) FGMM_WIDTH(64)
  return vec ? f(std::integral_constant<int, 128>{}, std::integral_constant<int, 4>{})
             : f(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
#undef FGMM_WIDTH
}

template <typename T>
int route_forward_t(const T *z, const RouteArgs &a, float *w, int32_t *idx, cudaStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(z) % (4 * sizeof(T)) == 0 && a.stride % 4 == 0;
  return by_row_width(a.K, vec, [&](auto vpt, auto v) {
    route_kernel<T, vpt(), v()><<<(unsigned)cdiv(a.N, 4), 128, 0, st>>>(z, a, w, idx);
    FGMM_LAUNCH_CHECK("route_kernel");
    return FGMM_OK;
  });
}

template <typename T>
int route_backward_t(const float *dw, const T *z, const int32_t *idx, const RouteArgs &a, T *dz, cudaStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(z) % (4 * sizeof(T)) == 0 && a.stride % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(dz) % (4 * sizeof(T)) == 0 && a.K % 4 == 0;
  return by_row_width(a.K, vec, [&](auto vpt, auto v) {
    route_backward_kernel<T, vpt(), v()><<<(unsigned)cdiv(a.N, 4), 128, 0, st>>>(dw, z, idx, a, dz);
    FGMM_LAUNCH_CHECK("route_backward_kernel");
    return FGMM_OK;
  });
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

int route_forward(const void *scores, int dtype, int64_t N, int K, int64_t stride, const float *bias,
                  int top_k, int func, int n_groups, int top_groups, bool renorm, float scale,
                  float *weights, int32_t *indices, cudaStream_t st) {
  const RouteArgs a{N, stride, K, top_k, func, n_groups, top_groups, bias, renorm, scale};
  if (dtype == FGMM_F32) return route_forward_t((const float *)scores, a, weights, indices, st);
  if (dtype == FGMM_BF16) return route_forward_t((const __nv_bfloat16 *)scores, a, weights, indices, st);
  return route_forward_t((const __half *)scores, a, weights, indices, st);
}

int route_backward(const float *dw, const void *scores, int dtype, int64_t N, int K, int64_t stride,
                   const int32_t *indices, int top_k, int func, bool renorm, float scale, void *dz,
                   cudaStream_t st) {
  const RouteArgs a{N, stride, K, top_k, func, 1, 1, nullptr, renorm, scale};
  if (dtype == FGMM_F32) return route_backward_t(dw, (const float *)scores, indices, a, (float *)dz, st);
  if (dtype == FGMM_BF16) return route_backward_t(dw, (const __nv_bfloat16 *)scores, indices, a, (__nv_bfloat16 *)dz, st);
  return route_backward_t(dw, (const __half *)scores, indices, a, (__half *)dz, st);
}

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
