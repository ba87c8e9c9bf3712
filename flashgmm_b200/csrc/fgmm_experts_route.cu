// Routing to experts: the choice of every point's experts, their weights, and the scores' gradient.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fgmm_experts.cuh"

namespace fgmm {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// ------------------------------------------------------------------------------ routing
//
// s = softmax(z), sigmoid(z) or z; c = s + bias; the top_groups groups with the largest sums of
// their two best c stay; the top_k experts by c, ties to the lowest index; w = s, divided by the
// chosen ones' sum where asked, times the scale.  Without bias and groups the order of c is that of z,
// and z itself is compared.  A score of -inf or NaN is masked; +inf counts as the largest finite value.
//
// A row is held in registers by 8, 16 or 32 lanes.  c is fp32; the order is defined on 64-bit values, so where two deciding
// values lie closer than the fp32 error allows (and are not the same score and bias), they are compared again in fp64:
// the groups next to the border between those that stay and go, the chosen ones a lane each.  Two values more than asked
// are chosen, so that a gap behind the last slot shows that nothing else can belong there; a row without one is decided
// whole, by route_row64.

// Unsigned order of floats; 0 is below every float.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 and 0 are equal
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// A score as it counts: masked ones as -inf.
__device__ __forceinline__ float clean(float z) { return fminf(fmaxf(z, -INFINITY), FLT_MAX); }  // fmaxf drops a NaN

struct RouteArgs {
  int64_t N, stride;
  int K, top_k, func, n_groups, top_groups, per;  // per: experts of a group
  const float *bias;
  bool renorm;
  float scale;
};

template <typename T> __device__ __forceinline__ float score_at(const T *row, int c) { return clean(to_f32(row[c])); }

// 1 / (1 + e^-z) to a few 2^-23 of itself.
__device__ __forceinline__ float sigmoid(float z) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + expf(-z)));
  return r;
}

// (v, i) comes before (w, j): a larger value, or an equal one of a lower index.
__device__ __forceinline__ bool before(double v, int i, double w, int j) { return v > w || (v == w && i < j); }

// c of one expert in 64 bits; m and total are the softmax's.  Masked values are -inf.
__device__ __noinline__ double exact_value(float z, float bias, int func, float m, double total) {
  double s = z;
  if (!(z > -INFINITY)) return -INFINITY;
  if (func == FGMM_SCORE_SOFTMAX) s = exp(s - (double)m) / total;
  else if (func == FGMM_SCORE_SIGMOID) s = 1.0 / (1.0 + exp(-s));
  return fmax(s + (double)bias, -INFINITY);  // -inf for NaN
}

// The sum of a row's softmax in 64 bits; L lanes have a row.
template <typename T, int L> __device__ __noinline__ double exact_total(const T *row, int K, float m) {
  double total = 0.0;
#pragma unroll 1
  for (int c = threadIdx.x % L; c < K; c += L) total += exp((double)score_at(row, c) - (double)m);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
  return total;
}

// The sum of group g's two best, in 64 bits, the whole warp on it.
template <typename T> __device__ __noinline__ double exact_group(const T *row, const RouteArgs &a, int g, float m, double total) {
  double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll 1
  for (int c = g * a.per + (int)(threadIdx.x & 31); c < (g + 1) * a.per; c += 32) {
    const double x = exact_value(score_at(row, c), a.bias ? __ldg(a.bias + c) : 0.0f, a.func, m, total);
    b2 = fmax(b2, fmin(b1, x));
    b1 = fmax(b1, x);
  }
  __syncwarp();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
    b2 = fmax(fmin(b1, o1), fmax(b2, o2));
    b1 = fmax(b1, o1);
  }
  return b2 > -INFINITY ? b1 + b2 : b1;
}

// Decides one row in 64 bits, the whole warp on it: a lane holds the values of columns lane, lane + 32, ...
// Lane j returns slot j's expert.  Rare; its values are kept in local memory (indexed at run time), because
// registers for them would halve the occupancy of the rows that do not come here.
template <typename T, int COLS>
__device__ __noinline__ int route_row64(const T *row, const RouteArgs &a) {
  const int lane = threadIdx.x & 31, per = a.per, n = (a.K - lane + 31) / 32;
  double v[COLS];
#pragma unroll 1
  for (int i = 0; i < n; ++i) v[i] = (double)score_at(row, lane + 32 * i);
  double m = -INFINITY, total = 0.0;
  if (a.func == FGMM_SCORE_SOFTMAX) {
#pragma unroll 1
    for (int i = 0; i < n; ++i) m = fmax(m, v[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(kFull, m, o));
#pragma unroll 1
    for (int i = 0; i < n; ++i) v[i] = v[i] > -INFINITY ? exp(v[i] - m) : -INFINITY;
#pragma unroll 1
    for (int i = 0; i < n; ++i) total += fmax(v[i], 0.0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
  }
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    double s = v[i];
    if (s > -INFINITY) {
      if (a.func == FGMM_SCORE_SOFTMAX) s /= total;
      else if (a.func == FGMM_SCORE_SIGMOID) s = 1.0 / (1.0 + exp(-s));
      if (a.bias) s += (double)__ldg(a.bias + lane + 32 * i);
      v[i] = fmax(s, -INFINITY);  // -inf for NaN
    }
  }
  if (a.n_groups > 1) {
    double mine = -INFINITY;  // lane g: group g's sum
    for (int g = 0; g < a.n_groups; ++g) {
      double b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const int c = lane + 32 * i;
        const double x = c >= g * per && c < (g + 1) * per ? v[i] : -INFINITY;
        b2 = fmax(b2, fmin(b1, x));
        b1 = fmax(b1, x);
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
      const double x = __shfl_sync(kFull, mine, g);
      if (before(x, g, mine, lane)) ++rank;
    }
    const unsigned kept = __ballot_sync(kFull, lane < a.n_groups && rank < a.top_groups);
#pragma unroll 1
    for (int i = 0; i < n; ++i)
      if (!((kept >> ((lane + 32 * i) / per & 31)) & 1u)) v[i] = -INFINITY;
  }
  int chosen = -1;
  for (int j = 0; j < a.top_k; ++j) {
    double bv = -INFINITY;
    int bi = a.K;
#pragma unroll 1
    for (int i = 0; i < n; ++i)
      if (v[i] > bv) { bv = v[i]; bi = lane + 32 * i; }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(kFull, bv, o);
      const int oi = __shfl_xor_sync(kFull, bi, o);
      if (before(ov, oi, bv, bi)) { bv = ov; bi = oi; }
    }
    if (bi >= a.K) break;
    if (lane == j) chosen = bi;
    if (lane == (bi & 31)) v[bi >> 5] = -INFINITY;
  }
  return chosen;
}

// A row belongs to L neighbouring lanes (32 / L rows a warp); reductions over them, in all of them.
template <int L> __device__ __forceinline__ float seg_max(float v) {
  if constexpr (L == 32) return of_key(__reduce_max_sync(kFull, key_of(v)));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <int L> __device__ __forceinline__ float seg_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
template <int L> __device__ __forceinline__ uint32_t seg_min(uint32_t v) {
  if constexpr (L == 32) return __reduce_min_sync(kFull, v);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = min(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <int L> __device__ __forceinline__ unsigned seg_ballot(bool p) {
  const unsigned b = __ballot_sync(kFull, p);
  if constexpr (L == 32) return b;
  return b >> ((threadIdx.x & 31) / L * L) & ((1u << L) - 1u);
}
template <int L, typename X> __device__ __forceinline__ X seg_get(X v, int from) { return __shfl_sync(kFull, v, from, L); }

// One row as it is in memory: value i of lane l of the row is this column, masked past K.
template <int V, int L> __device__ __forceinline__ int column(int i, int l) { return (i / V * L + l) * V + i % V; }
template <typename T, int VPT> struct alignas(16) Row {
  T v[VPT];
};
template <typename T, int VPT, int V, int L>
__device__ __forceinline__ void load_row(const T *row, int K, int l, Row<T, VPT> &r) {
#pragma unroll
  for (int i = 0; i < VPT; i += V) {
    const int c = column<V, L>(i, l);
    if (V > 1 && c + V <= K) {
      if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(r.v + i) = __ldg(reinterpret_cast<const uint4 *>(row + c));
      else if constexpr (V * sizeof(T) == 8) *reinterpret_cast<uint2 *>(r.v + i) = __ldg(reinterpret_cast<const uint2 *>(row + c));
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) r.v[i + v] = c + v < K ? row[c + v] : from_f32<T>(-INFINITY);
    }
  }
}

// z becomes exp(z - m), m its largest; returns their sum (0 for a row without a live score).
template <int VPT, int L> __device__ __forceinline__ float softmax_terms(float (&z)[VPT], float &m) {
  float total = 0.0f;
  m = z[0];
#pragma unroll
  for (int i = 1; i < VPT; ++i) m = fmaxf(m, z[i]);
  m = seg_max<L>(m);
  if (m == -INFINITY) m = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    z[i] = expf(z[i] - m);
    total += z[i];
  }
  return seg_sum<L>(total);
}

// Given values whose sum leaves fp32 on the way: at 2^-6 of their size 32 of them do not.
template <int L> __device__ __forceinline__ float large_share(float t, float &sum) {
  const bool large = !(fabsf(sum) < INFINITY);
  const float less = seg_sum<L>(0x1p-6f * t);
  if (large) sum = 0x1p6f * less;
  const float share = large ? 0x1p-6f * t / less : t / sum;
  return (large ? less : sum) == 0.0f ? 0.0f : share;
}
template <int L> __device__ __noinline__ float call_large_share(float t, float *sum) { return large_share<L>(t, *sum); }

// The chosen scores' shares of their sum (lane j: slot j), from the scores themselves, so that a ratio
// of values that both underflow is still their ratio; `sum` is the sum before the division.
// CALL: the rare case is a call, for the registers (16,384 x 256 with bias and groups 27.0 -> 25.7 us; 65,536 x 1,024 of
// the scores alone, where it is not, 63.2 against 64.3).
template <int L, bool CALL> __device__ __forceinline__ float chosen_share(float z, bool live, int func, float &sum) {
  float t = 0.0f;
  if (func == FGMM_SCORE_GIVEN) {
    t = live ? z : 0.0f;
  } else {
    float m = seg_max<L>(live ? z : -INFINITY);
    if (m == -INFINITY) m = 0.0f;
    if (func == FGMM_SCORE_SOFTMAX) t = live ? expf(z - m) : 0.0f;
    else t = live ? __fdividef(expf(fminf(z, 0.0f) - fminf(m, 0.0f)), 1.0f + expf(-fabsf(z))) : 0.0f;
  }
  sum = seg_sum<L>(t);
  if (func == FGMM_SCORE_GIVEN && __any_sync(kFull, !(fabsf(sum) < INFINITY))) {
    if constexpr (CALL) return call_large_share<L>(t, &sum);
    else return large_share<L>(t, sum);
  }
  return sum == 0.0f ? 0.0f : t / sum;
}

__device__ __forceinline__ void top_two(float &b1, float &b2, float v1, float v2) {
  b2 = fmaxf(fmaxf(b2, v2), fminf(b1, v1));
  b1 = fmaxf(b1, v1);
}

// Masks all but the top_groups groups of a warp's row.  tol: the largest error of an s in fp32.
template <typename T, int VPT, int V>
__device__ __forceinline__ void keep_groups(float (&c)[VPT], const T *row, const RouteArgs &a, int lane, float m, float tol,
                                            float2 *s_group) {
  const int per = a.per, span = per / V;
  // a group is `span` neighbouring lanes of one pack of V: all groups' best two meet in log2 span steps
  const bool even = per % V == 0 && span <= 32 && (span & (span - 1)) == 0;
  const int shift = 31 - __clz(max(span, 1));  // lane >> shift: the lane's group within a pack
  float2 mine = make_float2(-INFINITY, 0.0f);  // lane g: group g's sum, and the magnitudes in it
  auto put = [&](int g, float b1, float b2) {
    const bool two = b2 > -INFINITY;
    // (a live group's sum stays above -inf; its magnitude then is inf, and all groups are compared in 64 bits)
    s_group[g] = make_float2(two ? fmaxf(b1 + b2, -FLT_MAX) : b1, fabsf(b1) + (two ? fabsf(b2) : 0.0f));
  };
  __syncwarp();
  if (even) {
#pragma unroll
    for (int i = 0; i < VPT; i += V) {
      float b1 = c[i], b2 = -INFINITY;
#pragma unroll
      for (int v = 1; v < V; ++v) top_two(b1, b2, c[i + v], -INFINITY);
      for (int o = 1; o < span; o <<= 1) top_two(b1, b2, __shfl_xor_sync(kFull, b1, o), __shfl_xor_sync(kFull, b2, o));
      const int g = (i / V * 32 + lane) >> shift;
      if ((lane & (span - 1)) == 0 && g < a.n_groups) put(g, b1, b2);
    }
  } else {
    for (int g = 0; g < a.n_groups; ++g) {
      float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int col = column<V, 32>(i, lane);
        top_two(b1, b2, col >= g * per && col < (g + 1) * per ? c[i] : -INFINITY, -INFINITY);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top_two(b1, b2, __shfl_xor_sync(kFull, b1, o), __shfl_xor_sync(kFull, b2, o));
      if (lane == 0) put(g, b1, b2);
    }
  }
  __syncwarp();
  if (lane < a.n_groups) mine = s_group[lane];
  // the groups that stay, one by one; low: the last one's sum
  uint32_t key = mine.x > -INFINITY ? key_of(mine.x) : 0u, kept = 0u, low = 0u;
  const float most = seg_max<32>(key ? mine.y : 0.0f);
  for (int t = 0; t < a.top_groups; ++t) {
    const uint32_t best = __reduce_max_sync(kFull, key);
    if (best == 0u) break;
    low = best;
    const int g = __ffs(__ballot_sync(kFull, key == best)) - 1;
    kept |= 1u << g;
    if (lane == g) key = 0u;
  }
  const uint32_t high = __reduce_max_sync(kFull, key);  // the largest that goes
  // a group's sum is off by tol for each of its two, and by their roundings and its own
  const float lo = of_key(low), hi = of_key(high), cut = 4.0f * tol + 0x6p-24f * most + 1e-36f;
  if (high != 0u && !(lo - hi > cut)) {
    // those that could be on either side of the border
    const bool in = mine.x - hi > cut, out = !(mine.x > -INFINITY) || lo - mine.x > cut, near = !in && !out;
    kept = __ballot_sync(kFull, in);
    const unsigned some = __ballot_sync(kFull, near);
    const double total = a.func == FGMM_SCORE_SOFTMAX ? exact_total<T, 32>(row, a.K, m) : 0.0;
    double sum = -INFINITY;
    for (unsigned left = some; left; left &= left - 1) {
      const int g = __ffs(left) - 1;
      const double x = exact_group(row, a, g, m, total);
      if (lane == g) sum = x;
    }
    int rank = __popc(kept);
    for (unsigned left = some; left; left &= left - 1) {
      const int g = __ffs(left) - 1;
      if (before(__shfl_sync(kFull, sum, g), g, sum, lane)) ++rank;
    }
    kept |= __ballot_sync(kFull, near && rank < a.top_groups);
  }
  if (even) {
#pragma unroll
    for (int i = 0; i < VPT; i += V) {
      if (!((kept >> (((i / V * 32 + lane) >> shift) & 31)) & 1u)) {  // (columns past K are masked already)
#pragma unroll
        for (int v = 0; v < V; ++v) c[i + v] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (!((kept >> (column<V, 32>(i, lane) / per & 31)) & 1u)) c[i] = -INFINITY;
  }
}

// The row's `rounds` largest values in order (lane j: the j'th, -1 where none is left): the lanes' best ones are compared,
// and the lane that gave its best looks for its next.
template <int VPT, int V, int L>
__device__ __forceinline__ void pick_by_lane(float (&c)[VPT], int rounds, int l, int &chosen, float &value) {
  float most = c[0];
#pragma unroll
  for (int i = 1; i < VPT; ++i) most = fmaxf(most, c[i]);
  for (int j = 0; j < rounds; ++j) {
    const float best = seg_max<L>(most);
    if (L == 32 && best == -INFINITY) break;  // (other rows of a shared warp go on)
    // the first place of a lane that holds it
    uint32_t col = kFull;
    const bool holds = most == best && best > -INFINITY;
    if (holds) {
#pragma unroll
      for (int i = VPT - 1; i >= 0; --i)
        if (c[i] == best) col = column<V, L>(i, l);
    }
    const unsigned holders = seg_ballot<L>(holds);
    uint32_t first = seg_get<L>(col, holders ? __ffs(holders) - 1 : 0);
    if (__any_sync(kFull, (holders & (holders - 1)) != 0)) first = seg_min<L>(col);
    if (l == j && first != kFull) { chosen = (int)first; value = best; }
    if (holds && col == first) {
      most = -INFINITY;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (column<V, L>(i, l) == (int)first) c[i] = -INFINITY;
        most = fmaxf(most, c[i]);
      }
    }
  }
}

// (v, col) as a number that is larger where it comes first: a larger value, or an equal one of a lower column.
__device__ __forceinline__ uint64_t ranked(float v, int col) { return (uint64_t)key_of(v) << 32 | ~(uint32_t)col; }

// The same for a whole warp's row.  With bar the rounds'th largest of the lanes' maxima, what reaches bar is a handful, which
// move to a lane each (through s_cand) and are picked in order.  Where many equal bar (responsibilities are mostly exact
// zeros), only what is above it moves, and the slots that leaves are filled by index.  False where more than 32 are
// above.  c may hold NaN and +inf; value_of(column) gives a value as it counts.
template <int VPT, int V, typename F>
__device__ __forceinline__ bool pick_few(const float (&c)[VPT], int rounds, int lane, uint64_t *s_cand, F value_of, int &chosen, float &value) {
  float most = c[0];
#pragma unroll
  for (int i = 1; i < VPT; ++i) most = fmaxf(most, c[i]);
  most = clean(most);
  uint32_t left = most > -INFINITY ? key_of(most) : 0u, best = 0u;
#pragma unroll 2
  for (int r = 0; r < rounds; ++r) {  // (equal maxima are taken together: bar is that much lower)
    best = __reduce_max_sync(kFull, left);
    left = left == best ? 0u : left;
  }
  const float bar = best != 0u ? of_key(best) : -FLT_MAX;  // (masked values are below it)
  constexpr int kWords = (VPT + 31) / 32;
  uint32_t some[kWords], equal[kWords];
  int n = 0;
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    some[w] = equal[w] = 0u;
#pragma unroll
    for (int i = w * 32; i < VPT && i < w * 32 + 32; ++i)
      if (c[i] >= bar) some[w] |= 1u << (i & 31);
    n += __popc(some[w]);
  }
  int count = (int)__reduce_add_sync(kFull, (unsigned)n);
  if (count > 32) {
    if (bar == FLT_MAX) return false;  // (+inf, which c may hold, equals it)
    n = 0;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
#pragma unroll
      for (int i = w * 32; i < VPT && i < w * 32 + 32; ++i)
        if (c[i] == bar) equal[w] |= 1u << (i & 31);
      some[w] &= ~equal[w];
      n += __popc(some[w]);
    }
    count = (int)__reduce_add_sync(kFull, (unsigned)n);
    if (count > 32) return false;
  }
  __syncwarp();
  if (VPT <= 8) {
    int to = n;  // the lane's first place
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, to, o);
      if (lane >= o) to += v;
    }
    to -= n;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if ((some[0] >> i) & 1u) s_cand[to++] = ranked(clean(c[i]), column<V, 32>(i, lane));
  } else
  for (int base = 0; base < count;) {
    int i = -1;
#pragma unroll
    for (int w = kWords - 1; w >= 0; --w)
      if (some[w]) i = w * 32 + __ffs(some[w]) - 1;
    const unsigned have = __ballot_sync(kFull, i >= 0);
    if (i >= 0) {
      const int col = column<V, 32>(i, lane);
      s_cand[base + __popc(have & ((1u << lane) - 1u))] = ranked(value_of(col), col);
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        if (i / 32 == w) some[w] &= some[w] - 1;
    }
    base += __popc(have);
  }
  __syncwarp();
  // each candidate's place is the number of those before it; lane j then takes the j'th
  const uint64_t x = lane < count ? s_cand[lane] : 0ull;
  int place = 0;
#pragma unroll 4
  for (int q = 0; q < count; ++q) place += s_cand[q] > x;
  if (lane < count) s_cand[32 + place] = x;
  __syncwarp();
  int j = min(rounds, count);
  if (lane < j) {
    const uint64_t u = s_cand[32 + lane];
    chosen = (int)~(uint32_t)u;
    value = of_key((uint32_t)(u >> 32));
  }
  for (; j < rounds; ++j) {  // the lowest column that equals bar
    uint32_t mine = kFull;
#pragma unroll
    for (int w = kWords - 1; w >= 0; --w)
      if (equal[w]) mine = column<V, 32>(w * 32 + __ffs(equal[w]) - 1, lane);
    const uint32_t first = __reduce_min_sync(kFull, mine);
    if (first == kFull) break;
    if (lane == j) { chosen = (int)first; value = clean(bar); }
    bool taken = mine == first;
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      if (taken && equal[w]) { equal[w] &= equal[w] - 1; taken = false; }
  }
  return true;
}

constexpr int kRouteWarps = 4;

// BY_VALUE: with a bias or groups, where the values c decide; else the scores do.
template <typename T, int VPT, int V, int L, bool BY_VALUE>
__device__ __forceinline__ void route_row(const T *row, bool exists, const Row<T, VPT> &raw, const RouteArgs &a, int l, const float *s_bias,
                                          uint64_t *s_cand, float *weights, int32_t *indices) {
  float c[VPT], m = 0.0f, total = 1.0f, inv = 1.0f;
  // How far fp32 values are off, in 2^-24 of s: a softmax's by the exponent's rounding (|z - m|, of the terms of its sum 7 on average
  // at most), the sum's length in a lane and over the lanes, exp and the quotient; a sigmoid's by exp and the reciprocal.  c = s + bias
  // adds half a step of c (taken as 2^-23).  Two values that differ by more than both errors are in the right order.
  const auto error = [&](float z, float s, float c) {
    const float steps = a.func == FGMM_SCORE_SOFTMAX ? m - z + (VPT + 20.0f) : a.func == FGMM_SCORE_SIGMOID ? 8.0f : 0.0f;
    return fmaf(0x1p-24f * steps, fabsf(s), 0x1p-23f * fabsf(c));
  };
#pragma unroll
  for (int i = 0; i < VPT; ++i) c[i] = to_f32(raw.v[i]);
  if (L < 32 || BY_VALUE || (a.func == FGMM_SCORE_SOFTMAX && !a.renorm)) {  // (pick_few takes scores as they are)
#pragma unroll
    for (int i = 0; i < VPT; ++i) c[i] = clean(c[i]);
  }
  if (a.func == FGMM_SCORE_SOFTMAX && (BY_VALUE || !a.renorm)) {
    if constexpr (BY_VALUE) {
      uint32_t live[(VPT + 31) / 32] = {};
#pragma unroll
      for (int i = 0; i < VPT; ++i) live[i / 32] |= (uint32_t)(c[i] > -INFINITY) << (i & 31);
      total = softmax_terms<VPT, L>(c, m);
      inv = 1.0f / total;
#pragma unroll
      for (int i = 0; i < VPT; ++i) c[i] = ((live[i / 32] >> (i & 31)) & 1u) ? c[i] * inv : -INFINITY;
    } else {
      float e[VPT];
#pragma unroll
      for (int i = 0; i < VPT; ++i) e[i] = c[i];
      total = softmax_terms<VPT, L>(e, m);
    }
  }
  if constexpr (BY_VALUE) {
    if (a.func == FGMM_SCORE_SIGMOID) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) c[i] = c[i] > -INFINITY ? sigmoid(c[i]) : -INFINITY;
    }
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) c[i] = fmaxf(c[i] + s_bias[column<V, L>(i, l)], -INFINITY);  // -inf for NaN
    }
    if constexpr (L == 32)
      if (a.n_groups > 1)  // (the largest s is 1 / total or 1, and |z - m| s 0.4 of it at most)
        keep_groups<T, VPT, V>(c, row, a, l, m, error(m, inv, 0.0f), reinterpret_cast<float2 *>(s_cand));
  }
  const bool rounded = BY_VALUE && (a.func != FGMM_SCORE_GIVEN || a.bias);  // c is not exact
  const int rounds = min(L, rounded ? a.top_k + 2 : a.top_k);
  int chosen = -1;
  float value = 0.0f;
  bool done = false;
  if constexpr (L == 32) {
    done = pick_few<VPT, V>(c, rounds, l, s_cand, [&](int col) {
      float v = score_at(row, col);
      if constexpr (BY_VALUE) {
        if (a.func == FGMM_SCORE_SOFTMAX) v = expf(v - m) * inv;
        else if (a.func == FGMM_SCORE_SIGMOID) v = sigmoid(v);
        if (a.bias) v += s_bias[col];
      }
      return v;
    }, chosen, value);
    if (!done) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) c[i] = clean(c[i]);
    }
  }
  if (!done) pick_by_lane<VPT, V, L>(c, rounds, l, chosen, value);
  if (rounded) {
    const bool have = chosen >= 0;
    const float z = have ? score_at(row, chosen) : 0.0f, b = have && a.bias ? s_bias[chosen] : 0.0f;
    const float off = error(z, fminf(fabsf(value) + fabsf(b), inv), value);  // (s by its bounds: the largest is 1 / total or 1)
    const int prev = __shfl_up_sync(kFull, chosen, 1, L);
    const float pv = __shfl_up_sync(kFull, value, 1, L), pz = __shfl_up_sync(kFull, z, 1, L), pb = __shfl_up_sync(kFull, b, 1, L);
    const bool apart = pv - value > __shfl_up_sync(kFull, off, 1, L) + off + 1e-36f;  // (of the value before)
    const bool near = l > 0 && l <= a.top_k && have && prev >= 0 && !apart && !(pz == z && pb == b);
    const bool border = l < rounds && (have ? l >= a.top_k && prev >= 0 && apart : l >= a.top_k || l == rounds - 1);
    // (all lanes take part in what follows, whatever their rows need)
    const bool mixed = seg_ballot<L>(near) != 0, open = seg_ballot<L>(border) == 0;
    bool whole = false;
    if (__any_sync(kFull, open)) {
      // no gap behind the slots: whether all that is near the last value is the same score and bias (then its order is known)
      const float lv = seg_get<L>(value, rounds - 1), lz = seg_get<L>(z, rounds - 1), lb = seg_get<L>(b, rounds - 1), lo = seg_get<L>(off, rounds - 1);
      bool other = false;
#pragma unroll 1
      for (int q = 0; q < VPT * L; q += L) {
        const int col = q + l;
        if (col >= a.K) break;
        const float u = score_at(row, col), v = a.bias ? s_bias[col] : 0.0f;
        // (a group's masks are in c only: its experts count as near ones here)
        float t = u;
        if (a.func == FGMM_SCORE_SOFTMAX) t = expf(u - m) * inv;
        else if (a.func == FGMM_SCORE_SIGMOID) t = sigmoid(u);
        const float x = t + v;
        if (u > -INFINITY && x > -INFINITY && !(fabsf(lv - x) > lo + error(u, t, x) + 1e-36f)) other |= !(u == lz && v == lb);
      }
      whole = seg_ballot<L>(other) != 0 && open;
    }
    if (__any_sync(kFull, mixed && !whole)) {
      const double total = a.func == FGMM_SCORE_SOFTMAX ? exact_total<T, L>(row, a.K, m) : 0.0;
      const double exact = have ? exact_value(z, b, a.func, m, total) : -INFINITY;
      int rank = 0, moved = -1;
      for (int j = 0; j < rounds; ++j) {
        const double x = seg_get<L>(exact, j);
        const int i = seg_get<L>(chosen, j);
        rank += i >= 0 && before(x, i, exact, chosen);
      }
      if (!have || l >= rounds) rank = -1;
      for (int j = 0; j < rounds; ++j) {
        const int to = seg_get<L>(rank, j), i = seg_get<L>(chosen, j);
        if (to == l) moved = i;
      }
      if (mixed) chosen = moved;
    }
    unsigned unsure = __ballot_sync(kFull, whole && exists);
    while (unsure) {  // row by row, the whole warp on it
      const int from = (__ffs(unsure) - 1) / L * L, lane = threadIdx.x & 31;
      const T *at = reinterpret_cast<const T *>(__shfl_sync(kFull, (unsigned long long)row, from));
      const int exact = __shfl_sync(kFull, route_row64<T, (VPT * L + 31) / 32>(at, a), l);
      if (lane / L * L == from) chosen = exact;
      unsure &= ~((L == 32 ? kFull : (1u << L) - 1u) << from);
    }
  }
  if (l >= a.top_k) chosen = -1;
  const bool live = chosen >= 0;
  const float z = live ? score_at(row, chosen) : 0.0f;
  float w;
  if (a.renorm) {
    float sum;
    w = chosen_share<L, BY_VALUE>(z, live, a.func, sum);
  } else if (a.func == FGMM_SCORE_SOFTMAX) {
    w = expf(z - m) / total;
  } else {
    w = a.func == FGMM_SCORE_SIGMOID ? 1.0f / (1.0f + expf(-z)) : z;
  }
  if (l < a.top_k && exists) {
    weights[l] = live ? w * a.scale : 0.0f;
    indices[l] = chosen;
  }
}

// Instructions bound it where a row is short: at 16,384 bf16 rows of 256 (8 MB, 1.3 us) it takes 10.4 us for 8 of the scores
// and 25 us with a bias and groups (680 and 1,240 instructions a row, a warp a row; with near values decided by a warp a row, whose
// one row of 64-bit work others waited for, 37 us); 65,536 rows of 1,024 fp32 responsibilities take 62 us, 4.3 TB/s.
// Resident blocks an SM: where c decides, fewer than the plain rows' (16,384 x 256 10 -> 9: 28.8 -> 25.2 us; 16,384 x 512
// 7 -> 6: 40.1 -> 38.8; x 1,024 6 -> 5: 61.6 -> 59.9, but the responsibilities 61 -> 69).  At 9 blocks the instance with a bias and
// groups has 56 registers and spills 150 bytes.
// The next row is fetched while this one is decided for up to 16 values a lane (more would cost occupancy).
template <typename T, int VPT, int V, int L, bool BY_VALUE>
__global__ void __launch_bounds__(32 * kRouteWarps, VPT <= 8 ? (BY_VALUE ? 9 : 10) : VPT <= 16 ? (BY_VALUE ? 6 : 8) : VPT <= 32 ? (BY_VALUE ? 5 : 6) : 2)
route_kernel(const T *__restrict__ scores, const RouteArgs a, float *__restrict__ weights, int32_t *__restrict__ indices) {
  constexpr int RPW = 32 / L;  // rows a warp
  __shared__ uint64_t s_cand[kRouteWarps][L == 32 ? 64 : 1];  // candidates and their order (whole warps)
  extern __shared__ float s_bias[];  // [VPT * L], zeros behind K
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L, seg = lane / L;
  const int64_t stride = (int64_t)gridDim.x * kRouteWarps * RPW;
  int64_t n = ((int64_t)blockIdx.x * kRouteWarps + warp) * RPW + seg;  // the warp's first row is n - seg
  auto at = [&](int64_t r) { return scores + (r < a.N ? r : a.N - 1) * a.stride; };
  griddep_wait();
  griddep_launch();
  Row<T, VPT> raw;
  if (n - seg < a.N) load_row<T, VPT, V, L>(at(n), a.K, l, raw);
  if (BY_VALUE && a.bias) {
    for (int c = threadIdx.x; c < VPT * L; c += blockDim.x) s_bias[c] = c < a.K ? __ldg(a.bias + c) : 0.0f;
    __syncthreads();
  }
  if (n - seg >= a.N) return;
  for (;;) {
    const int64_t next = n + stride;
    constexpr bool kAhead = VPT <= 16;  // the next row is on its way while this one is decided
    Row<T, kAhead ? VPT : 1> ahead;
    const bool more = next - seg < a.N;
    if constexpr (kAhead)
      if (more) load_row<T, VPT, V, L>(at(next), a.K, l, ahead);
    const bool exists = n < a.N;
    route_row<T, VPT, V, L, BY_VALUE>(at(n), exists, raw, a, l, s_bias, s_cand[warp], weights + n * a.top_k, indices + n * a.top_k);
    if (!more) break;
    n = next;
    if constexpr (kAhead) raw = ahead;
    else load_row<T, VPT, V, L>(at(n), a.K, l, raw);
  }
}

// d z from d w.  With p the shares and g = scale dw: renormalised, the chosen get
// p (g - sum p g), times 1 - s for the sigmoid, or (g - sum p g) / sum for given values, and all
// others nothing; else the softmax gives s (g [chosen] - sum of g s over the chosen) to every score, and
// sigmoid and given values pass g s (1 - s) and g on.  The row without the chosen ones' part is written first (the
// scores are read for the softmax only), then the lane of each slot writes its element.  65,521 fp32 rows of 128 (33 MB read, 34
// written: 10.4 us) take 10.5 us where they stay in L2 (12.1 without the blocks an SM asked for).
template <typename T, int VPT, int V, int L, bool DENSE>
__global__ void __launch_bounds__(128, DENSE ? (VPT <= 16 ? 8 : 1) : 12) route_backward_kernel(const float *__restrict__ dw, const T *__restrict__ scores,
                                                             const int32_t *__restrict__ indices, const RouteArgs a,
                                                             T *__restrict__ dz) {
  const int lane = threadIdx.x & 31, l = lane % L;
  griddep_wait();
  griddep_launch();
  const int64_t stride = (int64_t)gridDim.x * (128 / L);
  for (int64_t n = (int64_t)blockIdx.x * (128 / L) + threadIdx.x / L; n - lane / L < a.N; n += stride) {
    const bool exists = n < a.N;
    const int64_t r = exists ? n : a.N - 1;
    const T *row = scores + r * a.stride;
    Row<T, DENSE ? VPT : 1> raw;
    if constexpr (DENSE) load_row<T, VPT, V, L>(row, a.K, l, raw);
    int chosen = l < a.top_k ? __ldg(indices + r * a.top_k + l) : -1;
    if (chosen < 0 || chosen >= a.K) chosen = -1;
    const float z = chosen >= 0 ? score_at(row, chosen) : -INFINITY;
    const bool live = z > -INFINITY;  // a masked score gets no gradient
    const float g = live ? __ldg(dw + r * a.top_k + l) * a.scale : 0.0f;
    float out[DENSE ? VPT : 1], d, base = 0.0f;
    if constexpr (DENSE) {
      float m;
#pragma unroll
      for (int i = 0; i < VPT; ++i) out[i] = clean(to_f32(raw.v[i]));
      const float total = softmax_terms<VPT, L>(out, m), inv = total > 0.0f ? 1.0f / total : 0.0f;
      const float s = live ? expf(z - m) * inv : 0.0f;
      d = s * g;
      const float all = -seg_sum<L>(d);
      base = s * all;
#pragma unroll
      for (int i = 0; i < VPT; ++i) out[i] = out[i] * inv * all;
    } else {
      if (a.renorm) {
        float sum;
        const float p = chosen_share<L, false>(z, live, a.func, sum);
        d = g - seg_sum<L>(p * g);
        if (a.func == FGMM_SCORE_GIVEN) d = sum == 0.0f ? 0.0f : d / sum;
        else d *= a.func == FGMM_SCORE_SIGMOID ? p / (1.0f + expf(z)) : p;
      } else {
        d = g;
        if (a.func == FGMM_SCORE_SIGMOID) {
          const float e = expf(-fabsf(z));
          d = g * e / ((1.0f + e) * (1.0f + e));
        }
      }
    }
    if (!live) { d = 0.0f; chosen = -1; }
    float sum = base;  // slots of one expert add up, in all of their lanes alike
    for (int j = 0; j < a.top_k; ++j) {
      const int cj = seg_get<L>(chosen, j);
      const float dj = seg_get<L>(d, j);
      if (cj == chosen) sum += dj;
    }
    T *to = dz + r * a.K;
    if (exists) {
#pragma unroll
      for (int i = 0; i < VPT; i += V) {
        const int c = column<V, L>(i, l);
        if (V > 1 && c + V <= a.K) {
          alignas(16) T pack[V];
#pragma unroll
          for (int v = 0; v < V; ++v) pack[v] = from_f32<T>(DENSE ? out[DENSE ? i + v : 0] : 0.0f);
          if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(to + c) = *reinterpret_cast<uint4 *>(pack);
          else if constexpr (V * sizeof(T) == 8) *reinterpret_cast<uint2 *>(to + c) = *reinterpret_cast<uint2 *>(pack);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (c + v < a.K) to[c + v] = from_f32<T>(DENSE ? out[DENSE ? i + v : 0] : 0.0f);
        }
      }
    }
    __syncwarp();  // orders the two writes of a chosen element
    if (exists && chosen >= 0) to[chosen] = from_f32<T>(sum);
  }
}

// Lanes L of a row and values VPT a lane holds, for K columns and `slots` lanes that the choices take.  A row of up to 256
// columns takes part of a warp where few are chosen, since what a row costs beside its values is then shared
// (K = 128, two chosen: 442 -> 187 instructions a row); more choices are picked faster by a warp's reductions.  us, part of a
// warp / whole: 65,536 x 64 with 6 chosen 23 / 33, 8 28 / 35, 10 74 / 38; 16,384 x 256 with 4 10 / 10, 8 16 / 11.
// Packs are 16 bytes (8 for a 16-bit row of up to 128 columns) where the rows are aligned for them.
template <typename T, typename F> int by_row_width(int K, int slots, bool vec, F f) {
  constexpr int V = 16 / sizeof(T);
#define FGMM_WIDTH(n, v, lanes) \
  return vec ? f(std::integral_constant<int, n>{}, std::integral_constant<int, v>{}, std::integral_constant<int, lanes>{}) \
             : f(std::integral_constant<int, n>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, lanes>{});
  if (K <= 32 && slots <= 8) FGMM_WIDTH(4, 4, 8)
  if (K <= 128 && slots <= 8) FGMM_WIDTH(16, V, 8)
  if (K <= 256 && slots <= 4) FGMM_WIDTH(16, V, 16)
  if (K <= 128) FGMM_WIDTH(4, 4, 32)
  if (K <= 256) FGMM_WIDTH(8, V, 32)
  if (K <= 512) FGMM_WIDTH(16, V, 32)
  if (K <= 1024) FGMM_WIDTH(32, V, 32)
  FGMM_WIDTH(128, V, 32)
#undef FGMM_WIDTH
}

template <typename T>
int route_forward_t(const T *z, const RouteArgs &a, float *w, int32_t *idx, cudaStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(z) % 16 == 0 && a.stride * sizeof(T) % 16 == 0;
  const int slots = a.n_groups > 1 ? 32 : a.top_k + (a.bias ? 1 : 0);  // (groups are kept by whole warps)
  return by_row_width<T>(a.K, slots, vec, [&](auto vpt, auto v, auto lanes) {
    // 64 warps an SM, more than are resident (as many as are: 16,384 x 256 13.4 -> 14.3 us)
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(a.N, kRouteWarps * (32 / lanes())), (int64_t)num_sms() * 64 / kRouteWarps);
    const size_t smem = a.bias ? vpt() * lanes() * sizeof(float) : 0;
    auto *kernel = a.bias || a.n_groups > 1 ? route_kernel<T, vpt(), v(), lanes(), true> : route_kernel<T, vpt(), v(), lanes(), false>;
    FGMM_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(32 * kRouteWarps), smem, st, z, a, w, idx));
    return FGMM_OK;
  });
}

template <typename T>
int route_backward_t(const float *dw, const T *z, const int32_t *idx, const RouteArgs &a, T *dz, cudaStream_t st) {
  const bool vec = reinterpret_cast<uintptr_t>(z) % 16 == 0 && a.stride * sizeof(T) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(dz) % 16 == 0 && a.K * sizeof(T) % 16 == 0;
  // (nothing is chosen here: up to 8 slots need 8 lanes and no more)
  return by_row_width<T>(a.K, a.top_k <= 8 ? (a.top_k + 1) / 2 : a.top_k, vec, [&](auto vpt, auto v, auto lanes) {
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(a.N, 128 / lanes()), (int64_t)num_sms() * 16);
    const bool dense = a.func == FGMM_SCORE_SOFTMAX && !a.renorm;
    FGMM_CUDA_TRY(launch_pdl(dense ? route_backward_kernel<T, vpt(), v(), lanes(), true> : route_backward_kernel<T, vpt(), v(), lanes(), false>,
                             dim3(grid), dim3(128), 0, st, dw, z, idx, a, dz));
    return FGMM_OK;
  });
}

}  // namespace

int route_forward(const void *scores, int dtype, int64_t N, int K, int64_t stride, const float *bias,
                  int top_k, int func, int n_groups, int top_groups, bool renorm, float scale,
                  float *weights, int32_t *indices, cudaStream_t st) {
  const RouteArgs a{N, stride, K, top_k, func, n_groups, top_groups, K / n_groups, bias, renorm, scale};
  if (dtype == FGMM_F32) return route_forward_t((const float *)scores, a, weights, indices, st);
  if (dtype == FGMM_BF16) return route_forward_t((const __nv_bfloat16 *)scores, a, weights, indices, st);
  return route_forward_t((const __half *)scores, a, weights, indices, st);
}

int route_backward(const float *dw, const void *scores, int dtype, int64_t N, int K, int64_t stride,
                   const int32_t *indices, int top_k, int func, bool renorm, float scale, void *dz,
                   cudaStream_t st) {
  const RouteArgs a{N, stride, K, top_k, func, 1, 1, K, nullptr, renorm, scale};
  if (dtype == FGMM_F32) return route_backward_t(dw, (const float *)scores, indices, a, (float *)dz, st);
  if (dtype == FGMM_BF16) return route_backward_t(dw, (const __nv_bfloat16 *)scores, indices, a, (__nv_bfloat16 *)dz, st);
  return route_backward_t(dw, (const __half *)scores, indices, a, (__half *)dz, st);
}

}  // namespace fgmm
