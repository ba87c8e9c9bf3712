// Products of experts on the tcgen05 tensor cores.
//
//   rows x weight    Y[r, o]     = sum_i X[point(r), i] W[e(r), o, i]
//   rows x weight^T  DX[r, i]    = sum_o DY[r, o] W[e(r), o, i]
//   sums over rows   DW[e, o, i] = sum_{r of e} DY[r, o] X[point(r), i]
//
// One persistent, warp-specialised kernel: a TMA warp and four gathering warps fill a ring of stages, one thread
// issues tcgen05.mma into a double-buffered tensor-memory accumulator, eight warps read it back and write
// the results, and the next tile's products run meanwhile.  A tile has M = 128 rows of one expert (or, for
// DW, 128 of its output dimensions) and NT columns; a stage holds 64 elements of the contraction.
//   * The points' rows of X are gathered straight from the points' matrix by 16-byte cp.async, in the
//     swizzled layout that TMA writes, so a grouped copy of X is never made.  (TMA gather4 measured 80 cycles for
//     four 128-byte rows; a grouped copy read by TMA made DW slower: 32,768 rows 1,024 x 2,048 197 -> 216 us, 8,186 rows
//     1,000 x 1,016 60 -> 107 us.)  Rows a tile does not have are not loaded: their accumulator rows hold leftovers
//     that nobody reads.  Where the rows are the contraction (DW), those behind the expert's last one are zeros in
//     both operands.
//   * W is fetched as a box of its 3-D tensor, K-major for Y, and MN-major, without a transposed copy, for DX.
//   * float32 operands are three bf16 planes (x = b0 + b1 + b2, 24 bits together), laid out by
//     split_planes_kernel, and the six products that matter (b0 b0 into one accumulator; b0 b1, b1 b0, b1 b1,
//     b0 b2 and b2 b0, 2^-8 and less of it, into another).  Tensor-memory accumulation truncates, so the
//     first is drained into fp32 registers every 256 elements of the contraction (the second with the tile: where every factor is the
//     same, so that its products have one sign, it loses 2^-21.6 of the result over 65,536 elements, 2^-17 over 2^20).
//   * 16-bit products are drained every 8,192 elements: truncation takes up to 2^-23 of the sum for every 8, of a sum of one sign
//     2^-27.3 an element (8,192: 2^-14.3, a tenth of the rounding to fp16; undrained 2^20 rows lost 0.6 %).  The sums of a
//     longer contraction wait in a tile of fp32 for each block, whose threads read and write their own elements only (dW of 64
//     experts of 16,384 rows, 256 -> 896: 645 -> 677 us; y of 32,768 -> 1,024, 4,096 rows: 239 -> 254).
//   * 16-bit operands whose rows are no multiple of 16 bytes are copied to padded rows first (TMA strides).
// What bounds it is shared memory at 128 bytes a cycle: a stage of 128 x 256 x 64 16-bit products writes and reads 96 KB, 768
// cycles, for 512 of tensor time; one of three planes and 128 columns 288 KB, 2,304 for 1,536.  8,192 points with 4 of 64
// experts, 1,024 -> 2,048 bf16: 152 us, 905 TFLOP/s, 55 % of a library matrix product's; 65,536 points with 2 of 256, 128 ->
// 128 fp32: 77 us with the planes' copies (20), six times its 57 TFLOP/s in bf16 products.  Two SMs on one tile would halve the
// weights' part of that, but its 256 rows fit the ends of the experts' rows worse (14 % more products there).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <algorithm>
#include <atomic>
#include <mutex>

#include "fgmm_experts.cuh"
#include "sm100_ptx.cuh"

namespace fgmm {
using namespace ptx;

namespace {

constexpr int BM = 128;       // tile rows (MMA M)
constexpr int KCH = 64;       // contraction elements of a stage (128-byte rows)
constexpr int kGather = 128;   // gathering threads: warps 2-5
constexpr int kEpiWarps = 8;   // warps 6-13: two per tensor-memory lane quarter, half of the columns each
constexpr int kThreads = 64 + kGather + 32 * kEpiWarps;  // warp 0 TMA, warp 1 MMA
constexpr int kList = 64;      // tiles of a block that are found ahead
constexpr int kSegment = 4;   // stages between drains of a float32 product (256 elements)
constexpr int kLong = 128;    // of a 16-bit product (8,192 elements)

// A load that stays where it is written (a plan's entry fetched a stage ahead of its use).
__device__ __forceinline__ int ld_now(const int32_t *p) {
  int v;
  asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

// A wait of this launch ran out: the host learns of it without synchronising.
__device__ __noinline__ void report(int *failed) {
  const int code = *(volatile int *)&g_dev_error;
  *(volatile int *)failed = code != 0 ? code : kErrWaitDrain;
  __threadfence_system();
}

enum { kForward = 0, kInputs = 1, kWeights = 2 };

template <int NT, bool SPLIT>
struct Shape {
  static constexpr int kPlanes = SPLIT ? 3 : 1;
  static constexpr int kA = BM * KCH * 2, kB = NT * KCH * 2;  // bytes of one plane's tile
  static constexpr int kStage = kPlanes * (kA + kB);
  static constexpr int kStages = (192 * 1024) / kStage;
  static constexpr int kOut = kEpiWarps * 16 * 128;  // a 16-row, 128-byte staging tile for each epilogue warp
  static constexpr int kBars = 320;
  static constexpr int smem(int K) { return 1024 + kStages * kStage + kOut + kBars + kList * 16 + (K + 1) * 4; }
  static_assert(kStages >= 2, "shared-memory budget");
  static_assert(smem(kMaxExperts) <= 227 * 1024, "shared-memory budget");
};

// DW is divided into pieces of at most `most` stages: piece by piece of an expert, all its tiles (so that the blocks at work
// read the same rows), the pieces going round the blocks.  An expert with most of the rows is shared by many blocks
// that way (65,536 points over 256 experts, 128 x 128: 137 us of one tile's block alone, while the others had 9 % of its
// work).  Where an expert has more than one piece, its pieces go as fp32 tiles to slots that join_pieces_kernel adds in order.
// An expert without rows has one piece, of zeros.
struct Pieces {
  const int *first;   // [K + 1] pieces (of a tile) of the experts before
  const int *slot;    // [K + 1] those of them that are joined
  const int *joined;  // [K + 1] experts before that are joined
  float *tiles;       // [slots][BM][NT]
  int most, slots;
};

struct TcArgs {
  RoutePlan plan;
  int d_in, d_out;
  int a_plane, b_plane;  // columns between the planes of A's and B's rows (float32)
  const uint16_t *a_rows, *b_rows;  // the same matrices for the gathering warps
  int a_cols, b_cols;               // columns of their rows in memory
  uint32_t idesc;
  Pieces pieces;  // DW
  float *sums;    // [blocks][NT][BM]: a tile whose contraction is longer than kLong stages (16 bits)
  uint32_t div_mul, div_shift;  // n / top_k = n * div_mul >> div_shift for n < 2^31
  int vec, vec32;  // rows of the result start on 16-byte, 32-byte boundaries
  int *failed;     // the host's word for a wait that ran out
};

// What one tile covers.  For Y and DX: `rows` rows from r0 of expert e, columns from n0.  For DW: `rows` output dimensions
// from m0, columns from n0, contraction over the rows [r0, r1).  Stages [c0, c1) of the contraction; a piece of
// a DW tile goes to slot `slot` of the partial results (-1: a whole tile).
struct Tile {
  int e, r0, r1, rows, m0, n0, c0, c1, slot;
};

// Last expert e with s_first[e] <= m.
__device__ __forceinline__ int find_expert(const int *s_first, int K, int m) {
  int lo = 0, hi = K;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s_first[mid] <= m) lo = mid; else hi = mid;
  }
  return lo;
}

// a + b up to `most` (all >= 0).  Offsets that do not ascend can claim more tiles than 32 bits count: those past `most` are left out.
__device__ __forceinline__ int add_to(int a, int b, int most) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)most); }

__device__ __forceinline__ int expert_stages(const RoutePlan &p, int e) {
  int lo, hi;
  expert_rows(p.offsets, e, (int)p.R, lo, hi);
  return max(1, (hi - lo + KCH - 1) / KCH);
}

// The tiles of this block, in order.
template <int MODE, int NT>
struct Tiles {
  const TcArgs &a;
  const int *s_first;   // tiles of rows (Y, DX) or pieces (DW) of the experts before
  const int4 *s_list;   // Y, DX: the block's first kList tiles, found by its threads at once
  int n_tiles, total, i = 0;

  __device__ Tiles(const TcArgs &args, const int *sf, const int4 *sl) : a(args), s_first(sf), s_list(sl) {
    n_tiles = ((MODE == kForward ? a.d_out : a.d_in) + NT - 1) / NT;
    total = s_first[a.plan.K] * (MODE == kWeights ? per() : n_tiles);
  }
  __device__ int per() const { return (a.d_out + BM - 1) / BM * n_tiles; }  // tiles of an expert's DW
  __device__ int4 find(int t) const {  // {expert, first row, rows, first column}
    const int m = t / n_tiles, e = find_expert(s_first, a.plan.K, m);
    int lo, hi;
    expert_rows(a.plan.offsets, e, (int)a.plan.R, lo, hi);
    lo += (m - s_first[e]) * BM;
    return make_int4(e, lo, max(0, min(BM, hi - lo)), t % n_tiles * NT);
  }
  __device__ bool next(Tile &x) {
    const int64_t t = blockIdx.x + (int64_t)i * gridDim.x;
    if (t >= total) return false;
    if (MODE == kWeights) {
      const int m = (int)t / per(), tile = (int)t % per();
      x.e = find_expert(s_first, a.plan.K, m);
      const int piece = m - s_first[x.e], pieces = s_first[x.e + 1] - s_first[x.e];
      x.m0 = tile / n_tiles * BM;
      x.n0 = tile % n_tiles * NT;
      x.rows = min(BM, a.d_out - x.m0);
      expert_rows(a.plan.offsets, x.e, (int)a.plan.R, x.r0, x.r1);
      x.c0 = piece * a.pieces.most;
      x.c1 = min(max(1, (x.r1 - x.r0 + KCH - 1) / KCH), x.c0 + a.pieces.most);
      x.slot = -1;
      if (pieces > 1) x.slot = (int)min(((int64_t)__ldg(a.pieces.slot + x.e) + piece) * per() + tile, (int64_t)a.pieces.slots - 1);
      ++i;
    } else {
      const int4 f = i < kList ? s_list[i] : find((int)t);
      ++i;
      x.e = f.x;
      x.r0 = f.y;
      x.rows = f.z;
      x.n0 = f.w;
      x.r1 = x.r0 + x.rows;
      x.m0 = x.c0 = 0;
      x.c1 = ((MODE == kForward ? a.d_in : a.d_out) + KCH - 1) / KCH;
      x.slot = -1;
    }
    return true;
  }
};

template <typename OUT>
__device__ __forceinline__ uint4 pack16(const float *v) {
  if constexpr (sizeof(OUT) == 4) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    OUT h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_f32<OUT>(v[i]);
    return *reinterpret_cast<uint4 *>(h);
  }
}

// LONG: a 16-bit contraction may have more than kLong stages (instances of their own for Y and DX, whose others keep their
// registers).
template <int MODE, int NT, bool SPLIT, bool LONG, typename OUT>
__global__ void __launch_bounds__(kThreads, 1)
experts_tc_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                  const __grid_constant__ TcArgs a, OUT *__restrict__ out) {
  using Sh = Shape<NT, SPLIT>;
  constexpr int P = Sh::kPlanes, S = Sh::kStages;
  constexpr int kSeg = SPLIT ? kSegment : LONG ? kLong : 1 << 26;  // (more than any contraction has)
  constexpr int kCols = SPLIT ? 4 * NT : 2 * NT;  // tensor-memory columns
  static_assert(kCols <= 512 && (kCols & (kCols - 1)) == 0, "TMEM budget");
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *s_out = smem + S * Sh::kStage;
  uint64_t *bars = reinterpret_cast<uint64_t *>(s_out + Sh::kOut);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(s_out + Sh::kOut + Sh::kBars - 96);
  int *s_warp = reinterpret_cast<int *>(s_out + Sh::kOut + Sh::kBars - 80);  // [warps]
  int4 *s_list = reinterpret_cast<int4 *>(s_out + Sh::kOut + Sh::kBars);      // [kList]
  int *s_first = reinterpret_cast<int *>(s_list + kList);                     // [K + 1]
  const uint32_t bar0 = smem_u32(bars);
  auto FULL = [&](int s) { return bar0 + 8u * s; };
  auto EMPTY = [&](int s) { return bar0 + 8u * (S + s); };
  auto TFULL = [&](int b) { return bar0 + 8u * (2 * S + b); };
  auto TEMPTY = [&](int b) { return bar0 + 8u * (2 * S + 2 + b); };
  const uint32_t DONE = bar0 + 8u * (2 * S + 4);
  static_assert(8 * (2 * S + 5) <= Sh::kBars - 96, "barrier space");
  static_assert(kThreads / 32 * 4 <= 80, "barrier space");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int R = (int)a.plan.R, K = a.plan.K;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) { mbar_init(FULL(i), MODE == kInputs ? 1 : 1 + kGather); mbar_init(EMPTY(i), 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(TFULL(b), 1); mbar_init(TEMPTY(b), kEpiWarps); }
    mbar_init(DONE, 1);
    fence_mbar_init();
    if (MODE != kForward) prefetch_tmap(&tm_a);
    if (MODE != kWeights) prefetch_tmap(&tm_b);
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), kCols);
    tmem_relinquish();
  }
  griddep_wait();
  if (MODE == kWeights) {
    for (int e = threadIdx.x; e <= K; e += kThreads) s_first[e] = a.pieces.slots > 1 ? __ldg(a.pieces.first + e) : e;
  } else {  // tiles of rows of the experts before each
    auto units = [&](int e) {
      int lo, hi;
      expert_rows(a.plan.offsets, e, R, lo, hi);
      return (hi - lo + BM - 1) / BM;
    };
    const int per = (K + kThreads - 1) / kThreads;
    const int e0 = min(K, (int)threadIdx.x * per), e1 = min(K, e0 + per);
    const int most = INT32_MAX / (((MODE == kForward ? a.d_out : a.d_in) + NT - 1) / NT);
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum = add_to(sum, units(e), most);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum = add_to(sum, v, most);
    }
    if (lane == 31) s_warp[warp] = sum;
    int run = __shfl_up_sync(0xffffffffu, sum, 1);
    if (lane == 0) run = 0;
    __syncthreads();
    for (int w = 0; w < warp; ++w) run = add_to(run, s_warp[w], most);
    for (int e = e0; e < e1; ++e) {
      s_first[e] = run;
      run = add_to(run, units(e), most);
    }
    if (threadIdx.x == kThreads - 1) s_first[K] = run;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch();
  const uint32_t tmem = *tmem_slot;
  Tiles<MODE, NT> tiles(a, s_first, s_list);
  if (MODE != kWeights) {
    const int64_t t = blockIdx.x + (int64_t)threadIdx.x * gridDim.x;
    if (threadIdx.x < kList && t < tiles.total) s_list[threadIdx.x] = tiles.find((int)t);
    __syncthreads();
  }

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    int stage = 0;
    uint32_t phase = 0;
    int filled = 0;  // stages ever armed, up to S
    bool ok = true;
    Tile x;
    while (lane == 0 && ok && tiles.next(x)) {
      for (int c = x.c0; c < x.c1; ++c) {
        if (!mbar_wait(EMPTY(stage), phase ^ 1, kErrWaitEmpty)) { ok = false; break; }
        const uint32_t base = smem_u32(smem + stage * Sh::kStage), base_b = base + P * Sh::kA;
        if (MODE == kWeights && x.r0 + (c + 1) * KCH > x.r1) {
          mbar_arrive(FULL(stage));  // the gathering warps fetch an expert's last rows of both operands
        } else {
          mbar_arrive_expect_tx(FULL(stage), P * ((MODE != kForward ? Sh::kA : 0) + (MODE != kWeights ? Sh::kB : 0)));
#pragma unroll
          for (int p = 0; p < P; ++p) {
            if (MODE == kForward) {
              tma_load_3d(base_b + p * Sh::kB, &tm_b, p * a.b_plane + c * KCH, x.n0, x.e, FULL(stage));
            } else if (MODE == kInputs) {
              tma_load_2d(base + p * Sh::kA, &tm_a, p * a.a_plane + c * KCH, x.r0, FULL(stage));
#pragma unroll
              for (int j = 0; j < NT / 64; ++j)
                tma_load_3d(base_b + p * Sh::kB + j * 64 * 128, &tm_b, p * a.b_plane + x.n0 + j * 64, c * KCH, x.e, FULL(stage));
            } else {
#pragma unroll
              for (int j = 0; j < BM / 64; ++j)
                tma_load_2d(base + p * Sh::kA + j * 64 * 128, &tm_a, p * a.a_plane + x.m0 + j * 64, x.r0 + c * KCH, FULL(stage));
            }
          }
        }
        filled = min(S, filled + 1);
        if (++stage == S) { stage = 0; phase ^= 1; }
      }
    }
    // no copy may land after the CTA ends: wait for the last fills of the ring
    if (lane == 0) {
      for (int i = 0; i < filled; ++i) {
        stage = stage == 0 ? S - 1 : stage - 1;
        if (stage == S - 1) phase ^= 1;
        ok = mbar_wait_drain(FULL(stage), phase) && ok;
      }
      if (!ok) report(a.failed);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (lane == 0) {
      // K-major tiles: 8-row groups 1 KB apart, a k-step of 16 elements is 32 bytes.  MN-major tiles: atoms of 64
      // columns 8 KB apart, 8-row groups 1 KB apart, a k-step of 16 rows is 2 KB.
      constexpr bool kAmn = MODE == kWeights, kBmn = MODE != kForward;
      const uint64_t a0 = sdesc_sw128(smem_u32(smem), kAmn ? KCH * 128 : 16, 1024);
      const uint64_t b0 = sdesc_sw128(smem_u32(smem) + P * Sh::kA, kBmn ? KCH * 128 : 16, 1024);
      constexpr uint64_t kStepA = kAmn ? 128 : 2, kStepB = kBmn ? 128 : 2;
      constexpr uint64_t kPlA = Sh::kA >> 4, kPlB = Sh::kB >> 4;
      int stage = 0, seg = 0, count = 0;
      uint32_t phase = 0;
      bool ok = true;
      Tile x;
      for (; ok && tiles.next(x); ++count) {
        const uint32_t low = tmem + (2 + (count & 1)) * NT;  // the smaller products of a float32 tile
        int c = x.c0;
        do {  // a segment: kSeg stages at most
          const int buf = seg & 1;
          if (!mbar_wait(TEMPTY(buf), ((seg >> 1) & 1) ^ 1, kErrWaitTmemEmpty)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d = tmem + buf * NT;
          const int first = c, end = min(x.c1, c + kSeg);
          for (; c < end; ++c) {
            if (!mbar_wait(FULL(stage), phase, kErrWaitFull)) { ok = false; break; }
            if (MODE != kInputs) fence_proxy_async_smem();  // the gathered rows were written through the generic proxy
            tc_fence_after();
            const uint64_t ad = a0 + (uint64_t)((stage * Sh::kStage) >> 4), bd = b0 + (uint64_t)((stage * Sh::kStage) >> 4);
#pragma unroll
            for (int kk = 0; kk < KCH / 16; ++kk) {
              const uint64_t ak = ad + kk * kStepA, bk = bd + kk * kStepB;
              if constexpr (SPLIT) {
                mma_f16(low, ak + 2 * kPlA, bk, a.idesc, (c != x.c0 || kk != 0) ? 1u : 0u);
                mma_f16(low, ak, bk + 2 * kPlB, a.idesc, 1u);
                mma_f16(low, ak + kPlA, bk + kPlB, a.idesc, 1u);
                mma_f16(low, ak + kPlA, bk, a.idesc, 1u);
                mma_f16(low, ak, bk + kPlB, a.idesc, 1u);
              }
              mma_f16(d, ak, bk, a.idesc, (c != first || kk != 0) ? 1u : 0u);
            }
            mma_commit(EMPTY(stage));
            if (++stage == S) { stage = 0; phase ^= 1; }
          }
          if (!ok) break;
          mma_commit(TFULL(buf));
          ++seg;
        } while (c < x.c1);
      }
      mma_commit(DONE);
      ok = mbar_wait_drain(DONE, 0) && ok;
      if (!ok) report(a.failed);
    }
    __syncwarp();
  } else if (warp < 2 + kGather / 32) {
    // ---------------------------------------------------------------- gathered rows
    if (MODE != kInputs) {
      // Eight threads share a 128-byte row of a tile, thread j its 16 bytes, stored at chunk j ^ (row % 8); a thread
      // takes the rows rr, rr + kStep, ...  Its arrival on a stage follows by itself when its copies are complete.
      constexpr int kStep = kGather / 8, kRows = (MODE == kForward ? BM : KCH) / kStep;
      const int j = lane & 7, rr = (threadIdx.x - 64) >> 3;
      const uint32_t at = rr * 128 + ((j ^ (rr & 7)) << 4);
      const uint16_t *matrix = MODE == kForward ? a.a_rows : a.b_rows;
      const int matrix_cols = MODE == kForward ? a.a_cols : a.b_cols;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int id[kRows];  // routes of this thread's rows, -1: none; fetched a tile (Y) or a stage (DW) ahead of their use
      auto routes = [&](int r0, int r1) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) id[i] = r0 + rr + kStep * i < r1 ? ld_now(a.plan.order + r0 + rr + kStep * i) : -1;
      };
      const uint16_t *src[kRows];
      int bytes[kRows];
      auto sources = [&](int col) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const bool in = id[i] >= 0 && id[i] < R;
          const int point = (int)(((uint64_t)(uint32_t)id[i] * a.div_mul) >> a.div_shift);
          src[i] = matrix + (in ? (int64_t)point * matrix_cols + col + j * 8 : 0);
          bytes[i] = in ? 16 : 0;
        }
      };
      Tile x, ahead;
      bool more = tiles.next(ahead);
      auto first_routes = [&] { routes(ahead.r0 + ahead.c0 * KCH, ahead.r1); };
      if (more) first_routes();
      while (more && ok) {
        x = ahead;
        more = tiles.next(ahead);
        if (MODE == kForward) {
          sources(0);
          if (more) first_routes();
        }
        int cols[NT / 64];  // DW: bytes of this thread's 16 in each 64 columns of the tile
#pragma unroll
        for (int n = 0; n < NT / 64; ++n) cols[n] = x.n0 + n * 64 + j * 8 < a.b_plane ? 16 : 0;
        for (int c = x.c0; c < x.c1; ++c) {
          const int r = x.r0 + c * KCH;
          if (MODE == kWeights) {
            sources(x.n0);
            if (c + 1 < x.c1) routes(r + KCH, x.r1);
            else if (more) first_routes();
          }
          ok = __all_sync(0xffffffffu, mbar_wait(EMPTY(stage), phase ^ 1, kErrWaitEmpty));
          if (!ok) break;
          const uint32_t base = smem_u32(smem + stage * Sh::kStage) + at;
          if (MODE == kForward) {
            const bool in = c * KCH + j * 8 < a.a_plane;  // columns behind the last are zeros (and not read)
            // a few rows (a decoding batch) take one copy a thread; with a test on each copy all tiles paid for it
            // (32,768 rows, 1,024 -> 2,048: 156 -> 169 us)
            if (x.rows <= kStep) {
#pragma unroll
              for (int p = 0; p < P; ++p) cp_async16(base + p * Sh::kA, src[0] + p * a.a_plane + c * KCH, in ? bytes[0] : 0);
            } else {
#pragma unroll
              for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < kRows; ++i)
                  cp_async16(base + p * Sh::kA + i * kStep * 128, src[i] + p * a.a_plane + c * KCH, in ? bytes[i] : 0);
            }
          } else {
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
              for (int i = 0; i < kRows; ++i)
#pragma unroll
                for (int n = 0; n < NT / 64; ++n)
                  cp_async16(base + P * Sh::kA + p * Sh::kB + n * KCH * 128 + i * kStep * 128, src[i] + p * a.b_plane + n * 64,
                             bytes[i] & cols[n]);
            if (r + KCH > x.r1) {  // the last rows of A too
#pragma unroll 1
              for (int p = 0; p < P; ++p)
#pragma unroll 1
                for (int i = 0; i < KCH; i += kStep)
#pragma unroll
                  for (int m = 0; m < BM / 64; ++m) {
                    const int row = r + rr + i, col = x.m0 + m * 64 + j * 8;
                    const bool on = row < x.r1 && col < a.a_plane;
                    cp_async16(base + p * Sh::kA + m * KCH * 128 + i * 128,
                               on ? a.a_rows + (int64_t)row * a.a_cols + p * a.a_plane + col : a.a_rows, on ? 16 : 0);
                  }
            }
          }
          cp_async_arrive(FULL(stage));
          if (++stage == S) { stage = 0; phase ^= 1; }
        }
      }
      cp_async_wait_all();
      if (!ok && lane == 0) report(a.failed);
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    constexpr int CW = 128 / sizeof(OUT), EPV = 16 / sizeof(OUT);  // columns of a staging row, of 16 bytes
    constexpr int HC = NT / 2;                                     // columns of this warp
    constexpr int W = SPLIT ? HC : CW;                             // columns held in registers
    static_assert(HC % CW == 0, "whole staging rows");
    const int q = warp & 3, half = (warp - 2 - kGather / 32) / 4 * HC;
    const uint32_t lane_tmem = tmem + ((uint32_t)(q * 32) << 16) + half;
    uint8_t *stg = s_out + (warp - 2 - kGather / 32) * 16 * 128;
    const int width = MODE == kForward ? a.d_out : a.d_in;
    int seg = 0, count = 0;
    bool ok = true;
    // 32 rows x CW columns (from column c0 of the tile) through shared memory, 16 rows at a time, so that the global
    // writes are whole lines
    auto write = [&](const float *v, const Tile &x, int c0) {
      if constexpr (sizeof(OUT) == 4) {
        // fp32: whole 32-byte sectors, a row a lane, past shared memory, whose bandwidth the products take (131,072 rows
        // 128 -> 128: 81 -> 75 us; 16-bit results lose that way, 18 -> 21 us)
        if (a.vec32) {
          const int row = q * 32 + lane;
          if (row < x.rows) {
            OUT *p = out + ((MODE == kWeights ? (int64_t)x.e * a.d_out + x.m0 : x.r0) + row) * width + x.n0 + c0;
#pragma unroll
            for (int j = 0; j < CW; j += 8)
              if (x.n0 + c0 + j < width) st_v8(p + j, v + j);
          }
          return;
        }
      }
      const int64_t row0 = MODE == kWeights ? (int64_t)x.e * a.d_out + x.m0 : x.r0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if ((lane >> 4) == h) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4 *>(stg + (lane & 15) * 128 + ((j ^ (lane & 7)) << 4)) = pack16<OUT>(v + j * EPV);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 4 + (lane >> 3), j = lane & 7;
          const int col = x.n0 + c0 + j * EPV, row = q * 32 + h * 16 + r;
          if (row < x.rows && col < width) {
            const uint4 u = *reinterpret_cast<const uint4 *>(stg + r * 128 + ((j ^ (r & 7)) << 4));
            OUT *p = out + (row0 + row) * width + col;
            if (a.vec) {  // then the width is a multiple of EPV
              *reinterpret_cast<uint4 *>(p) = u;
            } else {
              OUT e[EPV];
              *reinterpret_cast<uint4 *>(e) = u;
#pragma unroll
              for (int k = 0; k < EPV; ++k)
                if (col + k < width) p[k] = e[k];
            }
          }
        }
        __syncwarp();
      }
    };
    if (MODE == kForward) {  // rows of no expert, before the first tile is done
      const int64_t none = min(max(__ldg(a.plan.offsets + K), 0), R), first = none * a.d_out, end = (int64_t)R * a.d_out;
      const int step = a.vec ? 16 / sizeof(OUT) : 1;
      for (int64_t i = first + (int64_t)(blockIdx.x * 32 * kEpiWarps + threadIdx.x - 64 - kGather) * step; i < end; i += (int64_t)gridDim.x * 32 * kEpiWarps * step) {
        if (a.vec) *reinterpret_cast<uint4 *>(out + i) = make_uint4(0u, 0u, 0u, 0u);
        else out[i] = from_f32<OUT>(0.0f);
      }
    }
    // a piece of a tile: fp32, a row a lane
    auto write_piece = [&](const float *v, int n, const Tile &x, int c0) {
      float4 *to = reinterpret_cast<float4 *>(a.pieces.tiles + ((int64_t)x.slot * BM + q * 32 + lane) * NT + c0);
      for (int k = 0; k < n / 4; ++k) to[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    };
    // a segment of a long contraction: a row a lane, 32 columns at a time, added to the segments before in the block's tile of sums
    // and, with the last one, written
    auto add_segment = [&](const Tile &x, uint32_t from, bool first, bool last) {
      const int row = q * 32 + lane;
      float *sum = a.sums + ((int64_t)blockIdx.x * NT + half) * BM + row;
      OUT *to = out + ((MODE == kWeights ? (int64_t)x.e * a.d_out + x.m0 : x.r0) + row) * width + x.n0 + half;
#pragma unroll 1
      for (int i = 0; i < HC; i += 32, from += 32, sum += 32 * BM) {
        float v[32];
        tmem_ld32(from, v);
        tmem_wait_ld();
        if (!first) {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] += sum[k * BM];
        }
        if (!last) {
#pragma unroll
          for (int k = 0; k < 32; ++k) sum[k * BM] = v[k];
        } else if (MODE == kWeights && x.slot >= 0) {
          write_piece(v, 32, x, half + i);
        } else if (row < x.rows && a.vec) {  // (the width is a multiple of EPV)
#pragma unroll
          for (int k = 0; k < 32; k += EPV)
            if (x.n0 + half + i + k < width) *reinterpret_cast<uint4 *>(to + i + k) = pack16<OUT>(v + k);
        } else if (row < x.rows) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (x.n0 + half + i + k < width) to[i + k] = from_f32<OUT>(v[k]);
        }
      }
    };
    Tile x;
    for (; ok && tiles.next(x); ++count) {
      const bool live = q * 32 < x.rows && x.n0 + half < width;
      float acc[W];
      if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] = 0.0f;
      }
      int c = x.c0;
      do {
        const int buf = seg & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(TFULL(buf), (seg >> 1) & 1, kErrWaitTmemFull));
        if (!ok) break;
        tc_fence_after();
        c += kSeg;
        if constexpr (SPLIT) {
          if (live) {
            auto add = [&](uint32_t from, bool smaller) {
#pragma unroll
              for (int i = 0; i < HC / 32; ++i) {
                float v[32];
                tmem_ld32(from + i * 32, v);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const float sum = acc[i * 32 + k] + v[k];
                  acc[i * 32 + k] = smaller && isnan(sum) ? acc[i * 32 + k] : sum;
                }
              }
            };
            add(lane_tmem + buf * NT, false);
            // an infinite operand's products with lower planes (of either sign, or zero) say nothing
            if (c >= x.c1) add(lane_tmem + (2 + (count & 1)) * NT, true);
          }
        } else if (LONG && live && x.c1 - x.c0 > kSeg) {
          add_segment(x, lane_tmem + buf * NT, c - kSeg == x.c0, c >= x.c1);
        } else if (live) {
          for (int i = 0; i < HC / CW; ++i) {
            if (x.n0 + half + i * CW >= width) break;
#pragma unroll
            for (int k = 0; k < CW / 32; ++k) tmem_ld32(lane_tmem + buf * NT + i * CW + k * 32, *reinterpret_cast<float(*)[32]>(acc + k * 32));
            tmem_wait_ld();
            if (MODE == kWeights && x.slot >= 0) write_piece(acc, CW, x, half + i * CW);
            else write(acc, x, half + i * CW);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(TEMPTY(buf));
        if constexpr (SPLIT) {
          if (c >= x.c1 && live) {
            if (MODE == kWeights && x.slot >= 0) {
              write_piece(acc, HC, x, half);
            } else {
#pragma unroll
              for (int i = 0; i < HC / CW; ++i) write(acc + i * CW, x, half + i * CW);
            }
          }
        }
        ++seg;
      } while (c < x.c1);
    }
    if (!ok && lane == 0) report(a.failed);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kCols);
  }
}

// The pieces of DW: one block.
constexpr int kPlanThreads = 512;
__global__ void __launch_bounds__(kPlanThreads) plan_pieces_kernel(RoutePlan p, int most, int limit, int *__restrict__ first, int *__restrict__ slot,
                                                                   int *__restrict__ joined) {
  __shared__ int s_warp[kPlanThreads / 32][3];
  griddep_launch();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int run[3] = {0, 0, 0};
  for (int e0 = 0; e0 <= p.K; e0 += kPlanThreads) {
    const int e = e0 + threadIdx.x;
    const int n = e < p.K ? (expert_stages(p, e) + most - 1) / most : 0;
    const int mine[3] = {n, n > 1 ? n : 0, n > 1};
    int sum[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      sum[q] = min(mine[q], limit);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum[q], o);
        if (lane >= o) sum[q] = add_to(sum[q], v, limit);
      }
      if (lane == 31) s_warp[warp][q] = sum[q];
    }
    __syncthreads();
    int before[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const int prev = __shfl_up_sync(0xffffffffu, sum[q], 1);
      before[q] = add_to(run[q], lane > 0 ? prev : 0, limit);
      for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) before[q] = add_to(before[q], s_warp[w][q], limit);
        run[q] = add_to(run[q], s_warp[w][q], limit);
      }
    }
    if (e <= p.K) {
      first[e] = before[0];
      slot[e] = before[1];
      joined[e] = before[2];
    }
    __syncthreads();
  }
}

// Adds the pieces of the experts that have more than one, in their order: blockIdx.x counts their tiles, a block writes 1024
// results (with 32 rows a block, few had work: 28 -> 58 us for 4 experts of 16,384 rows, 256 x 256).
template <int NT, typename OUT>
__global__ void __launch_bounds__(256) join_pieces_kernel(const __grid_constant__ TcArgs a, OUT *__restrict__ out) {
  griddep_launch();
  griddep_wait();
  const int K = a.plan.K, n_tiles = (a.d_in + NT - 1) / NT, per = (a.d_out + BM - 1) / BM * n_tiles;
  const int u = blockIdx.x / per, tile = blockIdx.x % per;
  if (u >= __ldg(a.pieces.joined + K)) return;
  int lo = 0, hi = K;  // the expert that u experts with pieces to join come before
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.pieces.joined + mid) <= u) lo = mid; else hi = mid;
  }
  const int first = __ldg(a.pieces.slot + lo), n = __ldg(a.pieces.slot + lo + 1) - first;
  {
    const int r = blockIdx.y * (1024 / NT) + threadIdx.x / (NT / 4), c = threadIdx.x % (NT / 4) * 4;
    const int o = tile / n_tiles * BM + r, col = tile % n_tiles * NT + c;
    if (o >= a.d_out || col >= a.d_in) return;
    const float *from = a.pieces.tiles + (int64_t)r * NT + c;
    float f[4] = {};
#pragma unroll 8
    for (int q = 0; q < n; ++q) {
      const int64_t s = min(((int64_t)first + q) * per + tile, (int64_t)a.pieces.slots - 1);
      const float4 v = __ldg(reinterpret_cast<const float4 *>(from + s * BM * NT));
      f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
    }
    OUT *to = out + ((int64_t)lo * a.d_out + o) * a.d_in + col;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (col + k < a.d_in) to[k] = from_f32<OUT>(f[k]);
  }
}

// Rows of `cols` elements to rows of PLANES planes of `colsp` (zeros behind cols): float32 in three bf16
// planes whose sum it is (to 2^-24), 16-bit types as they are.  An infinite value keeps zeros in the lower planes.  One launch
// copies a call's operands.
struct Copies {
  struct {
    const void *src;
    uint16_t *dst;
    int64_t items;  // rows * colsp / 8
    int cols, colsp;
  } job[3];
  int n;
};
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) split_planes_kernel(const __grid_constant__ Copies copies) {
  griddep_wait();
  griddep_launch();
  for (int q = 0; q < copies.n; ++q) {
    const auto &job = copies.job[q];
    const T *__restrict__ src = static_cast<const T *>(job.src);
    uint16_t *__restrict__ dst = job.dst;
    const int cols = job.cols, colsp = job.colsp, per = colsp / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < job.items; i += (int64_t)gridDim.x * 256) {
      const int64_t r = i / per;
      const int c = (int)(i - r * per) * 8;
      const T *p = src + r * cols + c;
      alignas(16) uint16_t h[PLANES][8];
      if constexpr (PLANES == 3) {
        float v[8];
        if (cols % 4 == 0 && c + 8 <= cols) {
          *reinterpret_cast<float4 *>(v) = __ldg(reinterpret_cast<const float4 *>(p));
          *reinterpret_cast<float4 *>(v + 4) = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? to_f32(p[k]) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          __nv_bfloat16 b0 = __float2bfloat16_rn(v[k]);
          if (__hisinf(b0) && !isinf(v[k])) b0 = __ushort_as_bfloat16(v[k] > 0.0f ? 0x7f7f : 0xff7f);  // (rounded past the largest)
          float rest = v[k] - __bfloat162float(b0);
          if (!isfinite(rest)) rest = 0.0f;
          const __nv_bfloat16 b1 = __float2bfloat16_rn(rest);
          const __nv_bfloat16 b2 = __float2bfloat16_rn(rest - __bfloat162float(b1));
          h[0][k] = __bfloat16_as_ushort(b0);
          h[1][k] = __bfloat16_as_ushort(b1);
          h[2][k] = __bfloat16_as_ushort(b2);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) h[0][k] = c + k < cols ? reinterpret_cast<const uint16_t *>(p)[k] : (uint16_t)0;
      }
#pragma unroll
      for (int l = 0; l < PLANES; ++l)
        *reinterpret_cast<uint4 *>(dst + (r * PLANES + l) * colsp + c) = *reinterpret_cast<uint4 *>(h[l]);
    }
  }
}

// A word of pinned host memory for each device, which a product whose wait ran out sets: the next product on that device fails
// with it.  Allocated with the first product (also where that is being captured: nothing of it goes into the graph).
constexpr int kDevices = 16;  // (one cache line, which every call reads)
std::atomic<int *> g_failed{nullptr};
int *failed_words() {
  if (int *words = g_failed.load(std::memory_order_acquire)) return words;
  static std::mutex mutex;
  std::lock_guard<std::mutex> lock(mutex);
  if (int *words = g_failed.load(std::memory_order_acquire)) return words;
  void *p = nullptr;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  const cudaError_t e = cudaHostAlloc(&p, kDevices * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (e != cudaSuccess) return nullptr;
  std::fill(static_cast<int *>(p), static_cast<int *>(p) + kDevices, 0);
  g_failed.store(static_cast<int *>(p), std::memory_order_release);
  return static_cast<int *>(p);
}
// The current device's.
int *failed_word() {
  int dev = 0;
  int *words = cudaGetDevice(&dev) == cudaSuccess ? failed_words() : nullptr;
  return words ? words + dev % kDevices : nullptr;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// A matrix as the kernel reads it: rows of planes * plane 16-bit columns.
struct Operand {
  const void *p;
  int64_t rows;
  int cols;   // columns of a row in memory (all planes)
  int plane;  // columns of a plane
};

// 2-D map with a box of 64 columns x box_rows, or, with depth > 0, a 3-D one of `depth` matrices.
int make_map(CUtensorMap *m, const Operand &o, int bf16, int box_rows, int depth) {
  auto fn = encode_fn();
  if (!fn) return fail(FGMM_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int rank = depth > 0 ? 3 : 2;
  const int64_t rows = depth > 0 ? o.rows / depth : o.rows;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)rows, (cuuint64_t)depth};
  cuuint64_t strides[2] = {(cuuint64_t)o.cols * 2, (cuuint64_t)o.cols * 2 * rows};
  cuuint32_t box[3] = {KCH, (cuuint32_t)box_rows, 1}, estr[3] = {1, 1, 1};
  const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                        const_cast<void *>(o.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(FGMM_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string((int)r));
  return FGMM_OK;
}

bool needs_copy(int dtype, int cols) { return dtype == FGMM_F32 || cols % 8 != 0; }
int plane_cols(int dtype, int cols) { return (int)align_up(cols, dtype == FGMM_F32 ? KCH : 8); }
size_t copy_elems(int dtype, int64_t rows, int cols) {
  return needs_copy(dtype, cols) ? (size_t)rows * plane_cols(dtype, cols) * (dtype == FGMM_F32 ? 3 : 1) : 0;
}

// The operand of `src` [rows][cols], to be copied into `dst` where TMA cannot read it as it is.
Operand operand(const void *src, int dtype, int64_t rows, int cols, uint16_t *dst, Copies &copies) {
  if (!needs_copy(dtype, cols)) return {src, rows, cols, cols};
  const int colsp = plane_cols(dtype, cols);
  copies.job[copies.n++] = {src, dst, rows * (colsp / 8), cols, colsp};
  return {dst, rows, colsp * (dtype == FGMM_F32 ? 3 : 1), colsp};
}

int run_copies(const Copies &copies, int dtype, cudaStream_t st) {
  int64_t most = 0;
  for (int i = 0; i < copies.n; ++i) most = std::max(most, copies.job[i].items);
  if (most == 0) return FGMM_OK;
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(most, 256), 8 * num_sms());
  FGMM_CUDA_TRY(launch_pdl(dtype == FGMM_F32 ? split_planes_kernel<float, 3> : split_planes_kernel<__half, 1>, dim3(grid), dim3(256), 0, st, copies));
  return FGMM_OK;
}

// The pieces' division: none where every SM has three whole tiles (with pieces, their plan and their join 512 tiles of up to 16
// stages took 100 us instead of 60); else an SM's share of the stages at most, of float32's heavier ones (192 KB and 24
// products against 48 KB and 4, for a piece of 64 KB against 128 KB) a third of it, and four at least.  (With a third
// for all, 8 experts of 4,096 routes, 1,024 x 1,024 bf16, took 52 us instead of 28.)  A slot count that holds those of every routing:
// an expert of n > most >= 4 stages has at most 2 n / most pieces, and n is at most 5 / 4 of its rows / KCH.
struct PieceSizes {
  int64_t per, most, slots;
};
PieceSizes piece_sizes(int dtype, int64_t R, int K, int d_in, int d_out, int NT) {
  PieceSizes z;
  z.per = cdiv(d_out, BM) * cdiv(d_in, NT);
  z.most = K * z.per >= 3 * num_sms() ? INT32_MAX / 2 : std::max<int64_t>(4, cdiv((cdiv(R, KCH) + K) * z.per, (dtype == FGMM_F32 ? 3 : 1) * num_sms()));
  z.slots = cdiv(R, KCH) <= z.most ? 1 : (cdiv(5 * cdiv(R, KCH), 2 * z.most) + 1) * z.per;
  return z;
}
// Columns of a tile of DW.
int weights_tile(int dtype, int d_in) { return dtype == FGMM_F32 || d_in <= 128 ? 128 : 256; }

template <int MODE, int NT, bool SPLIT, bool LONG, typename OUT>
int launch(const Operand &oa, const Operand &ob, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, OUT *out,
           void *pieces, float *sums, cudaStream_t st) {
  using Sh = Shape<NT, SPLIT>;
  const int bf16 = dtype != FGMM_F16, width = MODE == kForward ? d_out : d_in;
  CUtensorMap ma{}, mb{};
  int rc = FGMM_OK;
  if (MODE != kForward) rc = make_map(&ma, oa, bf16, MODE == kInputs ? BM : KCH, 0);
  if (!rc && MODE != kWeights) rc = make_map(&mb, ob, bf16, MODE == kForward ? NT : KCH, p.K);
  if (rc) return rc;
  TcArgs a{};
  a.plan = p;
  a.d_in = d_in;
  a.d_out = d_out;
  a.a_plane = oa.plane;
  a.b_plane = ob.plane;
  a.a_rows = static_cast<const uint16_t *>(oa.p);
  a.b_rows = static_cast<const uint16_t *>(ob.p);
  a.a_cols = oa.cols;
  a.b_cols = ob.cols;
  // exact for n < 2^31: with 2^(l - 1) < top_k <= 2^l the multiplier exceeds 2^(31 + l) / top_k by less than 1
  a.div_shift = 31;
  while ((1u << (a.div_shift - 31)) < (uint32_t)p.top_k) ++a.div_shift;
  a.div_mul = (uint32_t)((((uint64_t)1 << a.div_shift) + p.top_k - 1) / p.top_k);
  a.idesc = idesc_f16(BM, NT, MODE == kWeights, MODE != kForward, bf16);
  a.vec32 = (width * sizeof(OUT)) % 32 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0;
  a.vec = (width * sizeof(OUT)) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  a.sums = sums;
  auto kernel = experts_tc_kernel<MODE, NT, SPLIT, LONG, OUT>;
  static std::atomic<bool> done[64];  // per device
  int dev = 0;
  FGMM_CUDA_TRY(cudaGetDevice(&dev));
  a.failed = failed_words();
  if (!a.failed) return fail(FGMM_ERR_CUDA, "no pinned memory for the products' error words");
  a.failed += dev % kDevices;
  if (dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
    FGMM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::smem(kMaxExperts)));
    if (dev < 64) done[dev].store(true, std::memory_order_release);
  }
  if (MODE == kWeights) {
    const PieceSizes z = piece_sizes(dtype, p.R, p.K, d_in, d_out, NT);
    if ((cdiv(p.R, KCH) + p.K) * z.per > INT32_MAX) return fail(FGMM_ERR_UNSUPPORTED, "more than 2^31 stages of the weights' gradient");
    Carve c(pieces);
    int *first = c.take<int>(p.K + 1), *slot = c.take<int>(p.K + 1), *joined = c.take<int>(p.K + 1);
    a.pieces = {first, slot, joined, c.take<float>(z.slots * BM * NT), (int)z.most, (int)z.slots};
    if (z.slots > 1)
      FGMM_CUDA_TRY(launch_pdl(plan_pieces_kernel, dim3(1), dim3(kPlanThreads), 0, st, p, (int)z.most, (int)(INT32_MAX / z.per), first, slot, joined));
    FGMM_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(num_sms(), (cdiv(p.R, KCH * z.most) + p.K) * z.per)), dim3(kThreads),
                             Sh::smem(p.K), st, ma, mb, a, out));
    if (z.slots > 1)
      FGMM_CUDA_TRY(launch_pdl(join_pieces_kernel<NT, OUT>, dim3((unsigned)(z.slots / 2), BM * NT / 1024), dim3(256), 0, st, a, out));
    return FGMM_OK;
  }
  const int64_t tiles = (cdiv(p.R, BM) + std::min<int64_t>(p.K, p.R)) * cdiv(width, NT);  // at most
  if (tiles > INT32_MAX) return fail(FGMM_ERR_UNSUPPORTED, "more than 2^31 tiles");
  FGMM_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)std::min<int64_t>(tiles, num_sms())), dim3(kThreads), Sh::smem(p.K), st, ma, mb, a, out));
  return FGMM_OK;
}

// Columns of a tile of Y or DX.  A stage's products are bound by shared memory: 64 KB written and read for 128 columns, 96 KB for
// 256, so the wider tile takes one and a half times as long and holds twice as much; it is taken where the SMs' rounds of such
// tiles cost less.  (Every expert's last tile counts as half a tile more.)
bool wide_tiles(int64_t R, int K, int width) {
  if (width <= 128) return false;
  const int64_t m = cdiv(R, BM) + std::min<int64_t>(K, R) / 2;
  return 3 * cdiv(m * cdiv(width, 256), num_sms()) <= 2 * cdiv(m * cdiv(width, 128), num_sms());
}
template <int MODE, typename OUT>
int launch16(const Operand &oa, const Operand &ob, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, OUT *out,
             void *pieces, float *sums, cudaStream_t st) {
  const int width = MODE == kForward ? d_out : d_in;
  constexpr bool kRows = MODE == kWeights;  // any of the experts may have a long contraction
  if (!kRows && (MODE == kForward ? d_in : d_out) > kLong * KCH)
    return launch<MODE, 256, false, true>(oa, ob, dtype, N, d_in, d_out, p, out, pieces, sums, st);
  if (kRows ? weights_tile(dtype, d_in) == 256 : wide_tiles(p.R, p.K, width))
    return launch<MODE, 256, false, kRows>(oa, ob, dtype, N, d_in, d_out, p, out, pieces, sums, st);
  return launch<MODE, 128, false, kRows>(oa, ob, dtype, N, d_in, d_out, p, out, pieces, sums, st);
}

size_t piece_bytes(int dtype, int64_t R, int K, int d_in, int d_out) {
  const int NT = weights_tile(dtype, d_in);
  Carve c(nullptr);
  for (int i = 0; i < 3; ++i) c.take<int>(K + 1);
  c.take<float>(piece_sizes(dtype, R, K, d_in, d_out, NT).slots * BM * NT);
  return c.bytes();
}

}  // namespace

int experts_device_error(bool reset) {
  const int code = read_dev_error(reset);
  volatile int *word = failed_word();
  const int told = word ? *word : 0;
  if (reset && word) *word = 0;
  return code ? code : told;
}

int *experts_error_word() { return failed_word(); }

// Takes an earlier product's failure.  The device's word is cleared in the stream's order, so that later waits do not give up
// for it; a capture leaves both words as they are.
int take_failure(cudaStream_t st) {
  const volatile int *words = g_failed.load(std::memory_order_acquire);
  int any = 0;
  for (int i = 0; words && i < kDevices; ++i) any |= words[i];
  if (any == 0) return FGMM_OK;  // (asking for the current device would cost a small call more)
  volatile int *word = failed_word();
  const int code = word ? *word : 0;
  if (code == 0) return FGMM_OK;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &status) != cudaSuccess) {
    cudaGetLastError();
    status = cudaStreamCaptureStatusActive;
  }
  if (status == cudaStreamCaptureStatusNone) {
    static const int zero = 0;
    *word = 0;
    FGMM_CUDA_TRY(cudaMemcpyToSymbolAsync(g_dev_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st));
  }
  return fail(FGMM_ERR_CUDA, "an earlier expert product on this device gave up a bounded wait (code " + std::to_string(code) +
                                 "): its results are incomplete");
}

namespace {
// The workspace: copies of the operands that TMA cannot read, DW's pieces, and the blocks' tiles of long 16-bit contractions.
struct TcSpace {
  uint16_t *x, *weight, *dy;
  char *pieces;
  float *sums;
  size_t bytes;
};
TcSpace tc_space(void *ws, int dtype, int64_t N, int K, int d_in, int d_out, int top_k, const TcParts &parts) {
  Carve c(ws);
  TcSpace s;
  s.x = c.take<uint16_t>(parts.forward || parts.weights ? copy_elems(dtype, N, d_in) : 0);
  s.weight = c.take<uint16_t>(parts.forward || parts.inputs ? copy_elems(dtype, (int64_t)K * d_out, d_in) : 0);
  s.dy = c.take<uint16_t>(parts.inputs || parts.weights ? copy_elems(dtype, N * top_k, d_out) : 0);
  s.pieces = c.take<char>(parts.weights ? piece_bytes(dtype, N * top_k, K, d_in, d_out) : 0);
  const int64_t longest = std::max<int64_t>({parts.forward ? d_in : 0, parts.inputs ? d_out : 0, parts.weights ? N * top_k : 0});
  s.sums = c.take<float>(dtype != FGMM_F32 && longest > kLong * KCH ? (size_t)num_sms() * BM * 256 : 0);
  s.bytes = c.bytes() + 256;
  return s;
}
}  // namespace

size_t products_tc_workspace(int dtype, int64_t N, int K, int d_in, int d_out, int top_k, const TcParts &parts) {
  return tc_space(nullptr, dtype, N, K, d_in, d_out, top_k, parts).bytes;
}

int products_tc(const void *x, const void *weight, int dtype, int64_t N, int d_in, int d_out, const RoutePlan &p, void *y,
                void *ws, cudaStream_t st) {
  const TcSpace s = tc_space(ws, dtype, N, p.K, d_in, d_out, p.top_k, {true, false, false});
  Copies copies{};
  const Operand ox = operand(x, dtype, N, d_in, s.x, copies), ow = operand(weight, dtype, (int64_t)p.K * d_out, d_in, s.weight, copies);
  int rc = run_copies(copies, dtype, st);
  if (rc) return rc;
  if (dtype == FGMM_F32) return launch<kForward, 128, true, false>(ox, ow, dtype, N, d_in, d_out, p, (float *)y, nullptr, nullptr, st);
  if (dtype == FGMM_BF16) return launch16<kForward>(ox, ow, dtype, N, d_in, d_out, p, (__nv_bfloat16 *)y, nullptr, s.sums, st);
  return launch16<kForward>(ox, ow, dtype, N, d_in, d_out, p, (__half *)y, nullptr, s.sums, st);
}

int products_tc_backward(const void *dy, const void *x, const void *weight, int dtype, int64_t N, int d_in, int d_out,
                         const RoutePlan &p, float *dx_rows, void *d_weight, const TcParts &parts, void *ws, cudaStream_t st) {
  const TcSpace s = tc_space(ws, dtype, N, p.K, d_in, d_out, p.top_k, parts);
  Copies copies{};
  const Operand og = operand(dy, dtype, p.R, d_out, s.dy, copies);
  const Operand ow = parts.inputs ? operand(weight, dtype, (int64_t)p.K * d_out, d_in, s.weight, copies) : Operand{};
  const Operand ox = parts.weights ? operand(x, dtype, N, d_in, s.x, copies) : Operand{};
  int rc = run_copies(copies, dtype, st);
  if (rc) return rc;
  if (parts.inputs) {
    rc = dtype == FGMM_F32 ? launch<kInputs, 128, true, false>(og, ow, dtype, N, d_in, d_out, p, dx_rows, nullptr, nullptr, st)
                           : launch16<kInputs>(og, ow, dtype, N, d_in, d_out, p, dx_rows, nullptr, s.sums, st);
    if (rc) return rc;
  }
  if (!parts.weights) return FGMM_OK;
  if (dtype == FGMM_F32) return launch<kWeights, 128, true, false>(og, ox, dtype, N, d_in, d_out, p, (float *)d_weight, s.pieces, nullptr, st);
  if (dtype == FGMM_BF16) return launch16<kWeights>(og, ox, dtype, N, d_in, d_out, p, (__nv_bfloat16 *)d_weight, s.pieces, s.sums, st);
  return launch16<kWeights>(og, ox, dtype, N, d_in, d_out, p, (__half *)d_weight, s.pieces, s.sums, st);
}

}  // namespace fgmm
