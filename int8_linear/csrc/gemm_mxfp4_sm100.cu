// The product of two MXFP4 operands for sm_100a:
//     out[m,n] = cast( sum_k A[m,k] * W[n,k] + bias[n] )
// with A and W in 4 bits (mxfp4.cuh), multiplied by tcgen05.mma.kind::mxf4, which applies
// both operands' block scales and accumulates in float32 in TMEM.
//
// Split tiles (mx_split_kernel), for batches of up to a few hundred tokens: the weight is
// the MMA's 128-row side and TN tokens its other side; the CTAs of a thread-block cluster
// share one tile's K, one tile per cluster.  Streaming the weight from HBM bounds these
// shapes, so the split exists to have more SMs loading; clusters double in size, so that tiles
// between half and all of the SMs leave the rest of them idle (96 of 148 load at N = 12288).
// Each CTA leaves its float32
// partial tile in its own shared memory; after a cluster barrier each CTA adds, for its
// share of the outputs, every CTA's partial in rank order through distributed shared
// memory.  So a shape's result does not vary from run to run.
//
// Pair tiles (mx_pair_kernel), for larger batches, bound by the tensor cores: two CTAs on
// two SMs compute tiles of 256 tokens x 256 weight rows with cta_group::2 MMAs, each loading
// half of both operands' rows, so an SM fills 32 KB per 256 values of K where one CTA alone
// would need 48.  Scales: each CTA holds its own tokens' and, since it computes every column
// of its 128 rows, the whole weight tile's.  TMEM's 512 columns do not hold two accumulators
// of 256 and the scales, so every other tile has 192 weight rows: 256 + 192 columns of
// accumulators leave 64 for the scales, and one tile's epilogue runs beside the next tile's
// MMAs.  4096 x 12288 x 2048 takes 48 to 50 us (4.2 PFLOP/s; 5.8 at K = 8192).  Two things bound
// it.  The outputs: with K = 256 the product still takes 29 us, for 100 MB that the copy rate
// would write in 15.  And the operands' way from L2: every further 1024 of K takes 11 to 13 us
// up to K = 2048 and 15 from 4096 on, 7 PFLOP/s, where the same MMAs with the loads left out ran at
// 8.3.  The outputs' part is hidden behind the operands' only in part until that is the longer
// one.  Other tilings measured: 256 x 256 with two
// accumulators sharing 32 columns 53 us (each tile waits for the last one's shared columns),
// 256 x 192 throughout 53 us (a 256-row MMA takes the same time for 192 and 256 columns).
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "epilogue.cuh"
#include "internal.h"
#include "mxfp4.cuh"
#include "tmap.h"

namespace i8l {

constexpr int kMxRowBytes = 128;               // K bytes per stage: one swizzle row, 256 values
constexpr int kMxStageK = 2 * kMxRowBytes;     // values of K per stage
constexpr int kMxRows = 128;                   // MMA M: one CTA's rows of the first operand
constexpr int kSfStageBytes = 2 * kSfTileBytes;  // scales of 128 rows and one stage of K
constexpr int kSfWords = kSfTileBytes / 4;     // 32-bit words of a scale tile along its map's x

struct MxGemmArgs {
  int M, N, K;
  int kblocks;          // stages of K in all
  int tiles_n, tiles_m;
  int cluster;
  int stages;
  const void *bias;
  int bias_dtype;
  void *out;
  int out_dtype;
  long long ldc;
  int vec_store;        // four consecutive outputs of a row may be stored at once
  int early;            // see mx_weight_early
  int tma_out;          // pair tiles: outputs leave through shared memory by TMA stores
  FastDiv per_col;      // pair tiles: token tiles (a division per tile and role took 500 cycles)
  int *status;
};

// ------------------------------------------------------------------ split tiles

constexpr int kSplitThreads = 256;  // two warps for each quarter of the TMEM lanes
constexpr int kMaxCluster = 8;

template <int TN>
struct SplitLayout {
  static constexpr int kXBytes = kMxRows * kMxRowBytes;
  static constexpr int kYBytes = TN * kMxRowBytes;
  static constexpr int kStageBytes = kXBytes + kYBytes + 2 * kSfStageBytes;
  static constexpr int kSfCols = 16;  // TMEM columns of one stage's scales: 2 operands x 2 tiles x 4
  static constexpr int kTmemCols = TN + kSfCols <= 32 ? 32 : TN + kSfCols <= 64 ? 64 : TN + kSfCols <= 128 ? 128 : 256;
  static constexpr int kRedBytes = TN * kMxRows * 4;  // float32 partial tile, in the idle ring
  static constexpr size_t bytes(int stages) {
    const int ring = stages * kStageBytes;
    return 1024 /* alignment slack */ + (ring > kRedBytes ? ring : kRedBytes) + (2 * stages + 2) * 8 + 16;
  }
};

__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Units u0..u1-1 (four floats each) of the partial tiles at `red` in every CTA of a cluster of
// at most C, added in rank order and handed to finish(unit, sum).  A read of another CTA's
// shared memory takes some 700 cycles, so those of kAhead units and all CTAs are on their way
// together.
template <int C, int kAhead, typename Finish>
__device__ __forceinline__ void add_partials(uint32_t red, int u0, int u1, int cluster, Finish finish) {
  for (int u = u0 + static_cast<int>(threadIdx.x); u < u1; u += kAhead * kSplitThreads) {
    float4 f[kAhead][C];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int p = 0; p < C; ++p)
        if (p < cluster && u + i * kSplitThreads < u1)
          f[i][p] = ld_cluster_v4(map_to_rank(red + (u + i * kSplitThreads) * 16, static_cast<uint32_t>(p)));
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (u + i * kSplitThreads >= u1) break;
      float4 sum = f[i][0];
#pragma unroll
      for (int p = 1; p < C; ++p)
        if (p < cluster) {
          sum.x += f[i][p].x;
          sum.y += f[i][p].y;
          sum.z += f[i][p].z;
          sum.w += f[i][p].w;
        }
      finish(u + i * kSplitThreads, sum);
    }
  }
}

// Stores outputs n0..n0+3 of token row m.
__device__ __forceinline__ void store_out4(const MxGemmArgs &a, int m, int n0, const float (&v)[4]) {
  const long long at = static_cast<long long>(m) * a.ldc + n0;
  if (a.out_dtype == I8L_F32) {
    float *o = static_cast<float *>(a.out) + at;
    if (a.vec_store && n0 + 4 <= a.N) {
      *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < a.N) o[j] = v[j];
    }
  } else {
    uint16_t *o = static_cast<uint16_t *>(a.out) + at;
    const uint32_t p0 = pack16x2(a.out_dtype, v[0], v[1]), p1 = pack16x2(a.out_dtype, v[2], v[3]);
    if (a.vec_store && n0 + 4 <= a.N) {
      *reinterpret_cast<uint2 *>(o) = make_uint2(p0, p1);
    } else {
      const uint32_t b[4] = {p0 & 0xffffu, p0 >> 16, p1 & 0xffffu, p1 >> 16};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j < a.N) o[j] = static_cast<uint16_t>(b[j]);
    }
  }
}

template <int TN>
__global__ void __launch_bounds__(kSplitThreads)
    mx_split_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                    const __grid_constant__ CUtensorMap map_sfx, const __grid_constant__ CUtensorMap map_sfy,
                    const MxGemmArgs a) {
  using L = SplitLayout<TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int S = a.stages;
  uint8_t *sx = smem, *sy = sx + S * L::kXBytes, *ssx = sy + S * L::kYBytes, *ssy = ssx + S * kSfStageBytes;
  float *red = reinterpret_cast<float *>(smem);
  const int ring = S * L::kStageBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + (ring > L::kRedBytes ? ring : L::kRedBytes));
  uint64_t *empty = full + S, *done = empty + S, *drain = done + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0), lane = threadIdx.x % 32;
  const int rank = a.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / a.cluster;
  const int tx = tile % a.tiles_n, ty = tile / a.tiles_n;
  const int kb0 = a.kblocks * rank / a.cluster, kb1 = a.kblocks * (rank + 1) / a.cluster;

  const uint64_t pol_w = policy_evict_first(), pol_a = policy_evict_last();
  const int pre = a.early ? min(S, kb1 - kb0) : 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    // The weight tiles of the first stages wait neither for the other warps nor for the
    // previous kernel.
    for (int i = 0; i < pre; ++i) {
      mbar_arrive_expect_tx(&full[i], L::kStageBytes);
      tma_load_2d(sx + i * L::kXBytes, &map_x, &full[i], (kb0 + i) * kMxRowBytes, tx * kMxRows, pol_w);
      tma_load_2d(ssx + i * kSfStageBytes, &map_sfx, &full[i], (kb0 + i) * 2 * kSfWords, tx, pol_w);
    }
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_launch_dependents();

  if (warp == 0) {
    // The whole warp runs the producer's loop, one elected lane issues (see elect_one).
    const uint32_t elected = elect_one();
    const uint32_t x0 = smem_u32(sx), y0 = smem_u32(sy), sfx0 = smem_u32(ssx), sfy0 = smem_u32(ssy),
                   full0 = smem_u32(full);
    pdl_wait();
    bool ok = true;
    int issued = 0, st = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (issued >= pre) {
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[st], phase ^ 1u, abort_flag, a.status, kStatusProducerWait));
        if (!ok) break;
        mbar_expect_tx_elected(elected, full0 + 8 * st, L::kStageBytes);
        tma_load_2d_elected(elected, x0 + st * L::kXBytes, &map_x, full0 + 8 * st, kb * kMxRowBytes, tx * kMxRows, pol_w);
        tma_load_2d_elected(elected, sfx0 + st * kSfStageBytes, &map_sfx, full0 + 8 * st, kb * 2 * kSfWords, tx, pol_w);
      }
      tma_load_2d_elected(elected, y0 + st * L::kYBytes, &map_y, full0 + 8 * st, kb * kMxRowBytes, ty * TN, pol_a);
      tma_load_2d_elected(elected, sfy0 + st * kSfStageBytes, &map_sfy, full0 + 8 * st, kb * 2 * kSfWords,
                          ty * TN / kMxRows, pol_a);
      ++issued;
      if (++st == S) {
        st = 0;
        phase ^= 1u;
      }
    }
    if (!ok) {
      // Let the loads already issued land before the CTA's shared memory goes away.
      for (int i = 0; i < min(issued, S); ++i) {
        if (--st < 0) {
          st = S - 1;
          phase ^= 1u;
        }
        volatile int no_abort = 0;
        mbar_wait_bounded(&full[st], phase, &no_abort, a.status, kStatusDrainWait);
      }
    }
  } else if (warp == 1) {
    const uint32_t elected = elect_one();
    const uint32_t x_lo = desc_lo(smem_u32(sx)), y_lo = desc_lo(smem_u32(sy)), sfx_lo = desc_lo(smem_u32(ssx)),
                   sfy_lo = desc_lo(smem_u32(ssy));
    bool ok = true, any = false;
    int st = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[st], phase, abort_flag, a.status, kStatusMmaWait));
      if (!ok) break;
      tc_fence_after();
      const uint32_t al = x_lo + st * (L::kXBytes >> 4), bl = y_lo + st * (L::kYBytes >> 4),
                     xl = sfx_lo + st * (kSfStageBytes >> 4), yl = sfy_lo + st * (kSfStageBytes >> 4);
      const int left = a.K - kb * kMxStageK;  // steps of 64 values past K are left out
      constexpr uint32_t kId0 = idesc_mxf4(kMxRows, TN, 0), kId2 = idesc_mxf4(kMxRows, TN, 2);
      single_half_stage(elected, tmem, al, bl, xl, yl, tmem + TN, tmem + TN + 8, kId0, kId2, any ? 1u : 0u, left > 64);
      if (left > 128)
        single_half_stage(elected, tmem, al + 4, bl + 4, xl + (kSfTileBytes >> 4), yl + (kSfTileBytes >> 4),
                          tmem + TN + 4, tmem + TN + 12, kId0, kId2, 1u, left > 192);
      any = true;
      mma_commit_elected<false>(elected, smem_u32(&empty[st]));
      if (++st == S) {
        st = 0;
        phase ^= 1u;
      }
    }
    if (ok) {
      mma_commit_elected<false>(elected, smem_u32(done));
    } else if (any) {
      mma_commit_elected<false>(elected, smem_u32(drain));
      volatile int no_abort = 0;
      mbar_wait_bounded(drain, 0, &no_abort, a.status, kStatusDrainWait);
    }
  }
  __syncwarp();
  pdl_wait();  // this thread's outputs and bias follow the stream's order
  // The four weight rows of this thread's outputs, the same in all of them (the strides between
  // a thread's units are multiples of a token's): their bias is on its way before the MMAs end
  // (333 x 6144 x 4096 with bias 12.5 us with a load per output, 9.9 so).
  const int live = min(TN, a.M - ty * TN);       // tokens of this tile
  const int units = live * (kMxRows / 4);        // four consecutive outputs each
  const int u0 = units * rank / a.cluster, u1 = units * (rank + 1) / a.cluster;
  const int n0 = tx * kMxRows + (u0 + static_cast<int>(threadIdx.x)) % (kMxRows / 4) * 4;
  float bias[4] = {};
  if (a.bias)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n0 + j < a.N) bias[j] = load_scalar_f(a.bias, a.bias_dtype, n0 + j);
  const bool ok = mbar_wait_bounded(done, 0, abort_flag, a.status, kStatusEpilogueWait);
  tc_fence_after();
  // Every MMA has read its operands: the ring holds the partial tile now, [token][128 n].
  if (__syncthreads_and(ok)) {
    const uint32_t taddr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    for (int c = (warp >> 2) * 16; c < live; c += 32) {
      uint32_t r[16];
      tmem_ld16(taddr + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) red[(c + j) * kMxRows + (warp & 3) * 32 + lane] = __uint_as_float(r[j]);
    }
  }
  tc_fence_before();
  if (a.cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  if (*abort_flag == 0) {
    auto finish = [&](int u, float4 f) {
      if (n0 >= a.N) return;
      float v[4] = {f.x, f.y, f.z, f.w};
      if (a.bias)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += bias[j];
      store_out4(a, ty * TN + u / (kMxRows / 4), n0, v);
    };
    if (a.cluster == 1) {
#pragma unroll 4
      for (int u = u0 + static_cast<int>(threadIdx.x); u < u1; u += kSplitThreads)
        finish(u, reinterpret_cast<const float4 *>(red)[u]);
    } else if (a.cluster <= 4) {
      add_partials<4, 4>(smem_u32(red), u0, u1, a.cluster, finish);
    } else {
      add_partials<kMaxCluster, 2>(smem_u32(red), u0, u1, a.cluster, finish);
    }
  }
  // No CTA leaves while another may still read its partial sums.
  if (a.cluster > 1) cluster_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

// ------------------------------------------------------------------ pair tiles

constexpr int kPairEpi = 8;        // epilogue warps: two for each quarter of the TMEM lanes
constexpr int kPairThreads = 64 + 32 * kPairEpi;  // and the producer and the MMA issuer
constexpr int kPairBufBytes = 4096;  // an epilogue warp's staging: 32 rows of 128 bytes
constexpr int kPairStaging = kPairEpi * kPairBufBytes;

// Weight rows of the two kinds of tile; each CTA holds half of a tile's rows.  Along N they
// take turns: 256 rows, 192, 256, ...  Both are multiples of 64, so that a tile's scales begin
// at an even TMEM column: the MMA's scale address takes no odd one.
constexpr int kWide = 256, kNarrow = 192, kBoth = kWide + kNarrow;
constexpr int kPairSfGroups = 3;  // 128-row scale groups that a tile's rows can lie in
constexpr int kPairXBytes = kMxRows * kMxRowBytes;
constexpr int kPairYBytes = kWide / 2 * kMxRowBytes;
constexpr int kPairStageBytes = kPairXBytes + kPairYBytes + (1 + kPairSfGroups) * kSfStageBytes;
// TMEM columns: a wide tile's accumulator, a narrow one's, then the scales of one stage: 8
// columns for the tokens' 128 rows, 12 and 12 for the weight's three groups.
constexpr int kPairSf = kBoth;

constexpr size_t pair_smem(int stages) {
  return 1024 /* alignment slack */ + static_cast<size_t>(stages) * kPairStageBytes + kPairStaging +
         static_cast<size_t>(2 * stages + 5) * 8 + 16;
}

// The tiles of one pair of CTAs: wide and narrow ones by turns while both last.  Pair p takes
// every `pairs`-th wide tile from p on and every `pairs`-th narrow one from pairs - 1 - p on,
// so that a pair with one wide tile more than others has no narrow one more too.
struct PairWalk {
  int wide, narrow;  // the next tile of each kind
  int step, turn;

  __device__ __forceinline__ PairWalk() {
    step = static_cast<int>(gridDim.x >> 1);
    wide = static_cast<int>(blockIdx.x >> 1);
    narrow = step - 1 - wide;
    turn = 0;
  }

  // The next tile's kind (0 wide, 1 narrow), token tile and first weight row; false at the end.
  __device__ __forceinline__ bool next(const MxGemmArgs &a, int &kind, int &tm, int &n0) {
    const int wide_cols = (a.N + kBoth - 1) / kBoth, narrow_cols = (a.N + kBoth - 1 - kWide) / kBoth;
    const bool more_wide = wide < a.tiles_m * wide_cols, more_narrow = narrow < a.tiles_m * narrow_cols;
    if (!more_wide && !more_narrow) return false;
    kind = (turn && more_narrow) || !more_wide ? 1 : 0;
    turn = kind ^ 1;
    const int t = kind ? narrow : wide;
    if (kind)
      narrow += step;
    else
      wide += step;
    // All token tiles of one weight tile, then the next: the pairs running at one time share
    // weight tiles in L2 (walking 4 or 8 token tiles at a time measured the same).
    const int col = static_cast<int>(a.per_col.div(static_cast<uint32_t>(t)));
    tm = t - col * a.tiles_m;
    n0 = col * kBoth + (kind ? kWide : 0);
    return true;
  }
};

// 32 lanes x 32 consecutive columns.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// 64 columns from n0 on of a warp's 32 token rows (the first is m0): bias, rounding and the
// stores, through the warp's staging buffer (rows of 128 bytes in the 128-byte swizzle), by a
// TMA store (two for float32) or, where TMA cannot address the output, by the lanes.  bias:
// lane i holds those of columns i and 32 + i.
template <int DT>
__device__ __forceinline__ void pair_emit(const MxGemmArgs &a, const CUtensorMap *map_out, int m0, int n0, int lane,
                                          const float (&bias)[2], const uint32_t (&r)[2][32], uint8_t *staging) {
  float v[64];
#pragma unroll
  for (int j = 0; j < 64; ++j) v[j] = __uint_as_float(r[j / 32][j % 32]);
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < 64; ++j) v[j] += __shfl_sync(0xffffffffu, bias[j / 32], j % 32);
  }
  constexpr int kBoxes = DT == I8L_F32 ? 2 : 1, kCols = 64 / kBoxes;
#pragma unroll
  for (int h = 0; h < kBoxes; ++h) {
    if (a.tma_out && lane == 0) bulk_wait_read<0>();  // the last store has read the buffer
    __syncwarp();
    uint8_t *rowp = staging + lane * 128;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint4 w;
      if constexpr (DT == I8L_F32)
        w = make_uint4(__float_as_uint(v[32 * h + 4 * c]), __float_as_uint(v[32 * h + 4 * c + 1]),
                       __float_as_uint(v[32 * h + 4 * c + 2]), __float_as_uint(v[32 * h + 4 * c + 3]));
      else
        w = make_uint4(pack16x2(DT, v[8 * c], v[8 * c + 1]), pack16x2(DT, v[8 * c + 2], v[8 * c + 3]),
                       pack16x2(DT, v[8 * c + 4], v[8 * c + 5]), pack16x2(DT, v[8 * c + 6], v[8 * c + 7]));
      *reinterpret_cast<uint4 *>(rowp + ((c ^ (lane & 7)) << 4)) = w;
    }
    if (a.tma_out) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (n0 + kCols * h < a.N && m0 < a.M) tma_store_2d(map_out, staging, n0 + kCols * h, m0);
        bulk_commit();
      }
    } else {
      // Row after row, neighbouring columns by neighbouring lanes: the rows of such an output
      // begin anywhere (4096 x 4099 x 2048 29.6 us; a row by each lane, from registers, 166).
      __syncwarp();
      using E = std::conditional_t<DT == I8L_F32, uint32_t, uint16_t>;
      const int rows = min(32, a.M - m0);
#pragma unroll 8
      for (int row = 0; row < rows; ++row) {
        E *o = static_cast<E *>(a.out) + static_cast<long long>(m0 + row) * a.ldc + n0 + kCols * h;
#pragma unroll
        for (int j = 0; j < kCols; j += 32) {
          const int at = (j + lane) * static_cast<int>(sizeof(E));
          const E e = *reinterpret_cast<const E *>(staging + row * 128 + ((((at >> 4) ^ row) & 7) << 4) + (at & 15));
          if (n0 + kCols * h + j + lane < a.N) o[j + lane] = e;
        }
      }
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(kPairThreads, 1)
    mx_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_wide,
                   const __grid_constant__ CUtensorMap map_narrow, const __grid_constant__ CUtensorMap map_sfx,
                   const __grid_constant__ CUtensorMap map_sfy, const __grid_constant__ CUtensorMap map_out,
                   const MxGemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int S = a.stages;
  uint8_t *sx = smem, *sy = sx + S * kPairXBytes, *ssx = sy + S * kPairYBytes, *ssy = ssx + S * kSfStageBytes;
  uint8_t *staging = ssy + S * kPairSfGroups * kSfStageBytes;
  uint64_t *full = reinterpret_cast<uint64_t *>(staging + kPairStaging);
  uint64_t *empty = full + S, *acc_full = empty + S, *acc_empty = acc_full + 2, *drain = acc_empty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) / 32, 0), lane = threadIdx.x % 32;
  const int rank = static_cast<int>(blockIdx.x & 1u);
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kPairEpi);  // both CTAs' epilogue warps
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_wide);
    tma_prefetch_desc(&map_narrow);
    tma_prefetch_desc(&map_sfx);
    tma_prefetch_desc(&map_sfy);
    if (a.tma_out) tma_prefetch_desc(&map_out);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  cluster_sync();  // both CTAs' barriers and TMEM are set up before either signals the other
  pdl_launch_dependents();

  int kind, tm, n0;
  if (warp == 0) {
    // The whole warp runs the producer's loop, one elected lane issues (see elect_one).  Every
    // load of a stage, of both CTAs, is counted on the even CTA's barrier.
    const uint32_t elected = elect_one(), arms = leader ? elected : 0u;
    const uint64_t pol = policy_evict_last();
    const uint32_t x0 = smem_u32(sx), y0 = smem_u32(sy), sfx0 = smem_u32(ssx), sfy0 = smem_u32(ssy);
    const uint32_t full0 = smem_u32(full), bar0 = map_to_rank(full0, 0);
    auto load_w = [&](int st, int kb) {
      mbar_expect_tx_elected(arms, full0 + 8 * st,
                             2u * (kPairStageBytes - (kind ? (kWide - kNarrow) / 2 * kMxRowBytes : 0)));
      tma_load_2d_pair_elected(elected, y0 + st * kPairYBytes, kind ? &map_narrow : &map_wide, bar0 + 8 * st,
                               kb * kMxRowBytes, n0 + rank * ((kind ? kNarrow : kWide) / 2), pol);
      tma_load_2d_pair_elected(elected, sfy0 + st * kPairSfGroups * kSfStageBytes, &map_sfy, bar0 + 8 * st,
                               kb * 2 * kSfWords, n0 / 128, pol);
    };
    auto load_a = [&](int st, int kb) {
      tma_load_2d_pair_elected(elected, x0 + st * kPairXBytes, &map_x, bar0 + 8 * st, kb * kMxRowBytes,
                               (2 * tm + rank) * kMxRows, pol);
      tma_load_2d_pair_elected(elected, sfx0 + st * kSfStageBytes, &map_sfx, bar0 + 8 * st, kb * 2 * kSfWords,
                               2 * tm + rank, pol);
    };
    PairWalk walk;
    bool more = walk.next(a, kind, tm, n0);
    // The first tile's weight stages do not wait for the previous kernel.
    int pre = 0;
    if (more && a.early)
      for (; pre < min(S, a.kblocks); ++pre) load_w(pre, pre);
    pdl_wait();
    bool ok = true;
    int st = 0;
    uint32_t phase = 0;
    int issued = 0;  // up to S
    for (; ok && more; more = walk.next(a, kind, tm, n0)) {
      for (int kb = 0; kb < a.kblocks; ++kb) {
        if (issued >= pre) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[st], phase ^ 1u, abort_flag, a.status, kStatusProducerWait));
          if (!ok) break;
          load_w(st, kb);
        }
        load_a(st, kb);
        issued = min(issued + 1, S);
        if (++st == S) {
          st = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && leader) {
      // Let the loads already issued land; the odd CTA stays until the even one leaves.
      for (int i = 0; i < issued; ++i) {
        if (--st < 0) {
          st = S - 1;
          phase ^= 1u;
        }
        volatile int no_abort = 0;
        mbar_wait_bounded(&full[st], phase, &no_abort, a.status, kStatusDrainWait);
      }
    }
  } else if (warp == 1) {
    if (leader) {
      const uint32_t elected = elect_one();
      const uint32_t x_lo = desc_lo(smem_u32(sx)), y_lo = desc_lo(smem_u32(sy)), sfx_lo = desc_lo(smem_u32(ssx)),
                     sfy_lo = desc_lo(smem_u32(ssy)), empty0 = smem_u32(empty);
      bool ok = true, any = false;
      int st = 0;
      uint32_t phase = 0;
      uint32_t phases = 0u;  // bit k: parity of the tiles done in accumulator k
      PairWalk walk;
      while (ok && walk.next(a, kind, tm, n0)) {
        const uint32_t d = tmem + (kind ? kWide : 0), sf = tmem + kPairSf;
        // The tile starts at a column (one per 32 rows) of its first scale group, and reaches
        // into a third group only where it has more than 256 - start rows.
        const int start = n0 % 128;
        const uint32_t sfy = sf + 8 + static_cast<uint32_t>(start / 32);
        const uint32_t third = elected && start + (kind ? kNarrow : kWide) > 256 ? 1u : 0u;
        const uint32_t id0 = kind ? idesc_mxf4(2 * kMxRows, kNarrow, 0) : idesc_mxf4(2 * kMxRows, kWide, 0);
        const uint32_t id2 = kind ? idesc_mxf4(2 * kMxRows, kNarrow, 2) : idesc_mxf4(2 * kMxRows, kWide, 2);
        // The last tile in this accumulator has been read.
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&acc_empty[kind], ((phases >> kind) & 1u) ^ 1u, abort_flag,
                                                       a.status, kStatusMmaWait));
        if (!ok) break;
        phases ^= 1u << kind;
        tc_fence_after();
        for (int kb = 0; kb < a.kblocks; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[st], phase, abort_flag, a.status, kStatusMmaWait));
          if (!ok) break;
          tc_fence_after();
          const uint32_t al = x_lo + st * (kPairXBytes >> 4), bl = y_lo + st * (kPairYBytes >> 4),
                         xl = sfx_lo + st * (kSfStageBytes >> 4), yl = sfy_lo + st * (kPairSfGroups * kSfStageBytes >> 4);
          const int left = a.K - kb * kMxStageK;
          any = true;
          pair_half_stage(elected, third, d, al, bl, xl, yl, sf, sf + 8, sfy, id0, id2, kb != 0, left > 64);
          if (left > 128)
            pair_half_stage(elected, third, d, al + 4, bl + 4, xl + (kSfTileBytes >> 4), yl + (kSfTileBytes >> 4),
                            sf + 4, sf + 20, sfy + 12, id0, id2, 1u, left > 192);
          mma_commit_elected<true>(elected, empty0 + 8 * st);
          if (++st == S) {
            st = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        mma_commit_elected<true>(elected, smem_u32(&acc_full[kind]));
      }
      if (!ok && any) {
        if (elected) mma_commit_pair(drain);
        __syncwarp();
        volatile int no_abort = 0;
        mbar_wait_bounded(drain, 0, &no_abort, a.status, kStatusDrainWait);
      }
    }
  } else {
    const int quarter = warp & 3;  // TMEM lanes this warp may access
    const int half = (warp - 2) >> 2;  // takes every other 64-column chunk, from this one on
    pdl_wait();
    uint8_t *buf = staging + (warp - 2) * kPairBufBytes;
    uint32_t phases = 0u;
    PairWalk walk;
    while (walk.next(a, kind, tm, n0)) {
      const int m0 = (2 * tm + rank) * kMxRows + quarter * 32;
      const int width = kind ? kNarrow : kWide, ncols = min(width, a.N - n0);
      float bias[2][2] = {};  // of this warp's chunks, fetched before the accumulator is ready
      if (a.bias)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = 64 * half + 128 * (i / 2) + 32 * (i % 2) + lane;
          if (c < ncols) bias[i / 2][i % 2] = load_scalar_f(a.bias, a.bias_dtype, n0 + c);
        }
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[kind], (phases >> kind) & 1u, abort_flag, a.status,
                                                     kStatusEpilogueWait)))
        break;
      phases ^= 1u << kind;
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (kind ? kWide : 0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c0 = 64 * half + 128 * i;
        const bool last = c0 + 128 >= width;
        const bool live = c0 < ncols;
        uint32_t r[2][32];
        if (live) {
          tmem_ld32(taddr + c0, r[0]);
          tmem_ld32(taddr + c0 + 32, r[1]);
          tmem_ld_wait();
        }
        if (last) {  // this warp has read its columns
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (leader)
              mbar_arrive(&acc_empty[kind]);
            else
              mbar_arrive_remote(map_to_rank(smem_u32(&acc_empty[kind]), 0));
          }
        }
        if (live) pair_emit<DT>(a, &map_out, m0, n0 + c0, lane, bias[i], r, buf);
        if (last) break;
      }
    }
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  // Neither CTA leaves while the other may still signal it or read its shared memory.
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------------------------------ host side

struct MxPlan {
  int pair;     // CTA pairs on 256 tokens x 256 and 192 weight rows
  int tn;       // tokens per tile
  int cluster;  // split tiles: CTAs sharing a tile's K
  int stages;
};

template <int TN>
static int launch_split(const CUtensorMap &mx, const CUtensorMap &my, const CUtensorMap &msx, const CUtensorMap &msy,
                        const MxGemmArgs &a, cudaStream_t stream) {
  static std::atomic<bool> allowed[kMaxDevices];
  const size_t smem = SplitLayout<TN>::bytes(a.stages);
  if (int e = allow_smem(mx_split_kernel<TN>, allowed, "shared memory of the mxfp4 gemm")) return e;
  cudaError_t e = launch(mx_split_kernel<TN>, dim3(static_cast<unsigned>(a.tiles_n) * a.tiles_m * a.cluster),
                         dim3(kSplitThreads), smem, stream, a.cluster, mx, my, msx, msy, a);
  if (e != cudaSuccess) return cuda_error(e, "mxfp4 gemm launch");
  e = cudaGetLastError();
  return e == cudaSuccess ? I8L_OK : cuda_error(e, "mxfp4 gemm launch");
}

template <int DT>
static int launch_pair(const CUtensorMap &mx, const CUtensorMap &my, const CUtensorMap &mn, const CUtensorMap &msx,
                       const CUtensorMap &msy, const CUtensorMap &mo, const MxGemmArgs &a, int pairs,
                       cudaStream_t stream) {
  static std::atomic<bool> allowed[kMaxDevices];
  const size_t smem = pair_smem(a.stages);
  if (int e = allow_smem(mx_pair_kernel<DT>, allowed, "shared memory of the mxfp4 gemm")) return e;
  cudaError_t e = launch(mx_pair_kernel<DT>, dim3(2 * pairs), dim3(kPairThreads), smem, stream, 2, mx, my, mn, msx,
                         msy, mo, a);
  if (e != cudaSuccess) return cuda_error(e, "mxfp4 gemm launch");
  e = cudaGetLastError();
  return e == cudaSuccess ? I8L_OK : cuda_error(e, "mxfp4 gemm launch");
}

// Shared memory of one of two CTAs on an SM (228 KB, 1 KB of it reserved per CTA).
constexpr int kHalfSmem = 233472 / 2 - 1024;

static int split_stage_bytes(int tn) { return kMxRows * kMxRowBytes + tn * kMxRowBytes + 2 * kSfStageBytes; }

// CTAs that share a split tile's K: doubled, to four at most, while they have SMs of their own
// and two stages each (us by CTAs: 16 x 2048 x 2048 4 5.1, 8 5.4; 64 x 2048 x 6144 4 7.3, 8
// 7.8; 256 x 4096 x 14336, 64 tiles, 2 14.7, 4 16.7; 512 x 4096 x 14336, 128 tiles, 1 19.2,
// 2 21.2).
static int split_cluster(int64_t tiles, int kblocks, int sms) {
  int c = 1;
  while (c < 4 && 2 * c * tiles <= sms && kblocks >= 4 * c) c *= 2;
  return c;
}

static int make_mx_plan(int M, int N, int K, const i8l_tile *tile, MxPlan *p) {
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  const int kblocks = (K + kMxStageK - 1) / kMxStageK;
  *p = MxPlan{};
  const i8l_tile t = tile ? *tile : i8l_tile{};
  if (t.split != 0 && t.split != 1 && t.split != 3 && t.split != 4)
    return set_error(I8L_ENOTSUP, "split mode %d unknown to 4-bit products (0 auto, 1 whole, 3 cluster, 4 CTA pairs, 5 CUDA cores)",
                     t.split);
  auto count = [&](int tn) { return (static_cast<int64_t>(N) + kMxRows - 1) / kMxRows * ((static_cast<int64_t>(M) + tn - 1) / tn); };
  p->pair = t.split == 4;
  // Pairs where 128-token split tiles are more than the SMs (us by split tiles and by pairs:
  // 128 x 12288 x 2048, 96 tiles, 9.4 and 9.9; 333 x 6144 x 4096, 144 tiles, 10.4 and 12.5;
  // 256 x 12288 x 2048, 192 tiles, 11.6 and 11.0).
  if (t.split == 0 && t.tok_tile == 0 && M > 64) p->pair = count(128) > di.sms;
  if (p->pair) {
    if (t.split == 4 && (t.swap_ab || t.tok_tile != 128 || t.w_tile != kWide))
      return set_error(I8L_ENOTSUP, "CTA pairs (split 4) take tok_tile 128 x w_tile %d tiles without swap_ab", kWide);
    p->tn = 2 * kMxRows;
    p->cluster = 2;
    const int most = (di.max_smem_optin - static_cast<int>(pair_smem(0))) / (kPairStageBytes + 16);
    p->stages = t.stages ? t.stages : most;
    if (p->stages < 2 || p->stages > most)
      return set_error(I8L_ENOTSUP, "stages %d outside [2, %d] for this tile", p->stages, most);
    return I8L_OK;
  }
  p->tn = t.tok_tile ? t.tok_tile : M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  if (p->tn != 16 && p->tn != 32 && p->tn != 64 && p->tn != 128)
    return set_error(I8L_ENOTSUP, "token tile %d is none of 16, 32, 64, 128", p->tn);
  if (p->tn < 128 && M > p->tn)
    return set_error(I8L_ENOTSUP, "a %d-token tile holds the whole batch, %d tokens given", p->tn, M);
  if (t.tok_tile && (!t.swap_ab || t.w_tile != 128))
    return set_error(I8L_ENOTSUP, "token tiles of 4-bit products take w_tile 128 with swap_ab");
  const int64_t tiles = count(p->tn);
  const int c = t.split == 1 ? 1 : t.cluster ? t.cluster : split_cluster(tiles, kblocks, di.sms);
  if (c < 1 || c > kMaxCluster || c > kblocks)
    return set_error(I8L_ENOTSUP, "cluster size %d outside [1, min(8, k-blocks=%d)]", c, kblocks);
  p->cluster = c;
  const int stage = split_stage_bytes(p->tn);
  const int most = std::min(16, (di.max_smem_optin - 1024 - 256) / stage);
  // More CTAs than SMs share an SM in twos.
  const int share = tiles * c > di.sms ? std::min(5, (kHalfSmem - 1024 - 256) / stage) : 6;
  p->stages = t.stages ? t.stages : std::min((kblocks + c - 1) / c, share);
  if (p->stages < 1 || p->stages > most)
    return set_error(I8L_ENOTSUP, "stages %d outside [1, %d] for this tile", p->stages, most);
  return I8L_OK;
}

static int operand_maps(CUtensorMap *mq, CUtensorMap *ms, const uint8_t *q, int64_t ldq, const uint8_t *sf, int rows,
                        int K, int box_rows, int sf_rows) {
  const int64_t ktiles = (K + 127) / 128;
  if (int e = make_map(mq, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, rows, K / 2, ldq, kMxRowBytes, box_rows,
                       CU_TENSOR_MAP_SWIZZLE_128B, "4-bit operand", CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
    return e;
  return make_map(ms, CU_TENSOR_MAP_DATA_TYPE_UINT32, sf, (rows + 127) / 128, ktiles * kSfWords,
                  ktiles * kSfTileBytes, 2 * kSfWords, sf_rows, CU_TENSOR_MAP_SWIZZLE_NONE, "block scales",
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

}  // namespace i8l

using namespace i8l;

extern "C" int i8l_w4a4_mm(const uint8_t *A, int64_t lda, const uint8_t *sa, const uint8_t *W, int64_t ldw,
                           const uint8_t *sw, const void *bias, int32_t bias_dtype, void *out, int32_t out_dtype,
                           int64_t ldc, int32_t M, int32_t N, int32_t K, const i8l_tile *tile, void *stream) {
  if (M < 0 || N < 0 || K < 0) return set_error(I8L_EINVAL, "negative size M=%d N=%d K=%d", M, N, K);
  if (out_dtype < I8L_BF16 || out_dtype > I8L_F32)
    return set_error(I8L_ENOTSUP, "output dtype code %d not supported (bf16, fp16 or fp32)", out_dtype);
  if (M == 0 || N == 0) return I8L_OK;
  if (K == 0) return set_error(I8L_ENOTSUP, "K=0 is not supported");
  if (K % kMxBlock) return set_error(I8L_ENOTSUP, "K=%d must be a multiple of 32 (whole blocks)", K);
  if (K > kMxMaxK) return set_error(I8L_ENOTSUP, "K=%d is above %d", K, kMxMaxK);
  constexpr int32_t kMost = INT32_MAX - 1024;  // tile coordinates stay inside 32 bits
  if (M > kMost || N > kMost) return set_error(I8L_ENOTSUP, "M=%d or N=%d is above %d", M, N, kMost);
  if (!A || !W || !sa || !sw || !out) return set_error(I8L_EINVAL, "NULL operand pointer");
  if (lda < K / 2 || ldw < K / 2 || ldc < N)
    return set_error(I8L_EINVAL, "leading dimensions lda=%lld ldw=%lld ldc=%lld too small",
                     static_cast<long long>(lda), static_cast<long long>(ldw), static_cast<long long>(ldc));
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(sa) |
       reinterpret_cast<uintptr_t>(sw)) % 16 || lda % 16 || ldw % 16)
    return set_error(I8L_ENOTSUP, "4-bit operands, their row strides and their scales must be 16-byte aligned");
  if (bias && (bias_dtype < I8L_BF16 || bias_dtype > I8L_F32))
    return set_error(I8L_ENOTSUP, "bias dtype code %d not supported", bias_dtype);
  const bool chosen = tile && (tile->split || tile->tok_tile);
  if (chosen ? tile->split == 5 : mx_gemv_wins(M, N, K)) {
    if (M > kMxGemvTokens || (chosen && (tile->swap_ab || tile->w_tile || (tile->tok_tile && tile->tok_tile < M))))
      return set_error(I8L_ENOTSUP, "CUDA-core tiles (split 5) of 4-bit products take at most 4 tokens, w_tile 0, no swap_ab");
    return mx_gemv_run(A, lda, sa, W, ldw, sw, bias, bias_dtype, out, out_dtype, ldc, M, N, K, stream);
  }
  MxPlan p;
  if (int e = make_mx_plan(M, N, K, tile, &p)) return e;
  MxGemmArgs a{};
  a.M = M;
  a.N = N;
  a.K = K;
  a.kblocks = (K + kMxStageK - 1) / kMxStageK;
  const int w_rows = p.pair ? kNarrow : kMxRows;
  a.tiles_n = (N + w_rows - 1) / w_rows;
  a.tiles_m = (M + p.tn - 1) / p.tn;
  a.cluster = p.cluster;
  a.early = mx_weight_early(N) ? 1 : 0;
  a.stages = p.stages;
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.out = out;
  a.out_dtype = out_dtype;
  a.ldc = ldc;
  const int esize = out_dtype == I8L_F32 ? 4 : 2;
  a.vec_store = reinterpret_cast<uintptr_t>(out) % (4 * esize) == 0 && ldc % 4 == 0 ? 1 : 0;
  a.status = status_ptr();
  CUtensorMap mx, my, msx, msy;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (static_cast<int64_t>(a.tiles_m) * a.tiles_n * p.cluster > INT32_MAX)
    return set_error(I8L_ENOTSUP, "%d x %d outputs are too many tiles", M, N);
  if (p.pair) {
    if (int e = operand_maps(&mx, &msx, A, lda, sa, M, K, kMxRows, 1)) return e;
    CUtensorMap mn;
    if (int e = operand_maps(&my, &msy, W, ldw, sw, N, K, kWide / 2, kPairSfGroups)) return e;
    if (int e = make_map(&mn, CU_TENSOR_MAP_DATA_TYPE_UINT8, W, N, K / 2, ldw, kMxRowBytes, kNarrow / 2,
                         CU_TENSOR_MAP_SWIZZLE_128B, "4-bit operand", CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
      return e;
    // A TMA store ends a row at a 16-byte boundary, with zeros past the last column, so rows
    // that end elsewhere are stored plainly.
    CUtensorMap mo{};
    if (reinterpret_cast<uintptr_t>(out) % 16 == 0 && (ldc * esize) % 16 == 0 &&
        (static_cast<int64_t>(N) * esize) % 16 == 0) {
      static const CUtensorMapDataType kTypes[3] = {CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                                    CU_TENSOR_MAP_DATA_TYPE_FLOAT32};
      if (int e = make_map(&mo, kTypes[out_dtype], out, M, N, ldc * esize, 128 / esize, 32, CU_TENSOR_MAP_SWIZZLE_128B,
                           "output"))
        return e;
      a.tma_out = 1;
    }
    a.per_col = FastDiv(static_cast<uint32_t>(a.tiles_m));
    DeviceInfo di;
    if (int e = device_info(&di)) return e;
    const int ctas = tile && tile->ctas ? tile->ctas : di.sms;
    const int64_t tiles = static_cast<int64_t>(a.tiles_m) * ((N + kBoth - 1) / kBoth + (N + kBoth - 1 - kWide) / kBoth);
    const int pairs = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(tiles, ctas / 2)));
    return out_dtype == I8L_BF16  ? launch_pair<I8L_BF16>(mx, my, mn, msx, msy, mo, a, pairs, s)
           : out_dtype == I8L_F16 ? launch_pair<I8L_F16>(mx, my, mn, msx, msy, mo, a, pairs, s)
                                  : launch_pair<I8L_F32>(mx, my, mn, msx, msy, mo, a, pairs, s);
  }
  if (int e = operand_maps(&mx, &msx, W, ldw, sw, N, K, kMxRows, 1)) return e;
  if (int e = operand_maps(&my, &msy, A, lda, sa, M, K, p.tn, 1)) return e;
  switch (p.tn) {
    case 16: return launch_split<16>(mx, my, msx, msy, a, s);
    case 32: return launch_split<32>(mx, my, msx, msy, a, s);
    case 64: return launch_split<64>(mx, my, msx, msy, a, s);
    default: return launch_split<128>(mx, my, msx, msy, a, s);
  }
}
