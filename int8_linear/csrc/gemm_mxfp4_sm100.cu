// The product of two MXFP4 operands for sm_100a:
//     out[m,n] = cast( sum_k A[m,k] * W[n,k] + bias[n] )
// with A and W in 4 bits (mxfp4.cuh), multiplied by tcgen05.mma.kind::mxf4, which applies
// both operands' block scales and accumulates in float32 in TMEM.
//
// Split tiles (mx_split_kernel), for batches of up to a few hundred tokens: the weight is
// the MMA's 128-row side and TN tokens its other side; the CTAs of a thread-block cluster
// share one tile's K, one tile per cluster.  Streaming the weight from HBM bounds these
// shapes, so the split exists to keep every SM loading.  Each CTA leaves its float32
// partial tile in its own shared memory; after a cluster barrier each CTA adds, for its
// share of the outputs, every CTA's partial in rank order through distributed shared
// memory.  So a shape's result does not vary from run to run.
#include <algorithm>

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
  int tma_out;          // pair tiles: outputs leave through shared memory by TMA stores
  int group;            // pair tiles: token tiles that walk over the weight together
  int *status;
};

// ------------------------------------------------------------------ split tiles

constexpr int kSplitThreads = 128;

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

// The MMAs of one stage: its scale tiles into TMEM, then up to four steps of 64 values.
// Steps past K are left out, so a scale tile past the end is never used.
template <int TN>
__device__ __forceinline__ void split_stage_mmas(uint32_t d, uint32_t sf, const uint8_t *x, const uint8_t *y,
                                                 const uint8_t *sfx, const uint8_t *sfy, int k_left, bool first) {
  const int steps = min(4, (k_left + 63) / 64);
  const uint64_t ad = sw128_kmajor_desc(smem_u32(x)), bd = sw128_kmajor_desc(smem_u32(y));
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (2 * t < steps) {
      sf_to_tmem(sf + 4 * t, sf_desc(smem_u32(sfx + t * kSfTileBytes)));
      sf_to_tmem(sf + 8 + 4 * t, sf_desc(smem_u32(sfy + t * kSfTileBytes)));
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k < steps)
      mma_mxf4(d, ad + 2 * k, bd + 2 * k, k & 1 ? idesc_mxf4(kMxRows, TN, 2) : idesc_mxf4(kMxRows, TN, 0),
               sf + 4 * (k >> 1), sf + 8 + 4 * (k >> 1), first && k == 0 ? 0u : 1u);
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

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = a.cluster > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / a.cluster;
  const int tx = tile % a.tiles_n, ty = tile / a.tiles_n;
  const int kb0 = a.kblocks * rank / a.cluster, kb1 = a.kblocks * (rank + 1) / a.cluster;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_sfx);
    tma_prefetch_desc(&map_y);
    tma_prefetch_desc(&map_sfy);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();

  if (warp == 0 && lane == 0) {
    // Weight tiles of the first stages do not wait for the previous kernel.
    const uint64_t pol_w = policy_evict_first(), pol_a = policy_evict_last();
    auto load_w = [&](int st, int kb) {
      mbar_arrive_expect_tx(&full[st], L::kStageBytes);
      tma_load_2d(sx + st * L::kXBytes, &map_x, &full[st], kb * kMxRowBytes, tx * kMxRows, pol_w);
      tma_load_2d(ssx + st * kSfStageBytes, &map_sfx, &full[st], kb * 2 * kSfWords, tx, pol_w);
    };
    const int pre = min(S, kb1 - kb0);
    for (int i = 0; i < pre; ++i) load_w(i, kb0 + i);
    pdl_wait();
    bool ok = true;
    int issued = 0, st = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (issued >= pre) {
        if (!mbar_wait_bounded(&empty[st], phase ^ 1u, abort_flag, a.status, kStatusProducerWait)) {
          ok = false;
          break;
        }
        load_w(st, kb);
      }
      tma_load_2d(sy + st * L::kYBytes, &map_y, &full[st], kb * kMxRowBytes, ty * TN, pol_a);
      tma_load_2d(ssy + st * kSfStageBytes, &map_sfy, &full[st], kb * 2 * kSfWords, ty * TN / kMxRows, pol_a);
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
  } else if (warp == 1 && lane == 0) {
    bool ok = true, any = false;
    int st = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_bounded(&full[st], phase, abort_flag, a.status, kStatusMmaWait)) {
        ok = false;
        break;
      }
      tc_fence_after();
      split_stage_mmas<TN>(tmem, tmem + TN, sx + st * L::kXBytes, sy + st * L::kYBytes, ssx + st * kSfStageBytes,
                           ssy + st * kSfStageBytes, a.K - kb * kMxStageK, !any);
      any = true;
      mma_commit(&empty[st]);
      if (++st == S) {
        st = 0;
        phase ^= 1u;
      }
    }
    if (ok) {
      mma_commit(done);
    } else if (any) {
      mma_commit(drain);
      volatile int no_abort = 0;
      mbar_wait_bounded(drain, 0, &no_abort, a.status, kStatusDrainWait);
    }
  }
  __syncwarp();
  const bool ok = mbar_wait_bounded(done, 0, abort_flag, a.status, kStatusEpilogueWait);
  tc_fence_after();
  const int live = min(TN, a.M - ty * TN);  // tokens of this tile
  // Every MMA has read its operands: the ring holds the partial tile now, [token][128 n].
  if (__syncthreads_and(ok)) {
    const uint32_t taddr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    for (int c = 0; c < live; c += 16) {
      uint32_t r[16];
      tmem_ld16(taddr + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) red[(c + j) * kMxRows + threadIdx.x] = __uint_as_float(r[j]);
    }
  }
  tc_fence_before();
  if (a.cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  pdl_wait();  // this thread's outputs and bias follow the stream's order
  if (*abort_flag == 0) {
    const int units = live * (kMxRows / 4);  // four consecutive outputs each
    const int u1 = units * (rank + 1) / a.cluster;
    for (int u = units * rank / a.cluster + static_cast<int>(threadIdx.x); u < u1; u += kSplitThreads) {
      const int m = u / (kMxRows / 4), c = (u % (kMxRows / 4)) * 4;
      const int n0 = tx * kMxRows + c;
      if (n0 >= a.N) continue;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      const uint32_t at = smem_u32(red + m * kMxRows + c);
      for (int p = 0; p < a.cluster; ++p) {
        const float4 f = a.cluster > 1 ? ld_cluster_v4(map_to_rank(at, static_cast<uint32_t>(p)))
                                       : *reinterpret_cast<const float4 *>(red + m * kMxRows + c);
        v[0] += f.x;
        v[1] += f.y;
        v[2] += f.z;
        v[3] += f.w;
      }
      if (a.bias)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + j < a.N) v[j] += load_scalar_f(a.bias, a.bias_dtype, n0 + j);
      store_out4(a, ty * TN + m, n0, v);
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

constexpr int kPairThreads = 192;  // producer, MMA issuer, four epilogue warps
constexpr int kPairEpi = 4;
constexpr int kPairN = 256;        // weight rows of a tile; each CTA holds half of them
constexpr int kPairXBytes = kMxRows * kMxRowBytes;
constexpr int kPairYBytes = kPairN / 2 * kMxRowBytes;
constexpr int kPairStageBytes = kPairXBytes + kPairYBytes + 3 * kSfStageBytes;
constexpr int kPairBufBytes = 2048;                              // 32 rows x 64 bytes of output
constexpr int kPairStaging = kPairEpi * 2 * kPairBufBytes;
// TMEM columns: two accumulators of 256 columns that share 32 of them, then the scales of
// one stage (8 for the tokens' 128 rows, 16 for the weight's 256).
constexpr int kPairAcc1 = 224;
constexpr int kPairSf = 480;

static size_t pair_smem(int stages) {
  return 1024 /* alignment slack */ + static_cast<size_t>(stages) * kPairStageBytes + kPairStaging +
         2 * kPairN * 4 /* bias, per accumulator */ + static_cast<size_t>(2 * stages + 6) * 8 + 16;
}

// Tile index -> (token tile, weight tile): `group` token tiles walk over the weight tiles
// together, so that the pairs running at one time share operands in L2.
__device__ __forceinline__ void pair_coords(const MxGemmArgs &a, int t, int &tm, int &tn) {
  const int per_group = a.group * a.tiles_n;
  const int g = t / per_group, first = g * a.group;
  const int gsz = min(a.tiles_m - first, a.group);
  const int r = t - g * per_group;
  tm = first + r % gsz;
  tn = r / gsz;
}

// One 32-column chunk of this thread's token row: bias, rounding, and the store through the
// warp's staging buffer (64-byte rows in the 64-byte swizzle, one TMA store) or straight to
// memory.
__device__ __forceinline__ void pair_emit(const MxGemmArgs &a, const CUtensorMap *map_out, int m0, int n0, int lane,
                                          const float *bias, const uint32_t (&r0)[16], const uint32_t (&r1)[16],
                                          uint8_t *staging, uint32_t &count) {
  float v[32];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    v[j] = __uint_as_float(r0[j]);
    v[16 + j] = __uint_as_float(r1[j]);
  }
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 b = *reinterpret_cast<const float4 *>(bias + j);
      v[j] += b.x;
      v[j + 1] += b.y;
      v[j + 2] += b.z;
      v[j + 3] += b.w;
    }
  }
  if (a.tma_out) {
    const int halves = a.out_dtype == I8L_F32 ? 2 : 1;  // boxes of 16 float32 or 32 16-bit columns
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h >= halves) break;
      if (count >= 2 && lane == 0) bulk_wait_read<1>();
      __syncwarp();
      uint8_t *buf = staging + (count & 1u) * kPairBufBytes;
      ++count;
      uint32_t w[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        w[j] = halves == 2 ? __float_as_uint(v[16 * h + j]) : pack16x2(a.out_dtype, v[2 * j], v[2 * j + 1]);
      uint8_t *rowp = buf + lane * 64;
      const int sw = (lane >> 1) & 3;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *reinterpret_cast<uint4 *>(rowp + ((c ^ sw) << 4)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        const int n = n0 + 16 * h;
        if (n < a.N && m0 < a.M) tma_store_2d(map_out, buf, n, m0);  // skip boxes wholly outside
        bulk_commit();
      }
    }
  } else if (m0 + lane < a.M) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float q[4] = {v[j], v[j + 1], v[j + 2], v[j + 3]};
      if (n0 + j < a.N) store_out4(a, m0 + lane, n0 + j, q);
    }
  }
}

__global__ void __launch_bounds__(kPairThreads, 1)
    mx_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y,
                   const __grid_constant__ CUtensorMap map_sfx, const __grid_constant__ CUtensorMap map_sfy,
                   const __grid_constant__ CUtensorMap map_out, const MxGemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int S = a.stages;
  uint8_t *sx = smem, *sy = sx + S * kPairXBytes, *ssx = sy + S * kPairYBytes, *ssy = ssx + S * kSfStageBytes;
  uint8_t *staging = ssy + S * 2 * kSfStageBytes;
  float *bias_cols = reinterpret_cast<float *>(staging + kPairStaging);
  uint64_t *full = reinterpret_cast<uint64_t *>(bias_cols + 2 * kPairN);
  uint64_t *empty = full + S, *acc_full = empty + S, *acc_empty = acc_full + 2, *shared_free = acc_empty + 2,
           *drain = shared_free + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = static_cast<int>(blockIdx.x & 1u);
  const bool leader = rank == 0;
  const int first_tile = static_cast<int>(blockIdx.x >> 1), step = static_cast<int>(gridDim.x >> 1);
  const int total = a.tiles_m * a.tiles_n;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kPairEpi);  // both CTAs' epilogue warps
    }
    mbar_init(shared_free, 2 * kPairEpi);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_y);
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
  const uint32_t tmem = *tmem_slot;
  cluster_sync();  // both CTAs' barriers and TMEM are set up before either signals the other
  pdl_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol = policy_evict_last();
      const uint32_t tx = 2u * kPairStageBytes;  // both CTAs' loads, counted on the even CTA's barrier
      auto load_w = [&](int st, int kb, int tn) {
        const uint32_t bar = map_to_rank(smem_u32(&full[st]), 0);
        tma_load_2d_pair(sy + st * kPairYBytes, &map_y, bar, kb * kMxRowBytes, tn * kPairN + rank * (kPairN / 2), pol);
        tma_load_2d_pair(ssy + st * 2 * kSfStageBytes, &map_sfy, bar, kb * 2 * kSfWords, tn * 2, pol);
      };
      auto load_a = [&](int st, int kb, int tm) {
        const uint32_t bar = map_to_rank(smem_u32(&full[st]), 0);
        tma_load_2d_pair(sx + st * kPairXBytes, &map_x, bar, kb * kMxRowBytes, (2 * tm + rank) * kMxRows, pol);
        tma_load_2d_pair(ssx + st * kSfStageBytes, &map_sfx, bar, kb * 2 * kSfWords, 2 * tm + rank, pol);
      };
      // The first tile's weight stages do not wait for the previous kernel.
      int tm, tn, pre = 0;
      if (first_tile < total) {
        pair_coords(a, first_tile, tm, tn);
        for (; pre < min(S, a.kblocks); ++pre) {
          if (leader) mbar_arrive_expect_tx(&full[pre], tx);
          load_w(pre, pre, tn);
        }
      }
      pdl_wait();
      bool ok = true;
      int st = 0;
      uint32_t phase = 0;
      long long issued = 0;
      for (int t = first_tile; ok && t < total; t += step) {
        pair_coords(a, t, tm, tn);
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (issued >= pre) {
            if (!mbar_wait_bounded(&empty[st], phase ^ 1u, abort_flag, a.status, kStatusProducerWait)) {
              ok = false;
              break;
            }
            if (leader) mbar_arrive_expect_tx(&full[st], tx);
            load_w(st, kb, tn);
          }
          load_a(st, kb, tm);
          ++issued;
          if (++st == S) {
            st = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && leader) {
        // Let the loads already issued land; the odd CTA stays until the even one leaves.
        for (long long i = 0; i < (issued < S ? issued : S); ++i) {
          if (--st < 0) {
            st = S - 1;
            phase ^= 1u;
          }
          volatile int no_abort = 0;
          mbar_wait_bounded(&full[st], phase, &no_abort, a.status, kStatusDrainWait);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      bool ok = true, any = false;
      int st = 0, n = 0;
      uint32_t phase = 0;
      for (int t = first_tile; ok && t < total; t += step, ++n) {
        const int acc = n & 1;
        // This accumulator's last tile has been read, and so have the columns that it
        // shares with the other accumulator's tile.
        if (!mbar_wait_bounded(&acc_empty[acc], ((n >> 1) & 1) ^ 1, abort_flag, a.status, kStatusMmaWait) ||
            (n > 0 && !mbar_wait_bounded(shared_free, (n - 1) & 1, abort_flag, a.status, kStatusMmaWait))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + (acc ? kPairAcc1 : 0), sf = tmem + kPairSf;
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait_bounded(&full[st], phase, abort_flag, a.status, kStatusMmaWait)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int steps = min(4, (a.K - kb * kMxStageK + 63) / 64);
          const uint64_t ad = sw128_kmajor_desc(smem_u32(sx + st * kPairXBytes));
          const uint64_t bd = sw128_kmajor_desc(smem_u32(sy + st * kPairYBytes));
          const uint64_t xd = sf_desc(smem_u32(ssx + st * kSfStageBytes));
          const uint64_t yd = sf_desc(smem_u32(ssy + st * 2 * kSfStageBytes));
          constexpr uint64_t kTileStep = kSfTileBytes >> 4;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (2 * h < steps) {
              sf_to_tmem_pair(sf + 4 * h, xd + h * kTileStep);
              sf_to_tmem_pair(sf + 8 + 8 * h, yd + h * kTileStep);
              sf_to_tmem_pair(sf + 12 + 8 * h, yd + (2 + h) * kTileStep);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k < steps)
              mma_mxf4_pair(d, ad + 2 * k, bd + 2 * k,
                            k & 1 ? idesc_mxf4(2 * kMxRows, kPairN, 2) : idesc_mxf4(2 * kMxRows, kPairN, 0),
                            sf + 4 * (k >> 1), sf + 8 + 8 * (k >> 1), kb == 0 && k == 0 ? 0u : 1u);
          }
          any = true;
          mma_commit_pair_mc(&empty[st], 0x3);
          if (++st == S) {
            st = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        mma_commit_pair_mc(&acc_full[acc], 0x3);
      }
      if (!ok && any) {
        mma_commit_pair(drain);
        volatile int no_abort = 0;
        mbar_wait_bounded(drain, 0, &no_abort, a.status, kStatusDrainWait);
      }
    }
  } else {
    const int quarter = warp & 3;  // TMEM lanes this warp may access
    const int tid = threadIdx.x - 64;
    auto release = [&](uint64_t *bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader)
          mbar_arrive(bar);
        else
          mbar_arrive_remote(map_to_rank(smem_u32(bar), 0));
      }
    };
    pdl_wait();
    uint8_t *buf = staging + quarter * 2 * kPairBufBytes;
    uint32_t count = 0;
    int n = 0;
    for (int t = first_tile; t < total; t += step, ++n) {
      int tm, tn;
      pair_coords(a, t, tm, tn);
      const int acc = n & 1;
      const int m0 = (2 * tm + rank) * kMxRows + quarter * 32, n0 = tn * kPairN;
      const int ncols = min(kPairN, a.N - n0);
      float *bias = bias_cols + acc * kPairN;
      if (a.bias)
        for (int c = tid; c < kPairN; c += kPairEpi * 32)
          bias[c] = c < ncols ? load_scalar_f(a.bias, a.bias_dtype, n0 + c) : 0.f;
      const bool ok = mbar_wait_bounded(&acc_full[acc], (n >> 1) & 1, abort_flag, a.status, kStatusEpilogueWait);
      // All four warps go on or all stop; the barrier also publishes the bias columns.
      if (!named_bar_and(2, kPairEpi * 32, ok)) break;
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (acc ? kPairAcc1 : 0);
      // The shared columns first: the last chunk of accumulator 0, the first of 1.
      for (int i = 0; i < kPairN / 32; ++i) {
        const int c0 = acc ? 32 * i : (i == 0 ? kPairN - 32 : 32 * (i - 1));
        uint32_t r0[16], r1[16];
        const bool live = c0 < ncols;
        if (live) {
          tmem_ld16(taddr + c0, r0);
          tmem_ld16(taddr + c0 + 16, r1);
          tmem_ld_wait();
        }
        if (i == 0) release(shared_free);
        if (i == kPairN / 32 - 1) release(&acc_empty[acc]);
        if (live) pair_emit(a, &map_out, m0, n0 + c0, lane, bias + c0, r0, r1, buf, count);
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
  int pair;     // CTA pairs on 256 x 256 tiles
  int tn;       // tokens per tile
  int cluster;  // split tiles: CTAs sharing a tile's K
  int stages;
};

template <typename Kernel>
static int allow_smem(Kernel kernel, size_t smem, size_t *configured) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_error(e, "cudaGetDevice");
  if (dev < 0 || dev >= 64 || smem > configured[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return cuda_error(e, "cudaFuncSetAttribute(mxfp4 gemm smem)");
    if (dev >= 0 && dev < 64) configured[dev] = smem;
  }
  return I8L_OK;
}

template <int TN>
static int launch_split(const CUtensorMap &mx, const CUtensorMap &my, const CUtensorMap &msx, const CUtensorMap &msy,
                        const MxGemmArgs &a, cudaStream_t stream) {
  static size_t configured[64] = {};
  const size_t smem = SplitLayout<TN>::bytes(a.stages);
  if (int e = allow_smem(mx_split_kernel<TN>, smem, configured)) return e;
  cudaError_t e = launch(mx_split_kernel<TN>, dim3(static_cast<unsigned>(a.tiles_n) * a.tiles_m * a.cluster),
                         dim3(kSplitThreads), smem, stream, a.cluster, mx, my, msx, msy, a);
  if (e != cudaSuccess) return cuda_error(e, "mxfp4 gemm launch");
  e = cudaGetLastError();
  return e == cudaSuccess ? I8L_OK : cuda_error(e, "mxfp4 gemm launch");
}

static int split_stage_bytes(int tn) { return kMxRows * kMxRowBytes + tn * kMxRowBytes + 2 * kSfStageBytes; }

static int make_mx_plan(int M, int N, int K, const i8l_tile *tile, MxPlan *p) {
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  const int kblocks = (K + kMxStageK - 1) / kMxStageK;
  *p = MxPlan{};
  if (tile && tile->split == 4 ? true : !(tile && (tile->tok_tile || tile->split)) && M > 256) {
    if (tile && tile->split == 4 && (tile->swap_ab || tile->tok_tile != 128 || tile->w_tile != 256))
      return set_error(I8L_ENOTSUP, "CTA pairs (split 4) take tok_tile 128 x w_tile 256 tiles without swap_ab");
    p->pair = 1;
    p->tn = 2 * kMxRows;
    p->cluster = 2;
    const int most = std::min(16, (di.max_smem_optin - static_cast<int>(pair_smem(0))) / (kPairStageBytes + 16));
    p->stages = tile && tile->stages ? tile->stages : most;
    if (p->stages < 2 || p->stages > most)
      return set_error(I8L_ENOTSUP, "stages %d outside [2, %d] for this tile", p->stages, most);
    return I8L_OK;
  }
  p->tn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  if (tile && tile->tok_tile) p->tn = tile->tok_tile;
  if (p->tn != 16 && p->tn != 32 && p->tn != 64 && p->tn != 128)
    return set_error(I8L_ENOTSUP, "token tile %d is none of 16, 32, 64, 128", p->tn);
  if (p->tn < 128 && M > p->tn)
    return set_error(I8L_ENOTSUP, "a %d-token tile holds the whole batch, %d tokens given", p->tn, M);
  const int tiles = ((N + kMxRows - 1) / kMxRows) * ((M + p->tn - 1) / p->tn);
  int c = 1;
  while (c < 8 && 2 * c * tiles <= di.sms && kblocks / (2 * c) >= 1) c *= 2;
  if (tile && tile->cluster) c = tile->cluster;
  if (c < 1 || c > 8 || c > kblocks)
    return set_error(I8L_ENOTSUP, "cluster size %d outside [1, min(8, k-blocks=%d)]", c, kblocks);
  p->cluster = c;
  const int most = std::min(16, (di.max_smem_optin - 1024 - 256) / split_stage_bytes(p->tn));
  int s = std::min((kblocks + c - 1) / c, p->tn <= 64 ? 5 : 6);
  if (tile && tile->stages) s = tile->stages;
  if (s < 1 || s > most) return set_error(I8L_ENOTSUP, "stages %d outside [1, %d] for this tile", s, most);
  p->stages = s;
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
  if (!A || !W || !sa || !sw || !out) return set_error(I8L_EINVAL, "NULL operand pointer");
  if (lda < K / 2 || ldw < K / 2 || ldc < N)
    return set_error(I8L_EINVAL, "leading dimensions lda=%lld ldw=%lld ldc=%lld too small",
                     static_cast<long long>(lda), static_cast<long long>(ldw), static_cast<long long>(ldc));
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(sa) |
       reinterpret_cast<uintptr_t>(sw)) % 16 || lda % 16 || ldw % 16)
    return set_error(I8L_ENOTSUP, "4-bit operands, their row strides and their scales must be 16-byte aligned");
  if (bias && (bias_dtype < I8L_BF16 || bias_dtype > I8L_F32))
    return set_error(I8L_ENOTSUP, "bias dtype code %d not supported", bias_dtype);
  MxPlan p;
  if (int e = make_mx_plan(M, N, K, tile, &p)) return e;
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  MxGemmArgs a{};
  a.M = M;
  a.N = N;
  a.K = K;
  a.kblocks = (K + kMxStageK - 1) / kMxStageK;
  const int w_rows = p.pair ? kPairN : kMxRows;
  a.tiles_n = (N + w_rows - 1) / w_rows;
  a.tiles_m = (M + p.tn - 1) / p.tn;
  a.cluster = p.cluster;
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
    if (int e = operand_maps(&my, &msy, W, ldw, sw, N, K, kPairN / 2, 2)) return e;
    CUtensorMap mo{};
    // A TMA store ends a row at a 16-byte boundary, with zeros past the last column, so rows
    // that end elsewhere are stored plainly.
    if (reinterpret_cast<uintptr_t>(out) % 16 == 0 && (ldc * esize) % 16 == 0 &&
        (static_cast<int64_t>(N) * esize) % 16 == 0) {
      static const CUtensorMapDataType kTypes[3] = {CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                                    CU_TENSOR_MAP_DATA_TYPE_FLOAT32};
      if (int e = make_map(&mo, kTypes[out_dtype], out, M, N, ldc * esize, 64 / esize, 32, CU_TENSOR_MAP_SWIZZLE_64B,
                           "output"))
        return e;
      a.tma_out = 1;
    }
    a.group = std::min(8, a.tiles_m);
    static size_t configured[64] = {};
    const size_t smem = pair_smem(a.stages);
    if (int e = allow_smem(mx_pair_kernel, smem, configured)) return e;
    const int pairs = std::min(a.tiles_m * a.tiles_n, (tile && tile->ctas ? tile->ctas : di.sms) / 2);
    cudaError_t e = launch(mx_pair_kernel, dim3(2 * std::max(1, pairs)), dim3(kPairThreads), smem, s, 2, mx, my, msx,
                           msy, mo, a);
    if (e != cudaSuccess) return cuda_error(e, "mxfp4 gemm launch");
    e = cudaGetLastError();
    return e == cudaSuccess ? I8L_OK : cuda_error(e, "mxfp4 gemm launch");
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
