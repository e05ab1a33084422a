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

// ------------------------------------------------------------------ host side

struct MxPlan {
  int tn;       // tokens per split tile
  int cluster;  // CTAs sharing a tile's K
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
  MxGemmArgs a{};
  a.M = M;
  a.N = N;
  a.K = K;
  a.kblocks = (K + kMxStageK - 1) / kMxStageK;
  a.tiles_n = (N + kMxRows - 1) / kMxRows;
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
  if (int e = operand_maps(&mx, &msx, W, ldw, sw, N, K, kMxRows, 1)) return e;
  if (int e = operand_maps(&my, &msy, A, lda, sa, M, K, p.tn, 1)) return e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p.tn) {
    case 16: return launch_split<16>(mx, my, msx, msy, a, s);
    case 32: return launch_split<32>(mx, my, msx, msy, a, s);
    case 64: return launch_split<64>(mx, my, msx, msy, a, s);
    default: return launch_split<128>(mx, my, msx, msy, a, s);
  }
}
