// The product of two MXFP4 operands for a few tokens (split mode 5 of w4a4_mm): CUDA cores.
//     out[m,n] = cast( sum over blocks of 2^(sa + sw) * (A block . W block) + bias[n] )
//
// Twice an e2m1 value is an integer of at most 12, so a block's 32 products are exact in
// int8 dot products (dp4a), and only the blocks' sums, each times its two powers of two, are
// added in float32, in a fixed order.  A word of eight codes becomes int8 magnitudes by two
// byte permutes that look the codes up; a third and fourth give a mask of the negative ones,
// whose share is taken off twice: a . w = a . |w| - 2 a . (|w| where w < 0).
//
// With one to four tokens the weight's bytes bound the product, and a tensor-core tile adds
// the latencies of its set-up, its barriers and the exchange of partial sums between CTAs.
// Here a CTA owns eight whole output columns: the weight rows that share the 32-byte sectors
// of their scale tiles (rows 2j, 2j+1 and those 32, 64 and 96 further on).  A thread takes
// one 16-byte load, a whole block, of four of the rows at a time, all in flight together and,
// as weights do not depend on the previous kernel, before the dependency wait.  Measured at
// 2048 x 2048 (2.2 MB): 2.6 us for one token, 4.0 for four, a launch of an empty kernel being
// about 1.5; a tensor-core tile takes 4.8 to 5.0.  The permutes and dot products, half-rate
// instructions, bound it from about 4096 x 2048 on (4.0 us).
#include <algorithm>

#include "common.cuh"
#include "epilogue.cuh"
#include "internal.h"
#include "mxfp4.cuh"

namespace i8l {

struct MxGemvArgs {
  const uint8_t *A, *sa, *W, *sw;
  long long lda, ldw;
  int M, N;
  int blocks, ktiles;
  int early;  // see mx_weight_early
  const void *bias;
  int bias_dtype;
  void *out;
  int out_dtype;
  long long ldc;
};

// Twice the magnitudes of the four codes in the low 16 bits of w, one per byte.
__device__ __forceinline__ uint32_t e2m1_mag4(uint32_t w) { return __byte_perm(0x03020100u, 0x0c080604u, w & 0x7777u); }
// Per byte 0xff where that code is negative, else 0x80: bit 3 of a selector nibble spreads the
// top bit of the byte it selects.
__device__ __forceinline__ uint32_t e2m1_neg4(uint32_t w) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(r) : "r"(0x80808080u), "r"(w));
  return r;
}

// kSpan threads side by side along K; two sets of them share the octet's rows.
template <int MT, int kSpan>
__global__ void __launch_bounds__(2 * kSpan) mx_gemv_kernel(const MxGemvArgs a) {
  constexpr int kRows = 4;                 // rows a thread works on
  constexpr int kWarps = kSpan / 32;       // warps whose sums make an output
  __shared__ float part[2][kWarps][kRows * MT];
  const int set = threadIdx.x / kSpan, t = threadIdx.x % kSpan;
  const int tile = static_cast<int>(blockIdx.x) / 16, first = (static_cast<int>(blockIdx.x) % 16) * 2;
  auto row_of = [&](int e) { return tile * 128 + first + (e & 1) + 32 * (2 * set + (e >> 1)); };

  pdl_launch_dependents();
  const uint8_t *wrow[kRows];
  bool in[kRows];
#pragma unroll
  for (int e = 0; e < kRows; ++e) {
    in[e] = row_of(e) < a.N;
    wrow[e] = a.W + static_cast<long long>(in[e] ? row_of(e) : 0) * a.ldw;
  }
  uint4 w[kRows];
  uint2 s0, s1;  // scale words of the set's rows `first` and `first + 1`
  auto load_w = [&](int b) {
#pragma unroll
    for (int e = 0; e < kRows; ++e)
      w[e] = b < a.blocks && in[e] ? *reinterpret_cast<const uint4 *>(wrow[e] + b * 16) : make_uint4(0u, 0u, 0u, 0u);
    s0 = s1 = make_uint2(0u, 0u);
    if (b < a.blocks) {
      const uint8_t *p = a.sw + (static_cast<long long>(tile) * a.ktiles + (b >> 2)) * kSfTileBytes + first * 16 + set * 8;
      s0 = *reinterpret_cast<const uint2 *>(p);
      s1 = *reinterpret_cast<const uint2 *>(p + 16);
    }
  };
  if (a.early) load_w(t);
  pdl_wait();
  if (!a.early) load_w(t);

  float acc[kRows][MT] = {};
  for (int b = t; b < a.blocks; b += kSpan) {
    // This block of every token, as signed int8, and its scale.
    uint32_t x[MT][8];
    float sx[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const bool live = m < a.M;
      const uint4 v = live ? *reinterpret_cast<const uint4 *>(a.A + m * a.lda + b * 16) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t c[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t codes = h ? c[i] >> 16 : c[i];
          const uint32_t neg = (e2m1_neg4(codes) & 0x01010101u) * 0xffu;
          x[m][2 * i + h] = __vsub4(e2m1_mag4(codes) ^ neg, neg);
        }
      sx[m] = live ? mx_scale_value(a.sa[static_cast<long long>(b >> 2) * kSfTileBytes + m * 16 + (b & 3)]) : 0.f;
    }
    uint4 cur[kRows];
    float sw[kRows];
    const int shift = 8 * (b & 3);
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
      cur[e] = w[e];
      const uint2 s = e & 1 ? s1 : s0;
      sw[e] = 0.25f * mx_scale_value(((e >> 1 ? s.y : s.x) >> shift) & 0xffu);
    }
    if (b + kSpan < a.blocks) load_w(b + kSpan);
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
      const uint32_t c[4] = {cur[e].x, cur[e].y, cur[e].z, cur[e].w};
      int all[MT] = {}, neg[MT] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t codes = h ? c[i] >> 16 : c[i];
          const uint32_t mag = e2m1_mag4(codes), sub = mag & e2m1_neg4(codes) & 0x7f7f7f7fu;
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            all[m] = __dp4a(static_cast<int>(x[m][2 * i + h]), static_cast<int>(mag), all[m]);
            neg[m] = __dp4a(static_cast<int>(x[m][2 * i + h]), static_cast<int>(sub), neg[m]);
          }
        }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        // The smaller scale first: the sum times it is exact (an integer below 2^13 times
        // 2^-129 at least) and leaves float32's range only where the product does too.  By their
        // bits, which puts the scale of a NaN block last.
        const uint32_t ws = __float_as_uint(sw[e]), xs = __float_as_uint(sx[m]);
        acc[e][m] = fmaf(static_cast<float>(all[m] - 2 * neg[m]) * __uint_as_float(min(ws, xs)),
                         __uint_as_float(max(ws, xs)), acc[e][m]);
      }
    }
  }

  // The sums of a set's threads: a butterfly in each warp, then its warps in order.
#pragma unroll
  for (int e = 0; e < kRows; ++e)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float v = acc[e][m];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if ((threadIdx.x & 31) == 0) part[set][t / 32][e * MT + m] = v;
    }
  __syncthreads();
  if (t < kRows * MT) {
    const int e = t / MT, m = t % MT, n = row_of(e);
    if (m < a.M && n < a.N) {
      float v = part[set][0][t];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) v += part[set][i][t];
      if (a.bias) v += load_scalar_f(a.bias, a.bias_dtype, n);
      store_elem(a.out, a.out_dtype, m * a.ldc + n, 0, v);
    }
  }
}

// The arithmetic grows with the tokens, two, four or eight dot products a word, where a
// tensor-core tile's time does not (us here and there: 1 x 8192 x 2048 5.1 and 5.9,
// 1 x 12288 x 2048 7.1 and 6.3; 2 x 4096 x 2048 4.7 and 5.4, 2 x 2048 x 6144 6.9 and 5.9;
// 4 x 2048 x 2048 3.9 and 5.0, 4 x 4096 x 2048 6.1 and 5.5).
bool mx_gemv_wins(int M, int N, int K) {
  return M <= kMxGemvTokens && static_cast<int64_t>(N) * K * (M <= 2 ? M : 4) <= 1 << 24;
}

int mx_gemv_run(const uint8_t *A, int64_t lda, const uint8_t *sa, const uint8_t *W, int64_t ldw, const uint8_t *sw,
                const void *bias, int32_t bias_dtype, void *out, int32_t out_dtype, int64_t ldc, int32_t M, int32_t N,
                int32_t K, void *stream) {
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  MxGemvArgs a;
  a.A = A;
  a.sa = sa;
  a.W = W;
  a.sw = sw;
  a.lda = lda;
  a.ldw = ldw;
  a.M = M;
  a.N = N;
  a.blocks = K / kMxBlock;
  a.ktiles = (K + 127) / 128;
  a.early = mx_weight_early(N) ? 1 : 0;
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.out = out;
  a.out_dtype = out_dtype;
  a.ldc = ldc;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(N) + 127) / 128 * 16));
  // Twice the threads a column where K has blocks for them and the columns are few.
  const bool wide = a.blocks >= 128 && static_cast<int64_t>(grid.x) * 128 < 1024LL * di.sms;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (M == 1)
    e = wide ? launch(mx_gemv_kernel<1, 128>, grid, dim3(256), 0, s, 1, a) : launch(mx_gemv_kernel<1, 64>, grid, dim3(128), 0, s, 1, a);
  else if (M == 2)
    e = wide ? launch(mx_gemv_kernel<2, 128>, grid, dim3(256), 0, s, 1, a) : launch(mx_gemv_kernel<2, 64>, grid, dim3(128), 0, s, 1, a);
  else
    e = wide ? launch(mx_gemv_kernel<4, 128>, grid, dim3(256), 0, s, 1, a) : launch(mx_gemv_kernel<4, 64>, grid, dim3(128), 0, s, 1, a);
  if (e != cudaSuccess) return cuda_error(e, "mxfp4 gemv launch");
  e = cudaGetLastError();
  return e == cudaSuccess ? I8L_OK : cuda_error(e, "mxfp4 gemv launch");
}

}  // namespace i8l
