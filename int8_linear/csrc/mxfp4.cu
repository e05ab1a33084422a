// MXFP4 quantisers for sm_100a and the way back:
//   quant_mxfp4              block-quantise a bf16/fp16/fp32 matrix
//   silu_mul_quant_mxfp4     SiLU-and-mul, then the same
//   add_rmsnorm_quant_mxfp4  residual add + RMSNorm, then the same
//   dequant_mxfp4            the values that codes and scales stand for
// They stand beside the per-token int8 quantisers (quant.cu) and compute the same y; only
// what y is stored in differs.  A block's scale depends on its own 32 values, so there is
// no row reduction in the plain and SiLU quantisers: a lane takes eight values, four
// neighbouring lanes share a block (two shuffles), and the matrix is walked as one flat
// list of eight-value vectors or of blocks.  All four kernels move each byte once and are
// bound by HBM: at 8192 rows (inputs larger than L2) quant_mxfp4 and dequant_mxfp4 take 26 us
// of 8192 values, the measured copy rate; SiLU takes 40 us of 6144 (86 %; its arithmetic is
// what is left) and the norm 39 of 4096 with a residual (86 %).
//
// A 4-bit value next to the border between two steps flips on the last bit of y, so y is
// computed to the bit: the norm's mean in float64, and SiLU in float32 with a second, exact
// pass for the few values where the float32 error could change the rounding.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "mxfp4.cuh"
#include "rows.cuh"

namespace i8l {

constexpr int kFlatThreads = 128;

struct MxOut {
  uint8_t *q;
  long long ldq;  // bytes
  uint8_t *sf;
  int ktiles;  // 128-value tiles along K
};

// Writes one block's scale byte and, after the row's last block, the zero bytes up to the
// end of its word.
__device__ __forceinline__ void store_sf(const MxOut &o, long long row, int block, int blocks, uint32_t byte) {
  uint8_t *p = o.sf + sf_word_offset(row, block >> 2, o.ktiles);
  p[block & 3] = static_cast<uint8_t>(byte);
  if (block == blocks - 1)
    for (int i = (block & 3) + 1; i < 4; ++i) p[i] = 0;
}

// Zero words of the scale tiles below the last row: word i of (rows_pad - rows) * ktiles.
__device__ __forceinline__ void zero_pad_word(const MxOut &o, long long rows, long long i) {
  *reinterpret_cast<uint32_t *>(o.sf + sf_word_offset(rows + i / o.ktiles, static_cast<int>(i % o.ktiles), o.ktiles)) = 0u;
}

template <int DT>
__device__ __forceinline__ void load8(const void *base, long long idx, bool vec, float (&v)[8]) {
  using T = typename ActType<DT>::T;
  const T *p = static_cast<const T *>(base) + idx;
  if (vec) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 8 / kPer; ++h) {
      const uint4 raw = reinterpret_cast<const uint4 *>(p)[h];
      const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
      for (int i = 0; i < kPer; ++i) v[h * kPer + i] = ActType<DT>::to_f32(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ActType<DT>::to_f32(p[i]);
  }
}

// Eight 16-bit values from any alignment, as they lie in memory.
__device__ __forceinline__ uint4 load8_raw(const void *base, long long idx, bool vec) {
  const uint16_t *p = static_cast<const uint16_t *>(base) + idx;
  if (vec) return *reinterpret_cast<const uint4 *>(p);
  return make_uint4(p[0] | (static_cast<uint32_t>(p[1]) << 16), p[2] | (static_cast<uint32_t>(p[3]) << 16),
                    p[4] | (static_cast<uint32_t>(p[5]) << 16), p[6] | (static_cast<uint32_t>(p[7]) << 16));
}

template <int DT>
__device__ __forceinline__ void unpack8(const uint4 &w, float (&v)[8]) {
  unpack2<DT>(w.x, v[0], v[1]);
  unpack2<DT>(w.y, v[2], v[3]);
  unpack2<DT>(w.z, v[4], v[5]);
  unpack2<DT>(w.w, v[6], v[7]);
}

template <int DT>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7]));
}

// ------------------------------------------------------------------ SiLU

template <int N>
using Int = std::integral_constant<int, N>;

// ln(2)^k / k!
__host__ __device__ constexpr double exp2_term(int k) { return k == 0 ? 1. : exp2_term(k - 1) * (0.6931471805599453 / k); }

// float32(g / (1 + exp(-g)) * u) in float64, for g and u that are 16-bit values: within 2^-50
// of the exact value before its one rounding.  exp(-g) = 2^n 2^r with n the nearest integer to
// -g log2 e (adding 1.5 * 2^52 rounds to it and leaves it in the low bits) and 2^r its Taylor
// sum up to r^13 (|r| <= 1/2: the rest is below 2^-56), summed in pairs of pairs; the
// reciprocal is an approximation and two Newton steps.  g is held within +-690, beyond which
// 1 + exp(-g) is 1 or the product below float32's range.  An infinite g comes out as an
// infinity or a NaN, either of which makes its block NaN.  (With exp and a division the 4096 x
// 6144 kernel took 0.6 us more.)
__device__ __forceinline__ float silu_mul_exact(float g, float u) {
  constexpr double kLog2e = 1.4426950408889634, kRest = 2.0355273740931033e-17, kRound = 6755399441055744.;
  const double a = -static_cast<double>(fminf(fmaxf(g, -690.f), 690.f));
  const double t = fma(a, kLog2e, kRound), n = t - kRound;
  const double r = fma(a, kRest, fma(a, kLog2e, -n)), r2 = r * r, r4 = r2 * r2;
  auto pair = [&](auto k) {
    constexpr double lo = exp2_term(decltype(k)::value), hi = exp2_term(decltype(k)::value + 1);
    return fma(r, hi, lo);
  };
  const double c0 = fma(pair(Int<2>{}), r2, pair(Int<0>{})), c4 = fma(pair(Int<6>{}), r2, pair(Int<4>{}));
  const double c8 = fma(pair(Int<10>{}), r2, pair(Int<8>{})), c12 = pair(Int<12>{});
  const double e = fma(fma(c12, r4, c8), r4 * r4, fma(c4, r4, c0));
  const double d = fma(e, __hiloint2double((__double2loint(t) + 1023) << 20, 0), 1.);
  double q;
  asm("rcp.approx.ftz.f64 %0, %1;" : "=d"(q) : "d"(d));
  q = fma(q, fma(-d, q, 1.), q);
  q = fma(q, fma(-d, q, 1.), q);
  return static_cast<float>(static_cast<double>(g) * static_cast<double>(u) * q);
}

__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two values of y = round_DT(float32(silu(g) * u)), packed, the float32 rounding being that
// of the exact product: here in float64.
template <int DT>
__device__ __noinline__ uint32_t silu_mul2_exact(uint32_t gw, uint32_t uw) {
  float g[2], u[2];
  unpack2<DT>(gw, g[0], g[1]);
  unpack2<DT>(uw, u[0], u[1]);
  const bool zero0 = g[0] == 0.f || u[0] == 0.f, zero1 = g[1] == 0.f || u[1] == 0.f;
  if (zero0 && zero1) return pack2<DT>(g[0] * u[0], g[1] * u[1]);
  g[0] = zero0 ? g[0] * u[0] : silu_mul_exact(g[0], u[0]);
  g[1] = zero1 ? g[1] * u[1] : silu_mul_exact(g[1], u[1]);
  return pack2<DT>(g[0], g[1]);
}

// The same in float32, with `unsure` set where that does not settle the rounding.
//
// v = g * rcp(1 + 2^(-g log2 e)) * u.  In units of 2^-23 relative: the exponent's product and
// its constant are off by 0.61 |g| and ex2.approx by 2, both times s = e/(1 + e) with
// e = exp(-g); the sum, the two products and the ends of the interval below add 1/2 each and
// rcp.approx 1: 3 + (2 + 0.61 |g|) s.  For g > 0, s < 1/2 and |g| s < 0.28, so that is below
// 4.2; for g = -1, -2, -3, -4 it is 4.9, 5.8, 6.7 and 7.4 and grows by 0.61 from there on.  So
// v is within 4.25 + 0.83 max(-g, 0) of those units, and y is right wherever both ends of that
// interval round alike; about one bf16 value in 4000 is unsure.  (Over all gates and 512 ups each
// v was off by 0.66 of that at most.)  Where 1 / (1 + e) or v is below
// float32's normal range there is no such bound: see silu_deep and mx_tiny.
template <int DT>
__device__ __forceinline__ uint32_t silu_mul2(uint32_t gw, uint32_t uw, bool &unsure) {
  constexpr float kUnit = 1.0f / 8388608.0f;
  float g0, g1, u0, u1, p0, p1, d0, d1, v0, v1, e0, e1, l0, l1, h0, h1;
  unpack2<DT>(gw, g0, g1);
  unpack2<DT>(uw, u0, u1);
  mul2_rn(p0, p1, g0, g1, -1.4426950408889634f, -1.4426950408889634f);
  add2_rn(d0, d1, 1.0f, 1.0f, ex2_approx(p0), ex2_approx(p1));
  mul2_rn(v0, v1, g0, g1, rcp_approx(d0), rcp_approx(d1));
  mul2_rn(v0, v1, v0, v1, u0, u1);
  g0 = fminf(g0, 0.f);
  g1 = fminf(g1, 0.f);
  fma2_rn(e0, e1, g0, g1, 0.83f * kUnit, 0.83f * kUnit, -4.25f * kUnit, -4.25f * kUnit);  // minus the bound
  fma2_rn(l0, l1, v0, v1, e0, e1, v0, v1);
  fma2_rn(h0, h1, v0, v1, -e0, -e1, v0, v1);
  const uint32_t low = pack2<DT>(l0, l1), high = pack2<DT>(h0, h1);
  unsure = low != high;
  return low;
}

// Whether the larger half of `gates`, two bf16 gates, is below -87: 1 + e is above 2^126 then,
// its reciprocal may be taken for zero, and a large up brings the product back.  The negative
// gates furthest from zero (and NaN) have the largest bits as unsigned numbers.  (In fp16, ups
// end at 65504 and the product rounds to zero.)  The check takes 1.2 of 22 us of 4096 x 6144,
// taken here or within the loop over the pairs.
template <int DT>
__device__ __forceinline__ bool silu_deep(uint32_t gates) {
  return DT == I8L_BF16 && max(gates & 0xffffu, gates >> 16) > 0xc2aeu;
}

// Whether a block's largest y is so small that values below float32's normal range may decide
// its codes, from the magnitude's float32 bits.  In any other block such a value is far below
// half a step and only its sign is stored, which is right.  (fp16 has no such values: what is
// below float32's normal range rounds to zero.)
template <int DT>
__device__ __forceinline__ bool mx_tiny(uint32_t amax_bits) {
  return DT == I8L_BF16 && amax_bits < (127u - 110u) << 23;
}

// ------------------------------------------------------------------ flat quantisers

struct FlatArgs {
  const void *x;
  long long ldx;
  MxOut o;
  int rows, blocks;        // rows of this launch, 32-value blocks per row
  uint32_t vectors;        // rows * blocks * 4
  uint32_t pad_words;      // zero words below the last row
  FastDiv per_row;         // vectors per row
  int vec;                 // 1: 16-byte loads allowed, 2: 32-byte loads
  int q16;                 // 16-byte stores of codes allowed
  int rows_all;            // rows of the call
  int pdl;                 // launched with programmatic stream serialisation
};

// The plain quantiser's result may be a weight.  A product reads its weight before it waits for
// earlier kernels, and those let it start as soon as they have started themselves, so that it
// may run beside a kernel some launches before it.  From kWeightRows rows on, this one therefore
// lets nothing start at entry, and its stores have been performed when its CTAs are done; one
// thread's fence covers what its CTA wrote (8192 x 8192 26.3 us, with a fence in every thread
// 28.0, with no order at all 25.4).  Products wait before they read a weight of fewer rows,
// so that small batches of tokens keep the overlap (stand-in decoder, us a layer with and
// without the order for all: 8 tokens 25.8 and 24.7, 32 29.1 and 27.7, 128 40.3 and 40.8).
__device__ __forceinline__ void plain_begin(const FlatArgs &a) {
  if (a.rows_all < kWeightRows) pdl_launch_dependents();
}
// All threads of a CTA come here together.
__device__ __forceinline__ void plain_end(const FlatArgs &a) {
  if (a.pdl && a.rows_all >= kWeightRows) {
    __syncthreads();
    if (threadIdx.x == 0) __threadfence();
  }
}

// 32 bytes at a 32-byte boundary: a whole DRAM sector per lane.
__device__ __forceinline__ void ld_v8(const void *p, uint32_t *w) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void st_v8(void *p, const uint32_t *w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// A block of 32 16-bit values, two to a word.
__device__ __forceinline__ void load_block(const void *base, long long idx, int vec, uint32_t (&w)[16]) {
  const uint16_t *p = static_cast<const uint16_t *>(base) + idx;
  if (vec == 2) {
    ld_v8(p, w);
    ld_v8(p + 16, w + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = load8_raw(base, idx + 8 * i, vec);
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
  }
}

// Largest magnitude, as float32 bits, of 32 16-bit values.  The signed maximum of the bits is
// that of the positive values, the unsigned one that of the negative values where there are
// any; with the sign cleared, the larger of both is the block's (NaN and infinity included).
template <int DT>
__device__ __forceinline__ uint32_t mx_amax32(const uint32_t (&w)[16]) {
  uint32_t s = w[0], u = w[0];
#pragma unroll
  for (int i = 1; i < 15; i += 2) {
    s = __vimax3_s16x2(s, w[i], w[i + 1]);
    u = __vimax3_u16x2(u, w[i], w[i + 1]);
  }
  s = __vmaxs2(s, w[15]);
  u = __vmaxu2(u, w[15]);
  uint32_t m = __vmaxu2(s & 0x7fff7fffu, u & 0x7fff7fffu);
  m = max(m & 0xffffu, m >> 16);
  if constexpr (DT == I8L_BF16) return m << 16;
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
}

// Quantises a block that one thread holds, its largest magnitude given, and stores its codes
// and its scale.
template <int DT>
__device__ __forceinline__ void store_block(const MxOut &o, int q16, long long row, int block, int blocks,
                                            const uint32_t (&x)[16], uint32_t amax) {
  const uint32_t byte = mx_scale_byte(amax);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[8];
    unpack8<DT>(make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]), y);
    w[i] = byte == 255u ? 0u : mx_pack8(y, mx_inv_scale(byte));
  }
  uint8_t *q = o.q + row * o.ldq + block * 16;
  if (q16) {
    *reinterpret_cast<uint4 *>(q) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t *>(q)[i] = w[i];
  }
  store_sf(o, row, block, blocks, byte);
}

// Four lanes a block, one vector of eight values a thread.  kSilu: x holds [gate | up] rows
// of 2K values.
template <int DT, bool kSilu>
__global__ void __launch_bounds__(kFlatThreads) mx_quant_kernel(const FlatArgs a) {
  static_assert(!kSilu || DT != I8L_F32, "SiLU takes 16-bit activations");
  if constexpr (kSilu)
    pdl_launch_dependents();
  else
    plain_begin(a);
  pdl_wait();
  const uint32_t id = blockIdx.x * kFlatThreads + threadIdx.x;
  const uint32_t row = a.per_row.div(id), vec = id - row * a.per_row.d;
  const bool in = id < a.vectors;
  const long long at = row * a.ldx + vec * 8u;
  uint32_t byte, w;
  if constexpr (DT == I8L_F32) {
    float y[8] = {};
    if (in) load8<DT>(a.x, at, a.vec, y);
    w = mx_quantise8(y, byte);
  } else {
    uint4 x = in ? load8_raw(a.x, at, a.vec) : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (kSilu) {
      const long long K = static_cast<long long>(a.blocks) * kMxBlock;
      const uint4 up = in ? load8_raw(a.x, at + K, a.vec) : make_uint4(0u, 0u, 0u, 0u);
      const uint4 gate = x;
      auto settle = [](uint32_t g, uint32_t u) {
        bool unsure;
        const uint32_t y = silu_mul2<DT>(g, u, unsure);
        return unsure ? silu_mul2_exact<DT>(g, u) : y;
      };
      x = make_uint4(settle(gate.x, up.x), settle(gate.y, up.y), settle(gate.z, up.z), settle(gate.w, up.w));
      const bool deep = silu_deep<DT>(__vmaxu2(__vmaxu2(gate.x, gate.y), __vmaxu2(gate.z, gate.w)));
      if (mx_tiny<DT>(mx_amax8<DT>(x)) || deep)
        x = make_uint4(silu_mul2_exact<DT>(gate.x, up.x), silu_mul2_exact<DT>(gate.y, up.y),
                       silu_mul2_exact<DT>(gate.z, up.z), silu_mul2_exact<DT>(gate.w, up.w));
    }
    w = mx_quantise8<DT>(x, byte);
  }
  if (in) {
    *reinterpret_cast<uint32_t *>(a.o.q + row * a.o.ldq + vec * 4u) = w;
    if ((threadIdx.x & 3) == 0) store_sf(a.o, row, static_cast<int>(vec >> 2), a.blocks, byte);
  } else if (id - a.vectors < a.pad_words) {
    zero_pad_word(a.o, a.rows, id - a.vectors);
  }
  if constexpr (!kSilu) plain_end(a);
}

// The flat quantisers for matrices that fill the GPU: one thread takes a whole block, so
// there is nothing to exchange, and addresses, the scale and the index arithmetic are shared
// by 32 values instead of 8.  The four-lanes-a-block kernel above was bound by instruction
// issue (77 % of the slots, 111 instructions per 8 values; 8192 x 8192 42.6 us), but
// spreads a small matrix over four times as many threads.
// Threads: 128 (4096 x 4096 7.6 us, with 64 9.7); with SiLU 64, as a CTA stays as long as the
// last of its warps that has unsure values (4096 x 6144 22 us, with 128 23, with 32 26).
template <bool kSilu>
constexpr int kBlockThreads = kSilu ? 64 : 128;

template <int DT, bool kSilu>
__device__ __forceinline__ void mx_block(const FlatArgs &a) {
  static_assert(DT != I8L_F32, "16-bit values");
  const uint32_t id = blockIdx.x * kBlockThreads<kSilu> + threadIdx.x;
  const uint32_t total = a.vectors >> 2;
  if (id >= total) {
    if (id - total < a.pad_words) zero_pad_word(a.o, a.rows, id - total);
    return;
  }
  const uint32_t row = a.per_row.div(id), block = id - row * a.per_row.d;
  const long long at = row * a.ldx + block * static_cast<long long>(kMxBlock);
  uint32_t x[16];
  load_block(a.x, at, a.vec, x);
  uint32_t amax;
  if constexpr (kSilu) {
    uint32_t up[16];
    load_block(a.x, at + static_cast<long long>(a.blocks) * kMxBlock, a.vec, up);
    // The unsure pairs are few: they are read again and done after all others, which keeps
    // the slow code out of the unrolled loop.
    uint32_t todo = 0u, most = 0u;
#pragma unroll
    for (int i = 0; i < 16; i += 2) most = __vimax3_u16x2(most, x[i], x[i + 1]);
    const bool deep = silu_deep<DT>(most);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      bool unsure;
      x[i] = silu_mul2<DT>(x[i], up[i], unsure);
      if (unsure) todo |= 1u << i;
    }
    if (deep) todo = 0xffffu;
    for (bool all = false;; all = true) {
      while (todo) {
        const int i = __ffs(todo) - 1;
        todo &= todo - 1;
        const uint16_t *g = static_cast<const uint16_t *>(a.x) + at + 2 * i;
        const uint16_t *u = g + static_cast<long long>(a.blocks) * kMxBlock;
        const uint32_t y = silu_mul2_exact<DT>(g[0] | (static_cast<uint32_t>(g[1]) << 16),
                                               u[0] | (static_cast<uint32_t>(u[1]) << 16));
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = j == i ? y : x[j];
      }
      amax = mx_amax32<DT>(x);
      if (all || !mx_tiny<DT>(amax)) break;
      // Zero rows, as padding has them, need no second look (4096 x 6144 zeros 101 us with it).
      uint32_t g[16], any_g = 0u, any_u = 0u;
      load_block(a.x, at, a.vec, g);
      load_block(a.x, at + static_cast<long long>(a.blocks) * kMxBlock, a.vec, up);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        any_g |= g[i];
        any_u |= up[i];
      }
      if (((any_g & 0x7fff7fffu) == 0u) || ((any_u & 0x7fff7fffu) == 0u)) break;
      todo = 0xffffu;
    }
  } else {
    amax = mx_amax32<DT>(x);
  }
  store_block<DT>(a.o, a.q16, row, static_cast<int>(block), a.blocks, x, amax);
}

template <int DT, bool kSilu>
__global__ void __launch_bounds__(kBlockThreads<kSilu>) mx_block_kernel(const FlatArgs a) {
  if constexpr (kSilu)
    pdl_launch_dependents();
  else
    plain_begin(a);
  pdl_wait();
  mx_block<DT, kSilu>(a);
  if constexpr (!kSilu) plain_end(a);
}

// ------------------------------------------------------------------ add + RMSNorm

struct MxNormArgs {
  const void *x;
  long long ldx;
  const void *res;
  long long ldr;
  const void *w;
  int w_dtype, w_vec;
  void *rout;
  long long ldro;
  MxOut o;
  int rows, K;
  double inv_k, eps;
  uint32_t pad_words;
  int vec;  // 1: 16-byte loads and stores allowed, 2: 32-byte ones
  int q16;  // 16-byte stores of codes allowed
};

// sum + x^2 in float64, which holds a float32's square exactly.  kFast: the float64 is put
// together from x's bits, an integer multiplication, as the conversion unit is slow (8192 rows of
// 4096 39.5 us with it, 38.8 so); infinities, NaN, zeros and values below float32's normal range
// come out as others, which plain_sum tells from the row's sum.
template <bool kFast>
__device__ __forceinline__ double add_square(double sum, float x) {
  const double d = kFast ? __longlong_as_double(static_cast<long long>(
                               static_cast<unsigned long long>(__float_as_uint(x) & 0x7fffffffu) * 0x20000000ull +
                               0x3800000000000000ull))
                         : static_cast<double>(x);
  return fma(d, d, sum);
}

// Whether a sum from add_square<true> is that of the values.  An infinity or NaN puts it above
// 2^255; the value that stands for a zero or a smaller one is below 2^-126, so that 2^18 of
// their squares change a sum from 2^-180 on by less than 2^-53 of it.
__device__ __forceinline__ bool plain_sum(double sum) { return sum > 0x1p-180 && sum < 0x1p255; }

// The sum of every thread's `sum`, for CTAs of at most eight warps.
__device__ __forceinline__ double cta_sum(double sum, double *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
  __syncthreads();
  double part[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) part[i] = i < static_cast<int>(blockDim.x >> 5) ? red[i] : 0.0;
  return ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
}

// float32(1 / sqrt(m)): an approximation and two Newton steps, within 2^-51 before the
// rounding, so that every thread of a row has it sooner than one could hand it round.
__device__ __forceinline__ float norm_factor(double m) {
  double r;
  asm("rsqrt.approx.ftz.f64 %0, %1;" : "=d"(r) : "d"(m));
  if (m >= 0x1p-1022 && m < 0x1p1023) {  // not zero, an infinity or NaN
    r = fma(0.5 * r, fma(-m * r, r, 1.), r);
    r = fma(0.5 * r, fma(-m * r, r, 1.), r);
  }
  return static_cast<float>(r);
}

// One row per CTA, the row in registers.  The squares are summed in float64 and
// 1/sqrt(mean + eps) is rounded once to float32, so the factor does not depend on the order of
// the sum.
template <int DT, int WDT, int NV>
__global__ void __launch_bounds__(256) mx_norm_quant_kernel(const MxNormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  using T = typename ActType<DT>::T;
  const long long row = blockIdx.x;
  if (row >= a.rows) {  // zero words of the scale tiles below the last row
    const long long i = (row - a.rows) * blockDim.x + threadIdx.x;
    if (i < a.pad_words) zero_pad_word(a.o, a.rows, i);
    return;
  }
  __shared__ double red[8];
  uint4 xr[NV], rr[NV];
  float h[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = col_of<8>(v);
    xr[v] = rr[v] = make_uint4(0u, 0u, 0u, 0u);
    if (col < a.K) {
      xr[v] = load8_raw(a.x, row * a.ldx + col, a.vec);
      if (a.res) rr[v] = load8_raw(a.res, row * a.ldr + col, a.vec);
    }
  }
  double ss = 0.0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    unpack8<DT>(xr[v], h[v]);
    const int col = col_of<8>(v);
    if (a.res) {
      float r[8];
      unpack8<DT>(rr[v], r);
#pragma unroll
      for (int i = 0; i < 8; i += 2) add2_rn(h[v][i], h[v][i + 1], h[v][i], h[v][i + 1], r[i], r[i + 1]);
      if (col < a.K) {
        T *p = static_cast<T *>(a.rout) + row * a.ldro + col;
        if (a.vec) {
          *reinterpret_cast<uint4 *>(p) = pack8<DT>(h[v]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] = ActType<DT>::from_f32(h[v][i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = add_square<false>(ss, h[v][i]);
  }
  ss = cta_sum(ss, red);
  const float rs = norm_factor(fma(ss, a.inv_k, a.eps));
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int col = col_of<8>(v);
    if (col < a.K) {
      float w[8];
      load_weight_vec<8>(a.w, WDT, col, a.w_vec != 0, w);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        float n0, n1;
        mul2_rn(n0, n1, h[v][i], h[v][i + 1], rs, rs);
        round2_through<WDT>(n0, n1);
        mul2_rn(h[v][i], h[v][i + 1], n0, n1, w[i], w[i + 1]);
      }
    }
    uint32_t byte;
    const uint32_t packed = mx_quantise8<DT>(pack8<DT>(h[v]), byte);
    if (col < a.K) {
      *reinterpret_cast<uint32_t *>(a.o.q + row * a.o.ldq + col / 2) = packed;
      if ((threadIdx.x & 3) == 0) store_sf(a.o, row, col / kMxBlock, a.K / kMxBlock, byte);
    }
  }
}

// The same for batches of many rows of up to 8192 values, with a whole block per thread: the
// reductions, the scale and the addresses are shared by 32 values.
template <int DT, int WDT>
__global__ void __launch_bounds__(256) mx_norm_block_kernel(const MxNormArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  using T = typename ActType<DT>::T;
  const long long row = blockIdx.x;
  if (row >= a.rows) {  // zero words of the scale tiles below the last row
    const long long i = (row - a.rows) * blockDim.x + threadIdx.x;
    if (i < a.pad_words) zero_pad_word(a.o, a.rows, i);
    return;
  }
  __shared__ double red[8];
  const int blocks = a.K / kMxBlock, block = static_cast<int>(threadIdx.x);
  const bool in = block < blocks;
  uint32_t x[16], r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = r[i] = 0u;
  if (in) {
    load_block(a.x, row * a.ldx + block * kMxBlock, a.vec, x);
    if (a.res) load_block(a.res, row * a.ldr + block * kMxBlock, a.vec, r);
  }
  float h[32];
  double ss = 0.0, ss1 = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    unpack2<DT>(x[i], h[2 * i], h[2 * i + 1]);
    if (a.res) {
      float r0, r1;
      unpack2<DT>(r[i], r0, r1);
      add2_rn(h[2 * i], h[2 * i + 1], h[2 * i], h[2 * i + 1], r0, r1);
      r[i] = pack2<DT>(h[2 * i], h[2 * i + 1]);
    }
    ss = add_square<true>(ss, h[2 * i]);
    ss1 = add_square<true>(ss1, h[2 * i + 1]);
  }
  if (in && a.res) {
    T *p = static_cast<T *>(a.rout) + row * a.ldro + block * kMxBlock;
    if (a.vec == 2) {
      st_v8(p, r);
      st_v8(p + 16, r + 8);
    } else if (a.vec) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        reinterpret_cast<uint4 *>(p)[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) p[i] = ActType<DT>::from_f32(h[i]);
    }
  }
  ss = cta_sum(ss + ss1, red);
  if (!plain_sum(ss)) {
    __syncthreads();  // `red` has been read
    ss = 0.0;
#pragma unroll
    for (int i = 0; i < 32; ++i) ss = add_square<false>(ss, h[i]);
    ss = cta_sum(ss, red);
  }
  if (!in) return;
  const float rs = norm_factor(fma(ss, a.inv_k, a.eps));
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    float w[8];
    load_weight_vec<8>(a.w, WDT, block * kMxBlock + 8 * v, a.w_vec != 0, w);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float n0, n1;
      mul2_rn(n0, n1, h[8 * v + i], h[8 * v + i + 1], rs, rs);
      round2_through<WDT>(n0, n1);
      mul2_rn(n0, n1, n0, n1, w[i], w[i + 1]);
      x[4 * v + i / 2] = pack2<DT>(n0, n1);
    }
  }
  store_block<DT>(a.o, a.q16, row, block, blocks, x, mx_amax32<DT>(x));
}

// ------------------------------------------------------------------ dequantisation

struct DeqArgs {
  const uint8_t *q;
  long long ldq;
  const uint8_t *sf;
  int ktiles;
  void *out;
  long long ldo;
  uint32_t blocks;  // in all
  FastDiv per_row;
  int vec;  // 32-byte stores allowed
  int q16;  // 16-byte loads of codes allowed
};

// One thread per block.
template <int DT>
__global__ void __launch_bounds__(kFlatThreads) mx_dequant_kernel(const DeqArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  using T = typename ActType<DT>::T;
  const uint32_t id = blockIdx.x * kFlatThreads + threadIdx.x;
  if (id >= a.blocks) return;
  const uint32_t row = a.per_row.div(id), block = id - row * a.per_row.d;
  const uint8_t *q = a.q + row * a.ldq + block * 16u;
  uint32_t w[4];
  if (a.q16) {
    const uint4 v = *reinterpret_cast<const uint4 *>(q);
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t *>(q)[i];
  }
  const float s = mx_scale_value(a.sf[sf_word_offset(row, static_cast<int>(block >> 2), a.ktiles) + (block & 3)]);
  T *out = static_cast<T *>(a.out) + row * a.ldo + block * static_cast<long long>(kMxBlock);
  constexpr int kWords = DT == I8L_F32 ? 8 : 4;  // of eight values
  uint32_t o[2 * kWords];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[8];
    mx_unpack8(w[i], v);
#pragma unroll
    for (int j = 0; j < 8; j += 2) mul2_rn(v[j], v[j + 1], v[j], v[j + 1], s, s);
    uint32_t *p = o + (i & 1) * kWords;
    if constexpr (DT == I8L_F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = __float_as_uint(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = pack2<DT>(v[2 * j], v[2 * j + 1]);
    }
    if (!a.vec) {
#pragma unroll
      for (int j = 0; j < 8; ++j) out[8 * i + j] = ActType<DT>::from_f32(v[j]);
    } else if (i & 1) {
#pragma unroll
      for (int j = 0; j < 2 * kWords; j += 8) st_v8(reinterpret_cast<uint32_t *>(out) + (i - 1) * kWords + j, o + j);
    }
  }
}

}  // namespace i8l

using namespace i8l;

namespace {

int finish_launch(cudaError_t err, const char *what) {
  if (err != cudaSuccess) return cuda_error(err, what);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? I8L_OK : cuda_error(e, what);
}

// Shape and output checks that the quantisers share.
int check_mx(int32_t M, int32_t K, const void *q, int64_t ldq, const void *sf) {
  if (M < 0 || K < 0) return set_error(I8L_EINVAL, "negative size M=%d K=%d", M, K);
  if (K % kMxBlock) return set_error(I8L_ENOTSUP, "K=%d must be a multiple of 32 (whole blocks)", K);
  if (K > kMxMaxK) return set_error(I8L_ENOTSUP, "K=%d is above %d", K, kMxMaxK);
  if (M == 0 || K == 0) return I8L_OK;
  if (!q || !sf) return set_error(I8L_EINVAL, "NULL pointer argument");
  if (M > 1 && ldq < K / 2) return set_error(I8L_EINVAL, "packed row stride %lld < K/2", static_cast<long long>(ldq));
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(sf)) % 4 || ldq % 4)
    return set_error(I8L_ENOTSUP, "packed rows and scales must be 4-byte aligned");
  return I8L_OK;
}

int act_size(int dtype) { return dtype == I8L_F32 ? 4 : 2; }

bool vec_rows(const void *p, int64_t ld, int dtype) { return aligned16(p) && (ld * act_size(dtype)) % 16 == 0; }

// Rows of one launch of a flat kernel: the vector count stays below 2^31 with the padding
// words on top, in whole scale tiles.
int64_t flat_rows(int32_t K) {
  const int64_t rows = ((1LL << 30) / (K / 8)) & ~127LL;
  return std::max<int64_t>(rows, 128);
}

template <bool kSilu>
int run_flat(const void *x, int64_t ldx, int dtype, uint8_t *q, int64_t ldq, uint8_t *sf, int32_t M, int32_t K,
             void *stream, const char *what) {
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  const int blocks = K / kMxBlock, ktiles = (K + 127) / 128;
  const int64_t step = flat_rows(K);
  for (int64_t r0 = 0; r0 < M; r0 += step) {
    const int rows = static_cast<int>(std::min<int64_t>(step, M - r0));
    const int pad = (128 - rows % 128) % 128;
    FlatArgs a;
    a.x = static_cast<const uint8_t *>(x) + r0 * ldx * act_size(dtype);
    a.ldx = ldx;
    a.o = MxOut{q + r0 * ldq, ldq, sf + (r0 / 128) * ktiles * kSfTileBytes, ktiles};
    a.rows = rows;
    a.blocks = blocks;
    a.vectors = static_cast<uint32_t>(rows) * (blocks * 4u);
    a.pad_words = static_cast<uint32_t>(pad) * ktiles;
    a.vec = vec_rows(x, ldx, dtype) && (!kSilu || (static_cast<int64_t>(K) * act_size(dtype)) % 16 == 0) ? 1 : 0;
    a.q16 = aligned16(q) && ldq % 16 == 0 ? 1 : 0;
    a.rows_all = M;
    a.pdl = pdl_enabled() ? 1 : 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t err;
    // A thread per block from 256 blocks an SM on (SiLU: 512); with fewer, four lanes a block
    // finish sooner (us by threads and by lanes: 18944 blocks 1.69 and 1.63, 37888 1.79 and 1.91,
    // 151552 2.8 and 4.4; fp32 stays with four lanes, 8192 x 8192 46.7 us, the copy rate; SiLU
    // 37888 3.6 and 3.3, 56832 4.1 and 4.1, 75776 4.6 and 4.8).
    const int64_t total = a.vectors / 4;
    if (dtype != I8L_F32 && total >= (kSilu ? 512 : 256) * di.sms) {
      if (a.vec && reinterpret_cast<uintptr_t>(x) % 32 == 0 && (ldx * 2) % 32 == 0) a.vec = 2;
      a.per_row = FastDiv(blocks);
      constexpr int kThreads = kBlockThreads<kSilu>;
      const dim3 grid(static_cast<unsigned>((total + a.pad_words + kThreads - 1) / kThreads));
      if (dtype == I8L_BF16)
        err = launch(mx_block_kernel<I8L_BF16, kSilu>, grid, dim3(kThreads), 0, s, 1, a);
      else
        err = launch(mx_block_kernel<I8L_F16, kSilu>, grid, dim3(kThreads), 0, s, 1, a);
    } else {
      a.per_row = FastDiv(blocks * 4u);
      const int64_t work = static_cast<int64_t>(a.vectors) + a.pad_words;
      const dim3 grid(static_cast<unsigned>((work + kFlatThreads - 1) / kFlatThreads));
      if (dtype == I8L_BF16)
        err = launch(mx_quant_kernel<I8L_BF16, kSilu>, grid, dim3(kFlatThreads), 0, s, 1, a);
      else if (dtype == I8L_F16)
        err = launch(mx_quant_kernel<I8L_F16, kSilu>, grid, dim3(kFlatThreads), 0, s, 1, a);
      else if constexpr (!kSilu)
        err = launch(mx_quant_kernel<I8L_F32, false>, grid, dim3(kFlatThreads), 0, s, 1, a);
      else
        err = cudaErrorInvalidValue;
    }
    if (int e = finish_launch(err, what)) return e;
  }
  return I8L_OK;
}

}  // namespace

extern "C" size_t i8l_mxfp4_scale_bytes(int32_t rows, int32_t K) {
  if (rows <= 0 || K <= 0) return 0;
  return static_cast<size_t>((static_cast<int64_t>(rows) + 127) / 128) * ((static_cast<int64_t>(K) + 127) / 128) *
         kSfTileBytes;
}

extern "C" int i8l_quant_mxfp4(const void *x, int64_t ldx, int32_t dtype, uint8_t *q, int64_t ldq, uint8_t *scale,
                               int32_t M, int32_t K, void *stream) {
  if (dtype < I8L_BF16 || dtype > I8L_F32)
    return set_error(I8L_ENOTSUP, "dtype code %d not supported (bf16, fp16 or fp32)", dtype);
  if (int e = check_mx(M, K, q, ldq, scale)) return e;
  if (M == 0 || K == 0) return I8L_OK;
  if (!x) return set_error(I8L_EINVAL, "NULL pointer argument");
  if (M == 1) ldx = std::max<int64_t>(ldx, K);  // a single row's stride is never used
  if (ldx < K) return set_error(I8L_EINVAL, "row stride smaller than K");
  return run_flat<false>(x, ldx, dtype, q, ldq, scale, M, K, stream, "quant_mxfp4 launch");
}

extern "C" int i8l_silu_mul_quant_mxfp4(const void *gate_up, int64_t ld, int32_t act_dtype, uint8_t *q, int64_t ldq,
                                        uint8_t *scale, int32_t M, int32_t I, void *stream) {
  if (act_dtype != I8L_BF16 && act_dtype != I8L_F16)
    return set_error(I8L_ENOTSUP, "activation dtype code %d not supported (bf16 or fp16)", act_dtype);
  if (int e = check_mx(M, I, q, ldq, scale)) return e;
  if (M == 0 || I == 0) return I8L_OK;
  if (!gate_up) return set_error(I8L_EINVAL, "NULL pointer argument");
  if (M == 1) ld = std::max<int64_t>(ld, 2LL * I);
  if (ld < 2LL * I) return set_error(I8L_EINVAL, "row stride too small");
  return run_flat<true>(gate_up, ld, act_dtype, q, ldq, scale, M, I, stream, "silu_mul_quant_mxfp4 launch");
}

extern "C" int i8l_add_rmsnorm_quant_mxfp4(const void *x, int64_t ldx, const void *residual, int64_t ldr,
                                           const void *weight, int32_t act_dtype, int32_t w_dtype, uint8_t *q,
                                           int64_t ldq, uint8_t *scale, void *rout, int64_t ldro, int32_t M,
                                           int32_t K, double eps, void *stream) {
  if (act_dtype != I8L_BF16 && act_dtype != I8L_F16)
    return set_error(I8L_ENOTSUP, "activation dtype code %d not supported (bf16 or fp16)", act_dtype);
  if (w_dtype < I8L_BF16 || w_dtype > I8L_F32)
    return set_error(I8L_ENOTSUP, "weight dtype code %d not supported", w_dtype);
  if (int e = check_mx(M, K, q, ldq, scale)) return e;
  if (M == 0 || K == 0) return I8L_OK;
  if (!x || !weight) return set_error(I8L_EINVAL, "NULL pointer argument");
  if ((residual == nullptr) != (rout == nullptr))
    return set_error(I8L_EINVAL, "residual and residual_out must be given together");
  if (M == 1) {
    ldx = std::max<int64_t>(ldx, K);
    ldr = std::max<int64_t>(ldr, K);
  }
  if (ldx < K || (residual && (ldr < K || ldro < K))) return set_error(I8L_EINVAL, "row stride smaller than K");
  const bool vec = vec_rows(x, ldx, act_dtype) &&
                   (!residual || (vec_rows(residual, ldr, act_dtype) && vec_rows(rout, ldro, act_dtype)));
  RowShape rs;
  if (!row_shape(K, 8, &rs)) return set_error(I8L_ENOTSUP, "row of %d values is too long", K);
  const int ktiles = (K + 127) / 128;
  // a CTA per row and, behind them, a few per 128-value tile of K for the zero scales
  if (M > INT32_MAX - 128 * ktiles) return set_error(I8L_ENOTSUP, "M=%d rows are too many", M);
  MxNormArgs a;
  a.x = x;
  a.ldx = ldx;
  a.res = residual;
  a.ldr = ldr;
  a.w = weight;
  a.w_dtype = w_dtype;
  a.w_vec = aligned16(weight) ? 1 : 0;
  a.rout = rout;
  a.ldro = ldro;
  a.o = MxOut{q, ldq, scale, ktiles};
  a.rows = M;
  a.K = K;
  a.inv_k = 1.0 / K;
  a.eps = eps;
  a.pad_words = static_cast<uint32_t>((128 - M % 128) % 128) * ktiles;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  a.vec = vec ? 1 : 0;
  a.q16 = aligned16(q) && ldq % 16 == 0 ? 1 : 0;
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  // A block per thread from 384 of them an SM on; fewer finish sooner spread over four times the
  // threads, and so do rows that leave half a warp idle (us by block and by vector: 592 rows of
  // 2048 3.6 and 3.5, 888 4.1 and 4.4; 296 rows of 4096 3.8 and 3.9, 1184 7.2 and 8.0; 8192
  // rows of 512 10.5 and 9.3, of 1024 12.2 and 13.7).
  const bool blocks = static_cast<int64_t>(M) * K >= 384 * kMxBlock * static_cast<int64_t>(di.sms) && K >= 1024 && K <= 8192;
  if (blocks && vec) {
    auto wide = [](const void *p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 32 == 0 && ld % 16 == 0; };
    if (wide(x, ldx) && (!residual || (wide(residual, ldr) && wide(rout, ldro)))) a.vec = 2;
  }
  const int nv = rs.nv, th = blocks ? (K / kMxBlock + 31) / 32 * 32 : rs.threads;
  const dim3 grid(static_cast<unsigned>(M) + (a.pad_words + th - 1) / th);
  cudaError_t err = cudaSuccess;
#define I8L_MX_NORM(ADT, WDTV)                                                                          \
  if (blocks) {                                                                                         \
    err = launch(mx_norm_block_kernel<ADT, WDTV>, grid, dim3(th), 0, s, 1, a);                          \
  } else {                                                                                              \
    I8L_DISPATCH_NV(nv, (err = launch(mx_norm_quant_kernel<ADT, WDTV, NV>, grid, dim3(th), 0, s, 1, a))) \
  }
#define I8L_MX_NORM_W(ADT)                                              \
  if (w_dtype == I8L_BF16) { I8L_MX_NORM(ADT, I8L_BF16) }               \
  else if (w_dtype == I8L_F16) { I8L_MX_NORM(ADT, I8L_F16) }            \
  else { I8L_MX_NORM(ADT, I8L_F32) }
  if (act_dtype == I8L_BF16) {
    I8L_MX_NORM_W(I8L_BF16)
  } else {
    I8L_MX_NORM_W(I8L_F16)
  }
#undef I8L_MX_NORM_W
#undef I8L_MX_NORM
  return finish_launch(err, "add_rmsnorm_quant_mxfp4 launch");
}

extern "C" int i8l_dequant_mxfp4(const uint8_t *q, int64_t ldq, const uint8_t *scale, void *out, int64_t ldo,
                                 int32_t out_dtype, int32_t M, int32_t K, void *stream) {
  if (out_dtype < I8L_BF16 || out_dtype > I8L_F32)
    return set_error(I8L_ENOTSUP, "dtype code %d not supported (bf16, fp16 or fp32)", out_dtype);
  if (int e = check_mx(M, K, q, ldq, scale)) return e;
  if (M == 0 || K == 0) return I8L_OK;
  if (!out) return set_error(I8L_EINVAL, "NULL pointer argument");
  if (ldo < K) return set_error(I8L_EINVAL, "row stride smaller than K");
  const int ktiles = (K + 127) / 128;
  const int64_t step = flat_rows(K);
  for (int64_t r0 = 0; r0 < M; r0 += step) {
    const int rows = static_cast<int>(std::min<int64_t>(step, M - r0));
    DeqArgs a;
    a.q = q + r0 * ldq;
    a.ldq = ldq;
    a.sf = scale + (r0 / 128) * ktiles * kSfTileBytes;
    a.ktiles = ktiles;
    a.out = static_cast<uint8_t *>(out) + r0 * ldo * act_size(out_dtype);
    a.ldo = ldo;
    a.blocks = static_cast<uint32_t>(rows) * (K / kMxBlock);
    a.per_row = FastDiv(K / kMxBlock);
    a.vec = reinterpret_cast<uintptr_t>(out) % 32 == 0 && (ldo * act_size(out_dtype)) % 32 == 0 ? 1 : 0;
    a.q16 = aligned16(q) && ldq % 16 == 0 ? 1 : 0;
    const dim3 grid((a.blocks + kFlatThreads - 1) / kFlatThreads);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t err;
    if (out_dtype == I8L_BF16)
      err = launch(mx_dequant_kernel<I8L_BF16>, grid, dim3(kFlatThreads), 0, s, 1, a);
    else if (out_dtype == I8L_F16)
      err = launch(mx_dequant_kernel<I8L_F16>, grid, dim3(kFlatThreads), 0, s, 1, a);
    else
      err = launch(mx_dequant_kernel<I8L_F32>, grid, dim3(kFlatThreads), 0, s, 1, a);
    if (int e = finish_launch(err, "dequant_mxfp4 launch")) return e;
  }
  return I8L_OK;
}
