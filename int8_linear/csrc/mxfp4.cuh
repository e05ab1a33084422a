// Microscaled 4-bit floating point (MXFP4) on the device: blocks of 32 consecutive
// values along K, each value in e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives),
// each block with one power-of-two scale in e8m0 (byte b stands for 2^(b - 127), 0xFF for
// NaN).
//
// Packed codes: row r at q + r*ldq bytes, value 2j in the low and 2j+1 in the high nibble
// of byte j.  Scales: tiles of 128 rows x 4 blocks (128 values), 512 bytes each, the tiles
// of one 128-row group in order of K:
//     byte of (row r, block b) = ((r/128) * ceil(K/128) + b/4) * 512
//                                + (r%32)*16 + ((r/32)%4)*4 + b%4
// which is the order that a tensor core takes block scales in, so the GEMM copies a tile
// as it lies.  Bytes of a tile past the last row or the last block are 0.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace i8l {

constexpr int kMxBlock = 32;       // values per scale
constexpr int kSfTileBytes = 512;  // 128 rows x 4 blocks
constexpr int kMxMaxK = 1 << 26;   // 128 rows of eight-value vectors fit a 31-bit index

// Whether a product reads its weight before the kernels before it are done: under programmatic
// launch not where quant_mxfp4, for as few rows, may still be writing it.
constexpr int kWeightRows = 128;
inline bool mx_weight_early(int rows) { return rows >= kWeightRows || !pdl_enabled(); }

// Byte offset of the word that holds the scales of blocks 4*kt .. 4*kt+3 of a row.
__host__ __device__ __forceinline__ long long sf_word_offset(long long row, int kt, int ktiles) {
  return ((row >> 7) * ktiles + kt) * kSfTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// Scale byte of a block whose largest magnitude has the float32 bits `amax` (sign clear):
// 2^(floor(log2 amax) - 2), so the largest value lands in [4, 8) and saturates at 6; at
// least 2^-127.  The float's biased exponent minus 2 is that byte, subnormals included
// (their exponent field 0 clamps to 0).  Infinity or NaN anywhere makes the block NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  const uint32_t e = amax >> 23;
  return e == 255u ? 255u : (e < 2u ? 0u : e - 2u);
}

// 2^(127 - byte): the factor that takes a block's values into e2m1 range, exact for the
// bytes mx_scale_byte gives (0..252).  A product with it is exact too, or too small to
// round to anything but zero.
__device__ __forceinline__ float mx_inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// 2^(byte - 127), NaN for 0xFF; 2^-127 is a float32 subnormal.
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : (byte == 0u ? 0x00400000u : byte << 23));
}

// Unsigned division by a constant of the launch: floor(n / d) for n < 2^31 as a multiply
// and a shift (the round-up method: m = ceil(2^(32+s) / d), s = ceil(log2 d)).
struct FastDiv {
  uint32_t d, m, s;
  __host__ FastDiv(uint32_t div = 1) : d(div), m(0), s(0) {
    while ((1ull << s) < d) ++s;
    m = static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    const uint32_t t = __umulhi(n, m);
    return (t + n) >> s;  // t + n < 2^32 for n < 2^31
  }
};

// ---------------------------------------------------------------- tensor cores
// tcgen05.mma.kind::mxf4 multiplies packed e2m1 tiles, 64 values (32 bytes) of K per
// instruction, with the scales of both operands in TMEM: a scale tile (128 rows x 4 blocks)
// is four columns there, row r in lane r % 32 of column r / 32, its four blocks in the four
// bytes; an instruction takes two of the bytes, chosen by the scale ids of its descriptor.

// The issuing warp runs these converged, all lanes with the same operands, and `elected` set
// in one lane: the operands then stay in uniform registers, where one lane in a branch of
// its own would move each of them there before every instruction (measured on the pair
// tiles at 4096 x 12288 x 2048: 66 us so, 72 us that way; and 53 us, from 58, with the
// instructions of half a stage in one piece).

// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}

// Instruction descriptor: e2m1 x e2m1 with e8m0 scales, both K-major; `sf_id` (0 or 2) is
// the first of the two scale bytes, the same in both operands.
__host__ __device__ constexpr uint32_t idesc_mxf4(int m, int n, int sf_id) {
  return (static_cast<uint32_t>(sf_id) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (1u << 23) | (static_cast<uint32_t>(m >> 4) << 24) | (static_cast<uint32_t>(sf_id) << 29);
}

// Shared-memory descriptors: the low word holds the address, the high word what does not
// change: 128-byte swizzled K-major rows in groups of eight 1024 bytes apart (as
// sw128_kmajor_desc), or a scale tile's 32 rows of 16 bytes, no swizzle, eight 128 bytes apart.
constexpr uint32_t kSw128DescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kSfDescHi = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }

// Half a stage (128 values of K) of a CTA pair in one piece, so that nothing but the tensor
// instructions and a few additions stands between them: the scale tiles of the first operand
// (one) and the second (two, and a third where `third` is set in the elected lane), then two
// MMAs, or one without `second`.  alo .. ylo: low descriptor words; sfx, sfy: TMEM columns
// that the scales go to; sfy_at: that of the tile's first row.
__device__ __forceinline__ void pair_half_stage(uint32_t elected, uint32_t third, uint32_t d, uint32_t alo,
                                                uint32_t blo, uint32_t xlo, uint32_t ylo, uint32_t sfx, uint32_t sfy,
                                                uint32_t sfy_at, uint32_t idesc0, uint32_t idesc2, uint32_t accumulate,
                                                bool second) {
  asm volatile(
      "{\n\t.reg .pred p, q, r;\n\t"
      ".reg .b64 u, v;\n\t.reg .b32 t, w;\n\t"
      "setp.ne.b32 p, %9, 0;\n\tsetp.ne.b32 q, %10, 0;\n\tsetp.ne.b32 r, %11, 0;\n\t"
      "mov.b64 u, {%3, %13};\n\t"
      "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%5], u;\n\t"
      "mov.b64 u, {%4, %13};\n\t"
      "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%6], u;\n\t"
      "add.u32 t, %6, 4;\n\tadd.u32 w, %4, 64;\n\tmov.b64 u, {w, %13};\n\t"
      "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [t], u;\n\t"
      "add.u32 t, %6, 8;\n\tadd.u32 w, %4, 128;\n\tmov.b64 u, {w, %13};\n\t"
      "@r tcgen05.cp.cta_group::2.32x128b.warpx4 [t], u;\n\t"
      "mov.b64 u, {%1, %12};\n\tmov.b64 v, {%2, %12};\n\t"
      "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], u, v, %8, [%5], [%7], p;\n\t}" ::"r"(d),
      "r"(alo), "r"(blo), "r"(xlo), "r"(ylo), "r"(sfx), "r"(sfy), "r"(sfy_at), "r"(idesc0), "r"(accumulate),
      "r"(elected), "r"(third), "r"(kSw128DescHi), "r"(kSfDescHi)
      : "memory");
  if (second)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        ".reg .b64 u, v;\n\t.reg .b32 t, w;\n\t"
        "setp.ne.b32 q, %6, 0;\n\tsetp.eq.u32 p, 0, 0;\n\t"
        "add.u32 t, %1, 2;\n\tadd.u32 w, %2, 2;\n\tmov.b64 u, {t, %7};\n\tmov.b64 v, {w, %7};\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], u, v, %5, [%3], [%4], p;\n\t}" ::"r"(d),
        "r"(alo), "r"(blo), "r"(sfx), "r"(sfy_at), "r"(idesc2), "r"(elected), "r"(kSw128DescHi)
        : "memory");
}

// The same for one CTA, whose second operand lies in one 128-row scale group.
__device__ __forceinline__ void single_half_stage(uint32_t elected, uint32_t d, uint32_t alo, uint32_t blo,
                                                  uint32_t xlo, uint32_t ylo, uint32_t sfx, uint32_t sfy,
                                                  uint32_t idesc0, uint32_t idesc2, uint32_t accumulate, bool second) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      ".reg .b64 u, v;\n\t"
      "setp.ne.b32 p, %8, 0;\n\tsetp.ne.b32 q, %9, 0;\n\t"
      "mov.b64 u, {%3, %11};\n\t"
      "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%5], u;\n\t"
      "mov.b64 u, {%4, %11};\n\t"
      "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%6], u;\n\t"
      "mov.b64 u, {%1, %10};\n\tmov.b64 v, {%2, %10};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], u, v, %7, [%5], [%6], p;\n\t}" ::"r"(d),
      "r"(alo), "r"(blo), "r"(xlo), "r"(ylo), "r"(sfx), "r"(sfy), "r"(idesc0), "r"(accumulate), "r"(elected),
      "r"(kSw128DescHi), "r"(kSfDescHi)
      : "memory");
  if (second)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        ".reg .b64 u, v;\n\t.reg .b32 t, w;\n\t"
        "setp.ne.b32 q, %6, 0;\n\tsetp.eq.u32 p, 0, 0;\n\t"
        "add.u32 t, %1, 2;\n\tadd.u32 w, %2, 2;\n\tmov.b64 u, {t, %7};\n\tmov.b64 v, {w, %7};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], u, v, %5, [%3], [%4], p;\n\t}" ::"r"(d),
        "r"(alo), "r"(blo), "r"(sfx), "r"(sfy), "r"(idesc2), "r"(elected), "r"(kSw128DescHi)
        : "memory");
}

// TMA loads (as tma_load_2d_pair and tma_load_2d) and the arming of their barriers, likewise
// from a converged warp with one elected lane.
__device__ __forceinline__ void tma_load_2d_pair_elected(uint32_t elected, uint32_t dst, const void *map,
                                                         uint32_t bar_cluster, int32_t x, int32_t y, uint64_t policy) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "l"(policy), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d_elected(uint32_t elected, uint32_t dst, const void *map, uint32_t bar,
                                                    int32_t x, int32_t y, uint64_t policy) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "l"(policy), "r"(elected)
      : "memory");
}
__device__ __forceinline__ void mbar_expect_tx_elected(uint32_t elected, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes), "r"(elected)
      : "memory");
}

// Arrive once when every tcgen05 operation this thread issued so far has completed: on this
// CTA's mbarrier (its shared-memory address), or with kPair on those at the same offset in both CTAs of the pair.
template <bool kPair>
__device__ __forceinline__ void mma_commit_elected(uint32_t elected, uint32_t bar) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::
            "r"(bar),
        "h"(static_cast<uint16_t>(0x3)), "r"(elected)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
        "r"(elected)
        : "memory");
}

// Two fused multiply-adds in one instruction, each rounded as fmaf rounds.
__device__ __forceinline__ void fma2_rn(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0,
                                        float c1) {
  asm("{\n.reg .b64 ra, rb, rc, rd;\n"
      "mov.b64 ra, {%2, %3};\n"
      "mov.b64 rb, {%4, %5};\n"
      "mov.b64 rc, {%6, %7};\n"
      "fma.rn.f32x2 rd, ra, rb, rc;\n"
      "mov.b64 {%0, %1}, rd;\n}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

// Eight values times `inv`, rounded to e2m1 (nearest, ties to even, saturating), packed
// with the first value in the lowest nibble.
__device__ __forceinline__ uint32_t mx_pack8(const float (&y)[8], float inv) {
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) mul2_rn(p[i], p[i + 1], y[i], y[i + 1], inv, inv);
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(p[0]), "f"(p[1]), "f"(p[2]), "f"(p[3]), "f"(p[4]), "f"(p[5]), "f"(p[6]), "f"(p[7]));
  return w;
}

// Eight packed e2m1 codes as floats (exact).
__device__ __forceinline__ void mx_unpack8(uint32_t w, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Largest float32 magnitude, as bits, of eight values: NaN and infinity compare above
// every finite value, which a float maximum would not do for NaN.
__device__ __forceinline__ uint32_t mx_amax8(const float (&y)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
  return m;
}

// One lane's eight values of a block shared by four neighbouring lanes: the scale from the
// four lanes' maximum, then this lane's four packed bytes (zero codes in a NaN block).
// Every lane of the warp takes part; lanes without values pass zeros.
__device__ __forceinline__ uint32_t mx_quantise8(const float (&y)[8], uint32_t &byte) {
  uint32_t m = mx_amax8(y);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  byte = mx_scale_byte(m);
  return byte == 255u ? 0u : mx_pack8(y, mx_inv_scale(byte));
}

// Two 16-bit values as floats.
template <int DT>
__device__ __forceinline__ void unpack2(uint32_t w, float &v0, float &v1) {
  if constexpr (DT == I8L_BF16) {
    v0 = __uint_as_float(w << 16);
    v1 = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
    v0 = f.x;
    v1 = f.y;
  }
}

// Rounds two floats to the 16-bit type and packs them, v0 low.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float v0, float v1) {
  uint32_t p;
  if constexpr (DT == I8L_BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(v1), "f"(v0));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(v1), "f"(v0));
  return p;
}

// The same for eight bf16 or fp16 values as they lie in memory.  16-bit floats of one sign
// are ordered as their bits are, NaN and infinity last, so the maximum is taken two at a
// time on the bits.
template <int DT>
__device__ __forceinline__ uint32_t mx_amax8(const uint4 &w) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  uint32_t m = __vmaxu2(__vmaxu2(w.x & kAbs, w.y & kAbs), __vmaxu2(w.z & kAbs, w.w & kAbs));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
  m = max(m & 0xffffu, m >> 16);
  if constexpr (DT == I8L_BF16) return m << 16;
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
}

template <int DT>
__device__ __forceinline__ uint32_t mx_quantise8(const uint4 &w, uint32_t &byte) {
  byte = mx_scale_byte(mx_amax8<DT>(w));
  float y[8];
  unpack2<DT>(w.x, y[0], y[1]);
  unpack2<DT>(w.y, y[2], y[3]);
  unpack2<DT>(w.z, y[4], y[5]);
  unpack2<DT>(w.w, y[6], y[7]);
  return byte == 255u ? 0u : mx_pack8(y, mx_inv_scale(byte));
}

}  // namespace i8l
