// RMSNorm of every query and key head of a qkv product and the rotation by the token's
// position, in one pass, for sm_100a.  For a head x of `dim` values with norm weight w
// (one weight for queries, one for keys):
//     n = x / sqrt(mean(x^2) + eps) * w
//     y = n with its first `rot` values rotated in pairs (a, b) by the position's angles:
//         a' = a cos - b sin,  b' = b cos + a sin
// where pair i is (n[i], n[i + rot/2]), or (n[2i], n[2i + 1]) when interleaved.  Everything
// is float32 between the load and one rounding at the store.
//
// A group of lanes holds one head in registers, each lane two chunks of eight values that
// are rotated with one another: values 8c.. and rot/2 + 8c.. (or, interleaved, two chunks in
// a row), so that a lane needs eight angles and nothing from another lane but the sum of
// squares, a butterfly over the group.  (With neighbouring values in a lane and the pairs'
// other halves shuffled, the kernel took 42 us where it then took 36, 8192 tokens x 40 heads of
// 128.)  In a large batch a group of lanes takes two neighbouring heads of one token, which
// share its angles, and has the next two on their way meanwhile: with the latency of position,
// then angles, and 31 % occupancy the kernel waited for loads a third of its time without.
// It reads and writes each value once: 32 us is 80 % of the measured copy rate.  Heads a group
// and CTAs an SM otherwise (4096 tokens; 15.6 us so): 2 and 6 16.3, 2 and 7 18.9, 3 and 5 17.6,
// 4 and 4 16.6, 1 and 8 26.9; a CTA per four heads without the loop 17.5.
#include <algorithm>
#include <limits>

#include "common.cuh"
#include "internal.h"
#include "mxfp4.cuh"
#include "rows.cuh"

namespace i8l {

constexpr int kQkThreads = 128;
constexpr int kQkHeads = 2;  // heads per group in a large batch
constexpr int kQkCtas = 5;   // CTAs per SM then

// bf16 heads whose squares float32 may not hold: their sum overflows (values from about 2^60
// on), or the mean and eps leave less than this, beside which squares below 2^-149 could count.
// Their values are multiplied by a power of two first, and eps by its square, which n does not
// see: 2^-72 leaves 256 squares below 2^120, and what it takes out of float32's range is nothing
// in n; 2^96 brings the least value to 2^-37 and leaves the largest square, and eps, below 2^104.
// (fp16 values have no such squares.)  Looking for such heads takes 0.3 of 16.6 us of 4096 tokens
// x 40 heads of 128 in bf16, 17.9 where every head is one; by lane groups, without the warp's
// vote, 17.4.
constexpr float kLeastMean = 0x1p-100f;
constexpr float kInf = std::numeric_limits<float>::infinity();

struct QkArgs {
  const void *qkv;
  long long ld;
  const void *wq, *wk;
  int w_dtype;
  const void *positions;
  int pos64;
  const void *cos_sin;
  int cs_dtype;
  long long max_pos;
  void *q;
  long long ldq;  // elements between tokens; heads are `dim` apart
  void *k;
  long long ldk;
  int tokens, heads, kv_heads, dim, rot;
  int parts;       // groups per token, each with up to P heads
  uint32_t groups;  // tokens * parts, below 2^31
  FastDiv per_token;  // parts
  float eps, inv_dim;
  int interleaved;
  int w_vec, cs_vec;
};

// G lanes per head (a power of two, G * 16 >= dim), P heads per group.  With kLoop the grid
// covers the GPU once and a CTA goes on to further groups.  In place is fine: a lane stores the
// elements that it alone loaded.
template <int DT, int G, int P, bool kLoop>
__global__ void __launch_bounds__(kQkThreads, kLoop ? kQkCtas : 1) qk_norm_rope_kernel(const QkArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  using T = typename ActType<DT>::T;
  constexpr uint32_t kGroups = kQkThreads / G;
  const int lane = threadIdx.x % G;
  const int half = a.rot / 2;
  // The lane's chunks begin at c0 and c1; what lies behind the rotated values follows in order.
  const bool split = !a.interleaved && lane < a.rot / 16;
  const int c0 = split ? 8 * lane : 16 * lane, c1 = split ? half + 8 * lane : 16 * lane + 8;
  const bool has0 = c0 < a.dim, has1 = c1 < a.dim;
  const int all = a.heads + a.kv_heads;

  // A group's values and its token's position.
  struct Group {
    uint4 raw[P][2];
    long long token, pos;
    int head0;  // `all` behind the last group
  } next;
  auto fetch = [&](uint32_t id) {
    const bool in = id < a.groups;
    next.token = in ? a.per_token.div(id) : 0;
    next.head0 = in ? static_cast<int>(id - static_cast<uint32_t>(next.token) * a.parts) * P : all;
    const T *src = static_cast<const T *>(a.qkv) + next.token * a.ld + static_cast<long long>(next.head0) * a.dim;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const bool here = next.head0 + i < all;
      next.raw[i][0] = here && has0 ? *reinterpret_cast<const uint4 *>(src + i * a.dim + c0) : make_uint4(0u, 0u, 0u, 0u);
      next.raw[i][1] = here && has1 ? *reinterpret_cast<const uint4 *>(src + i * a.dim + c1) : make_uint4(0u, 0u, 0u, 0u);
    }
    next.pos = 0;
    if (in)
      next.pos = a.pos64 ? static_cast<const long long *>(a.positions)[next.token]
                         : static_cast<const int *>(a.positions)[next.token];
  };

  uint32_t id = blockIdx.x * kGroups + threadIdx.x / G;
  fetch(id);
  float w[16] = {};
  int loaded = -1;  // which weight `w` holds: 0 queries, 1 keys
  // Whole warps take part in every turn, for their shuffles.
  for (uint32_t first = blockIdx.x * kGroups; first < a.groups; first += gridDim.x * kGroups) {
    const Group now = next;
    // A position outside the table has no angles: the token's heads come out as NaN.
    const bool known = a.rot == 0 || (now.pos >= 0 && now.pos < a.max_pos);
    // Angles 8 lane .. 8 lane + 7; those past the last are none.
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cs[i] = 1.f;
      sn[i] = 0.f;
    }
    if (has0 && now.head0 < all && known && 8 * lane < half) {
      const uint8_t *table = static_cast<const uint8_t *>(a.cos_sin) + now.pos * a.rot * (a.cs_dtype == I8L_F32 ? 4 : 2);
      if (8 * lane + 8 <= half) {
        load_weight_vec<8>(table, a.cs_dtype, 8 * lane, a.cs_vec != 0, cs);
        load_weight_vec<8>(table, a.cs_dtype, half + 8 * lane, a.cs_vec != 0, sn);
      } else {  // interleaved, and four angles left
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          cs[i] = load_weight(table, a.cs_dtype, 8 * lane + i);
          sn[i] = load_weight(table, a.cs_dtype, half + 8 * lane + i);
        }
      }
    }

    if (kLoop) {  // the next group is on its way while this one is computed
      id += gridDim.x * kGroups;
      if (first + gridDim.x * kGroups < a.groups) fetch(id);
    }
#pragma unroll
    for (int turn = 0; turn < P; ++turn) {
      const int head = now.head0 + turn;
      const bool here = head < all;
      const int key = head >= a.heads ? 1 : 0;
      if (here && key != loaded) {
        const void *weight = key ? a.wk : a.wq;
        if (has0) load_weight_vec<8>(weight, a.w_dtype, c0, a.w_vec != 0, *reinterpret_cast<float(*)[8]>(w));
        if (has1) load_weight_vec<8>(weight, a.w_dtype, c1, a.w_vec != 0, *reinterpret_cast<float(*)[8]>(w + 8));
      }
      if (here) loaded = key;
      float x[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        unpack2<DT>(now.raw[turn][h].x, x[8 * h], x[8 * h + 1]);
        unpack2<DT>(now.raw[turn][h].y, x[8 * h + 2], x[8 * h + 3]);
        unpack2<DT>(now.raw[turn][h].z, x[8 * h + 4], x[8 * h + 5]);
        unpack2<DT>(now.raw[turn][h].w, x[8 * h + 6], x[8 * h + 7]);
      }
      auto squares = [&] {  // of the group's head
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) fma2_rn(s0, s1, x[i], x[i + 1], x[i], x[i + 1], s0, s1);
        float ss = s0 + s1;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, G);
        return ss;
      };
      float mean = fmaf(squares(), a.inv_dim, a.eps);
      if constexpr (DT == I8L_BF16) {
        const bool plain = mean >= kLeastMean && mean < kInf;
        if (!__all_sync(0xffffffffu, plain)) {
          const float s = plain ? 1.f : (mean < kLeastMean ? 0x1p96f : 0x1p-72f);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] *= s;
          mean = fmaf(squares(), a.inv_dim, a.eps * s * s);
        }
      }
      float rs = rsqrtf(mean);
      if (!known) rs = __int_as_float(0x7fc00000);
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        mul2_rn(x[i], x[i + 1], x[i], x[i + 1], rs, rs);
        mul2_rn(x[i], x[i + 1], x[i], x[i + 1], w[i], w[i + 1]);
      }
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x[2 * i], v = x[2 * i + 1];
          x[2 * i] = fmaf(u, cs[i], -(v * sn[i]));
          x[2 * i + 1] = fmaf(v, cs[i], u * sn[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          float t0, t1, r0, r1;
          mul2_rn(t0, t1, x[8 + i], x[9 + i], -sn[i], -sn[i + 1]);
          mul2_rn(r0, r1, x[i], x[i + 1], sn[i], sn[i + 1]);
          fma2_rn(x[i], x[i + 1], x[i], x[i + 1], cs[i], cs[i + 1], t0, t1);
          fma2_rn(x[8 + i], x[9 + i], x[8 + i], x[9 + i], cs[i], cs[i + 1], r0, r1);
        }
      }
      if (here) {
        T *dst = key ? static_cast<T *>(a.k) + now.token * a.ldk + static_cast<long long>(head - a.heads) * a.dim
                     : static_cast<T *>(a.q) + now.token * a.ldq + static_cast<long long>(head) * a.dim;
        if (has0)
          *reinterpret_cast<uint4 *>(dst + c0) = make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]),
                                                            pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7]));
        if (has1)
          *reinterpret_cast<uint4 *>(dst + c1) = make_uint4(pack2<DT>(x[8], x[9]), pack2<DT>(x[10], x[11]),
                                                            pack2<DT>(x[12], x[13]), pack2<DT>(x[14], x[15]));
      }
    }
    if (!kLoop) break;
  }
}

}  // namespace i8l

using namespace i8l;

namespace {

template <int DT, int P, bool kLoop>
cudaError_t launch_qk(const QkArgs &a, int lanes, int sms, cudaStream_t s) {
  const unsigned per_block = kQkThreads / lanes;
  unsigned ctas = (a.groups + per_block - 1) / per_block;
  if (kLoop) ctas = std::min<unsigned>(ctas, kQkCtas * sms);
  const dim3 grid(ctas);
  switch (lanes) {
    case 1: return launch(qk_norm_rope_kernel<DT, 1, P, kLoop>, grid, dim3(kQkThreads), 0, s, 1, a);
    case 2: return launch(qk_norm_rope_kernel<DT, 2, P, kLoop>, grid, dim3(kQkThreads), 0, s, 1, a);
    case 4: return launch(qk_norm_rope_kernel<DT, 4, P, kLoop>, grid, dim3(kQkThreads), 0, s, 1, a);
    case 8: return launch(qk_norm_rope_kernel<DT, 8, P, kLoop>, grid, dim3(kQkThreads), 0, s, 1, a);
    default: return launch(qk_norm_rope_kernel<DT, 16, P, kLoop>, grid, dim3(kQkThreads), 0, s, 1, a);
  }
}

}  // namespace

extern "C" int i8l_qk_norm_rope(const void *qkv, int64_t ld, int32_t act_dtype, const void *q_weight,
                                const void *k_weight, int32_t w_dtype, float eps, const void *positions,
                                int32_t positions_i64, const void *cos_sin, int32_t cs_dtype, int64_t max_pos,
                                void *q_out, int64_t ldq, void *k_out, int64_t ldk, int32_t tokens, int32_t heads,
                                int32_t kv_heads, int32_t head_dim, int32_t rot_dim, int32_t interleaved,
                                void *stream) {
  if (act_dtype != I8L_BF16 && act_dtype != I8L_F16)
    return set_error(I8L_ENOTSUP, "activation dtype code %d not supported (bf16 or fp16)", act_dtype);
  if (w_dtype < I8L_BF16 || w_dtype > I8L_F32 || cs_dtype < I8L_BF16 || cs_dtype > I8L_F32)
    return set_error(I8L_ENOTSUP, "weight dtype code %d or angle dtype code %d not supported", w_dtype, cs_dtype);
  if (tokens < 0 || heads < 0 || kv_heads < 0 || head_dim <= 0 || rot_dim < 0 || rot_dim > head_dim || max_pos < 0)
    return set_error(I8L_EINVAL, "bad size tokens=%d heads=%d kv_heads=%d head_dim=%d rot_dim=%d", tokens, heads,
                     kv_heads, head_dim, rot_dim);
  if (head_dim % 8 || head_dim > 256)
    return set_error(I8L_ENOTSUP, "head_dim %d must be a multiple of 8, at most 256", head_dim);
  if (rot_dim % (interleaved ? 8 : 16))
    return set_error(I8L_ENOTSUP, "rot_dim %d must be a multiple of %d", rot_dim, interleaved ? 8 : 16);
  const int64_t all = static_cast<int64_t>(heads) + kv_heads;
  if (all > INT32_MAX / 256) return set_error(I8L_ENOTSUP, "too many heads: %lld", static_cast<long long>(all));
  if (tokens == 0 || all == 0) return I8L_OK;
  if (!qkv || !positions || (rot_dim && !cos_sin) || (heads && (!q_weight || !q_out)) ||
      (kv_heads && (!k_weight || !k_out)))
    return set_error(I8L_EINVAL, "NULL pointer argument");
  if (tokens == 1) {  // distances between tokens are never used
    ld = all * head_dim;
    ldq = static_cast<int64_t>(heads) * head_dim;
    ldk = static_cast<int64_t>(kv_heads) * head_dim;
  }
  if (ld < all * head_dim || (heads && ldq < static_cast<int64_t>(heads) * head_dim) ||
      (kv_heads && ldk < static_cast<int64_t>(kv_heads) * head_dim))
    return set_error(I8L_EINVAL, "row stride smaller than the heads of a token");
  if (!aligned16(qkv) || ld % 8 || (heads && (!aligned16(q_out) || ldq % 8)) ||
      (kv_heads && (!aligned16(k_out) || ldk % 8)))
    return set_error(I8L_ENOTSUP, "qkv, q_out and k_out rows must be 16-byte aligned");
  QkArgs a{};
  a.qkv = qkv;
  a.ld = ld;
  a.wq = q_weight;
  a.wk = k_weight;
  a.w_dtype = w_dtype;
  a.positions = positions;
  a.pos64 = positions_i64 ? 1 : 0;
  a.cos_sin = cos_sin;
  a.cs_dtype = cs_dtype;
  a.max_pos = max_pos;
  a.q = q_out;
  a.ldq = ldq;
  a.k = k_out;
  a.ldk = ldk;
  a.tokens = tokens;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = head_dim;
  a.rot = rot_dim;
  a.eps = eps;
  a.inv_dim = 1.0f / static_cast<float>(head_dim);
  a.interleaved = interleaved ? 1 : 0;
  a.w_vec = (!heads || aligned16(q_weight)) && (!kv_heads || aligned16(k_weight)) ? 1 : 0;
  // every row of angles, and its second half, starts on 16 bytes
  a.cs_vec = aligned16(cos_sin) && (rot_dim / 2 * (cs_dtype == I8L_F32 ? 4 : 2)) % 16 == 0 ? 1 : 0;
  int lanes = 1;
  while (lanes * 16 < head_dim) lanes *= 2;
  // One head per group and no loop until the lanes fill half of the SMs' threads (us by one head
  // and by the loop, 40 heads of 128: 256 tokens 3.0 and 3.1, 512 4.2 and 3.5; 24 heads of 64:
  // 1536 tokens 3.4 and 3.5, 3000 5.2 and 5.1; 24 heads of 256: 256 3.2 and 3.3, 1024 6.8 and 6.1).
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  const bool many = static_cast<int64_t>(tokens) * all * lanes > 1024LL * di.sms;
  a.parts = static_cast<int>(many ? (all + kQkHeads - 1) / kQkHeads : all);
  const int64_t groups = static_cast<int64_t>(tokens) * a.parts;
  if (groups > INT32_MAX - kQkThreads)
    return set_error(I8L_ENOTSUP, "%d tokens x %lld heads is too large", tokens, static_cast<long long>(all));
  a.groups = static_cast<uint32_t>(groups);
  a.per_token = FastDiv(static_cast<uint32_t>(a.parts));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  if (act_dtype == I8L_BF16)
    err = many ? launch_qk<I8L_BF16, kQkHeads, true>(a, lanes, di.sms, s) : launch_qk<I8L_BF16, 1, false>(a, lanes, di.sms, s);
  else
    err = many ? launch_qk<I8L_F16, kQkHeads, true>(a, lanes, di.sms, s) : launch_qk<I8L_F16, 1, false>(a, lanes, di.sms, s);
  if (err != cudaSuccess) return cuda_error(err, "qk_norm_rope launch");
  err = cudaGetLastError();
  return err == cudaSuccess ? I8L_OK : cuda_error(err, "qk_norm_rope launch");
}
