// RMSNorm of every query and key head of a qkv product and the rotation by the token's
// position, in one pass, for sm_100a.  For a head x of `dim` values with norm weight w
// (one weight for queries, one for keys):
//     n = x / sqrt(mean(x^2) + eps) * w
//     y = n with its first `rot` values rotated in pairs (a, b) by the position's angles:
//         a' = a cos - b sin,  b' = b cos + a sin
// where pair i is (n[i], n[i + rot/2]), or (n[2i], n[2i + 1]) when interleaved.  Everything
// is float32 between the load and one rounding at the store.
//
// A group of lanes, eight values each, holds one head in registers: the sum of squares is
// a butterfly over the group, and the other half of a pair comes from another lane of the
// group by a shuffle.  A group takes up to P neighbouring heads of one token: their loads are
// all in flight together, and the token's angles are read once for them.  The kernel reads
// and writes each value once and is bound by HBM.
#include <algorithm>

#include "common.cuh"
#include "internal.h"
#include "mxfp4.cuh"
#include "rows.cuh"

namespace i8l {

constexpr int kQkThreads = 256;

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

// G lanes per head (a power of two, G * 8 >= dim), P heads per group; kFull: every value is
// rotated (rot == dim).  In place is fine: a lane stores the
// elements that it alone loaded, after every exchange within its head.
template <int DT, int G, int P, bool kFull>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kernel(const QkArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  using T = typename ActType<DT>::T;
  const uint32_t group = blockIdx.x * (kQkThreads / G) + threadIdx.x / G;
  const int lane = threadIdx.x % G;
  const bool live = group < a.groups;
  const long long token = live ? a.per_token.div(group) : 0;
  const int part = live ? static_cast<int>(group - static_cast<uint32_t>(token) * a.parts) : 0;
  const int c0 = lane * 8;
  const bool mine = live && c0 < a.dim;
  const int all = a.heads + a.kv_heads, head0 = part * P;
  const T *src = static_cast<const T *>(a.qkv) + token * a.ld + static_cast<long long>(head0) * a.dim + c0;
  uint4 raw[P];
#pragma unroll
  for (int i = 0; i < P; ++i)
    raw[i] = mine && head0 + i < all ? *reinterpret_cast<const uint4 *>(src + i * a.dim) : make_uint4(0u, 0u, 0u, 0u);
  const int half = a.rot / 2;

  long long pos = 0;
  if (live)
    pos = a.pos64 ? static_cast<const long long *>(a.positions)[token] : static_cast<const int *>(a.positions)[token];
  // A position outside the table has no angles: the token's heads come out as NaN.
  const bool known = a.rot == 0 || (pos >= 0 && pos < a.max_pos);
  const bool turns = mine && c0 < a.rot;
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
  }
  if (turns && known) {
    const uint8_t *table = static_cast<const uint8_t *>(a.cos_sin) +
                           pos * a.rot * (a.cs_dtype == I8L_F32 ? 4 : 2);
    if (a.interleaved) {
      // pairs (2i, 2i + 1): both take angle i
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = load_weight(table, a.cs_dtype, (c0 + i) / 2);
        sn[i] = load_weight(table, a.cs_dtype, half + (c0 + i) / 2);
      }
    } else {
      const int j = c0 < half ? c0 : c0 - half;
      load_weight_vec<8>(table, a.cs_dtype, j, a.cs_vec != 0, cs);
      load_weight_vec<8>(table, a.cs_dtype, half + j, a.cs_vec != 0, sn);
    }
    // the first value of a pair subtracts its partner's share
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (a.interleaved ? i % 2 == 0 : c0 < half) sn[i] = -sn[i];
  }
  // The lane of this group that holds the other values of this lane's pairs.
  const int partner = !a.interleaved && turns ? (c0 < half ? lane + half / 8 : lane - half / 8) : lane;

  float w[8] = {};
  int loaded = -1;  // which weight `w` holds: 0 queries, 1 keys
#pragma unroll
  for (int turn = 0; turn < P; ++turn) {
    const int head = head0 + turn;
    const bool here = mine && head < all;
    const int key = head >= a.heads ? 1 : 0;
    if (here && key != loaded) load_weight_vec<8>(key ? a.wk : a.wq, a.w_dtype, c0, a.w_vec != 0, w);
    loaded = key;
    float x[8];
    unpack2<DT>(raw[turn].x, x[0], x[1]);
    unpack2<DT>(raw[turn].y, x[2], x[3]);
    unpack2<DT>(raw[turn].z, x[4], x[5]);
    unpack2<DT>(raw[turn].w, x[6], x[7]);
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) fma2_rn(s0, s1, x[i], x[i + 1], x[i], x[i + 1], s0, s1);
    float ss = s0 + s1;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, G);
    float rs = rsqrtf(fmaf(ss, a.inv_dim, a.eps));
    if (!known) rs = __int_as_float(0x7fc00000);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      mul2_rn(x[i], x[i + 1], x[i], x[i + 1], rs, rs);
      mul2_rn(x[i], x[i + 1], x[i], x[i + 1], w[i], w[i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float o0, o1, t0, t1;
      if (a.interleaved) {
        o0 = x[i + 1];
        o1 = x[i];
      } else {
        o0 = __shfl_sync(0xffffffffu, x[i], partner, G);
        o1 = __shfl_sync(0xffffffffu, x[i + 1], partner, G);
      }
      mul2_rn(t0, t1, o0, o1, sn[i], sn[i + 1]);
      fma2_rn(t0, t1, x[i], x[i + 1], cs[i], cs[i + 1], t0, t1);
      y[i] = kFull || turns ? t0 : x[i];
      y[i + 1] = kFull || turns ? t1 : x[i + 1];
    }
    if (here) {
      T *dst = key ? static_cast<T *>(a.k) + token * a.ldk + static_cast<long long>(head - a.heads) * a.dim
                   : static_cast<T *>(a.q) + token * a.ldq + static_cast<long long>(head) * a.dim;
      *reinterpret_cast<uint4 *>(dst + c0) =
          make_uint4(pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]), pack2<DT>(y[4], y[5]), pack2<DT>(y[6], y[7]));
    }
  }
}

}  // namespace i8l

using namespace i8l;

namespace {

template <int DT, int P, bool kFull>
cudaError_t launch_qk(const QkArgs &a, int lanes, cudaStream_t s) {
  const unsigned per_block = kQkThreads / lanes;
  const dim3 grid((a.groups + per_block - 1) / per_block);
  switch (lanes) {
    case 1: return launch(qk_norm_rope_kernel<DT, 1, P, kFull>, grid, dim3(kQkThreads), 0, s, 1, a);
    case 2: return launch(qk_norm_rope_kernel<DT, 2, P, kFull>, grid, dim3(kQkThreads), 0, s, 1, a);
    case 4: return launch(qk_norm_rope_kernel<DT, 4, P, kFull>, grid, dim3(kQkThreads), 0, s, 1, a);
    case 8: return launch(qk_norm_rope_kernel<DT, 8, P, kFull>, grid, dim3(kQkThreads), 0, s, 1, a);
    case 16: return launch(qk_norm_rope_kernel<DT, 16, P, kFull>, grid, dim3(kQkThreads), 0, s, 1, a);
    default: return launch(qk_norm_rope_kernel<DT, 32, P, kFull>, grid, dim3(kQkThreads), 0, s, 1, a);
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
  while (lanes * 8 < head_dim) lanes *= 2;
  // One head per group until the groups fill the SMs twice over, then four.
  DeviceInfo di;
  if (int e = device_info(&di)) return e;
  const bool four = static_cast<int64_t>(tokens) * all > 2LL * di.sms * (2048 / lanes);
  a.parts = static_cast<int>(four ? (all + 3) / 4 : all);
  const int64_t groups = static_cast<int64_t>(tokens) * a.parts;
  if (groups > INT32_MAX - kQkThreads)
    return set_error(I8L_ENOTSUP, "%d tokens x %lld heads is too large", tokens, static_cast<long long>(all));
  a.groups = static_cast<uint32_t>(groups);
  a.per_token = FastDiv(static_cast<uint32_t>(a.parts));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool full = rot_dim == head_dim;
  cudaError_t err;
  if (act_dtype == I8L_BF16)
    err = four ? (full ? launch_qk<I8L_BF16, 4, true>(a, lanes, s) : launch_qk<I8L_BF16, 4, false>(a, lanes, s))
               : launch_qk<I8L_BF16, 1, false>(a, lanes, s);
  else
    err = four ? (full ? launch_qk<I8L_F16, 4, true>(a, lanes, s) : launch_qk<I8L_F16, 4, false>(a, lanes, s))
               : launch_qk<I8L_F16, 1, false>(a, lanes, s);
  if (err != cudaSuccess) return cuda_error(err, "qk_norm_rope launch");
  err = cudaGetLastError();
  return err == cudaSuccess ? I8L_OK : cuda_error(err, "qk_norm_rope launch");
}
