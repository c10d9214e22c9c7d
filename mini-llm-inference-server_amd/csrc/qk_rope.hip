// RMSNorm of each query and key head with the rotary embedding in the same pass, and the append of the keys and values:
//   y = x rsqrt(mean(x^2) + eps) w,  out[d] = y[d] cos[d] + rotate_half(y)[d] sin[d],  rotate_half(y) = cat(-y[half:], y[:half])
// in fp32 from the 16-bit x, w, cos and sin to one rounding at the end (as torch expressions each step would round).
// Also the rotation alone into a 4-bit pool, which rounds as kv_append.hip's does.
//
// A row (token, head) of Dh elements belongs to Dh / 16 consecutive lanes, padded to a power of two: each holds 16 bytes
// of the first half and their partners of the second, so the rotation stays in the lane and the sum of squares takes a
// few lane exchanges.  Bound by the launch for a decode step (32 tokens, 32 and 8 heads of 128 dims, into a 16-bit pool: 3.5
// us), by memory for prompts: 4 x 2049 tokens without a pool, 172 MB, 28 us (6.1 TB/s).
#include "kv_common.h"

namespace mllm {
namespace {

enum Dest { kRows = 0, kPool16 = 1, kPoolFp8 = 2, kPoolFp4 = 3 };  // where the keys go: a tensor, or a pool

struct QkArgs {
  const char *q, *k, *v;  // strides in bytes: batch, token, head
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_st, v_sh;
  const char *cos, *sin;
  int64_t cs_sb, cs_st;
  const char *wq, *wk;
  float eps;
  char* q_out;
  int64_t qo_sb, qo_st, qo_sh;
  char* k_out;  // kRows
  int64_t ko_sb, ko_st, ko_sh;
  Fp4Pool kp, vp;  // pools (codes alone for 16-bit and fp8 ones)
  float k_inv, v_inv;
  int64_t num_slots;
  const int64_t* slots;
  unsigned tokens, T;  // all tokens; tokens of a batch entry
  int H, Hkv, dh, chunks, lanes_log2, bs;
};

template <typename T>
__device__ __forceinline__ void floats8(const Chunk& c, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = to_f32<T>(c.e[e]);
}

template <typename T, int DEST, bool NORM>
__global__ __launch_bounds__(256) void qk_rope_kernel(const QkArgs a) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  const unsigned rows = (unsigned)(a.H + (DEST == kRows ? a.Hkv : 2 * a.Hkv));
  const unsigned r = i >> a.lanes_log2, t = r / rows;
  const int row = (int)(r - t * rows), j = (int)(i & ((1u << a.lanes_log2) - 1));
  if (t >= a.tokens) return;
  const bool active = j < a.chunks;  // lanes past the row's chunks only take part in the exchanges
  const unsigned b = DEST == kRows ? t / a.T : 0, n = DEST == kRows ? t - b * a.T : t;
  const int half = a.dh;  // bytes of half a row
  const int lo = 16 * j;
  const bool is_q = row < a.H, is_v = row >= a.H + a.Hkv;
  const int h = is_q ? row : (is_v ? row - a.H - a.Hkv : row - a.H);
  int64_t slot = 0;
  if (DEST != kRows && !is_q) {
    slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) return;  // the whole row's lanes
  }
  const char* src = is_q ? a.q + b * a.q_sb + n * a.q_st + h * a.q_sh
                         : (is_v ? a.v + n * a.v_st + h * a.v_sh : a.k + b * a.k_sb + n * a.k_st + h * a.k_sh);
  Chunk x1, x2;
  x1.v = x2.v = u32x4{0, 0, 0, 0};
  if (active) {
    x1.v = ld16(src + lo);
    x2.v = ld16(src + half + lo);
  }
  if (!is_v) {
    const int at = active ? lo : 0;
    const char* cr = a.cos + b * a.cs_sb + n * a.cs_st + at;
    const char* sr = a.sin + b * a.cs_sb + n * a.cs_st + at;
    Chunk c1, c2, s1, s2;
    c1.v = ld16(cr);
    c2.v = ld16(cr + half);
    s1.v = ld16(sr);
    s2.v = ld16(sr + half);
    if constexpr (NORM) {
      float y1[8], y2[8], w1[8], w2[8];
      floats8<T>(x1, y1);
      floats8<T>(x2, y2);
      const char* w = (is_q ? a.wq : a.wk) + at;
      Chunk wc1, wc2;
      wc1.v = ld16(w);
      wc2.v = ld16(w + half);
      floats8<T>(wc1, w1);
      floats8<T>(wc2, w2);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += y1[e] * y1[e] + y2[e] * y2[e];
      for (int off = 1 << a.lanes_log2 >> 1; off > 0; off >>= 1) ss += __shfl_xor(ss, off, 64);
      const float rs = rsqrtf(ss / (float)a.dh + a.eps);
      float o1[8], o2[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = y1[e] * rs * w1[e], q = y2[e] * rs * w2[e];
        o1[e] = p * to_f32<T>(c1.e[e]) - q * to_f32<T>(s1.e[e]);
        o2[e] = q * to_f32<T>(c2.e[e]) + p * to_f32<T>(s2.e[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x1.v[e] = pack2<T>(o1[2 * e], o1[2 * e + 1]);
        x2.v[e] = pack2<T>(o2[2 * e], o2[2 * e + 1]);
      }
    } else {
      Chunk o1, o2;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o1.e[e] = rot1<T>(x1.e[e], c1.e[e], -to_f32<T>(x2.e[e]), s1.e[e]);
        o2.e[e] = rot1<T>(x2.e[e], c2.e[e], to_f32<T>(x1.e[e]), s2.e[e]);
      }
      x1 = o1;
      x2 = o2;
    }
  }
  if (is_q || DEST == kRows) {
    if (!active) return;
    char* dst = is_q ? a.q_out + b * a.qo_sb + n * a.qo_st + h * a.qo_sh : a.k_out + b * a.ko_sb + n * a.ko_st + h * a.ko_sh;
    st16(dst + lo, x1.v);
    st16(dst + half + lo, x2.v);
    return;
  }
  const Fp4Pool pool = is_v ? a.vp : a.kp;
  const int64_t prow = slot * a.Hkv + h;
  if constexpr (DEST == kPool16) {
    if (!active) return;
    char* dst = pool.codes + prow * 2 * half;
    st16(dst + lo, x1.v);
    st16(dst + half + lo, x2.v);
  } else if constexpr (DEST == kPoolFp8) {
    if (!active) return;
    const float inv = is_v ? a.v_inv : a.k_inv;
    char* dst = pool.codes + prow * half;
    st8(dst + lo / 2, quant8<T>(x1.v, inv));
    st8(dst + half / 2 + lo / 2, quant8<T>(x2.v, inv));
  } else {  // four lanes hold a block of 32 dims in either half (the chunks are a multiple of four)
    const uint32_t e1 = block_exp<T>(x1.v), e2 = block_exp<T>(x2.v);
    if (!active) return;
    char* dst = pool.codes + prow * (half / 2);
    *reinterpret_cast<uint32_t*>(dst + lo / 4) = fp4x8_from<T>(x1.v, e8m0_to_f32(e1));
    *reinterpret_cast<uint32_t*>(dst + half / 4 + lo / 4) = fp4x8_from<T>(x2.v, e8m0_to_f32(e2));
    if ((j & 3) == 0) {
      const int nblk = a.dh / kFp4Block, blk1 = j >> 2, blk2 = nblk / 2 + blk1;
      pool.scales[is_v ? v_scale_at(slot, h, blk1, a.Hkv, nblk, a.bs) : k_scale_at(slot, h, blk1, a.Hkv, nblk)] = (uint8_t)e1;
      pool.scales[is_v ? v_scale_at(slot, h, blk2, a.Hkv, nblk, a.bs) : k_scale_at(slot, h, blk2, a.Hkv, nblk)] = (uint8_t)e2;
    }
  }
}

int launch_qk(const std::string& fn, const QkArgs& in, int dtype, int dest, hipStream_t st) {
  QkArgs a = in;
  a.chunks = a.dh / 16;
  a.lanes_log2 = 0;
  while ((1 << a.lanes_log2) < a.chunks) ++a.lanes_log2;
  const int64_t rows = a.H + (dest == kRows ? 1 : 2) * (int64_t)a.Hkv;
  const int64_t per = 256 >> a.lanes_log2;  // rows per workgroup
  const int64_t groups = ((int64_t)a.tokens * rows + per - 1) / per;
  MLLM_REQUIRE(groups <= kMaxGroups256, MLLM_ERR_UNSUPPORTED, fn + ": too many tokens");
  auto launch = [&](auto tag) {
    using T = decltype(tag);
    const unsigned grid = (unsigned)groups;
    if (!a.wq)
      qk_rope_kernel<T, kPoolFp4, false><<<grid, 256, 0, st>>>(a);
    else if (dest == kRows)
      qk_rope_kernel<T, kRows, true><<<grid, 256, 0, st>>>(a);
    else if (dest == kPool16)
      qk_rope_kernel<T, kPool16, true><<<grid, 256, 0, st>>>(a);
    else if (dest == kPoolFp8)
      qk_rope_kernel<T, kPoolFp8, true><<<grid, 256, 0, st>>>(a);
    else
      qk_rope_kernel<T, kPoolFp4, true><<<grid, 256, 0, st>>>(a);
  };
  if (dtype == MLLM_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return check_launch(fn.c_str());
}

int check_qk(const std::string& fn, int32_t dtype, int64_t tokens, int32_t H, int32_t Hkv, int32_t dh, float eps) {
  MLLM_REQUIRE(dtype == MLLM_DTYPE_BF16 || dtype == MLLM_DTYPE_F16, MLLM_ERR_UNSUPPORTED,
               fn + ": dtype must be bfloat16 or float16");
  MLLM_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && H > 0 && Hkv > 0 && dh > 0 && H < (1 << 20) && Hkv < (1 << 20),
               MLLM_ERR_INVALID, fn + ": bad sizes");
  MLLM_REQUIRE(dh % 16 == 0 && dh <= 1024, MLLM_ERR_UNSUPPORTED, fn + ": head_dim must be a multiple of 16, at most 1024");
  MLLM_REQUIRE(eps >= 0.f, MLLM_ERR_INVALID, fn + ": eps must not be negative");
  return MLLM_OK;
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_qk_norm_rope_kv_append(const mllm_rope_append* r, const void* q_norm, const void* k_norm, float eps,
                                           void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_qk_norm_rope_kv_append";
  MLLM_REQUIRE(r, MLLM_ERR_INVALID, fn + ": null arguments");
  const int rc = check_qk(fn, r->dtype, r->num_tokens, r->num_heads, r->num_kv_heads, r->head_dim, eps);
  if (rc != MLLM_OK) return rc;
  MLLM_REQUIRE(known_pool(r->pool), MLLM_ERR_INVALID, fn + ": unknown pool type");
  const bool fp4 = r->pool == MLLM_POOL_FP4, scaled = fp4 || r->pool == MLLM_POOL_FP8_BLOCKS;
  MLLM_REQUIRE(!fp4 || r->head_dim % 64 == 0, MLLM_ERR_UNSUPPORTED, fn + ": head_dim must be a multiple of 64 for a 4-bit pool");
  MLLM_REQUIRE(!q_norm == !k_norm && (q_norm || scaled), MLLM_ERR_INVALID,
               fn + ": q_norm and k_norm go together (without them, 8-bit pools with block scales and 4-bit pools only)");
  MLLM_REQUIRE(r->num_blocks >= 0 && r->block_size > 0, MLLM_ERR_INVALID, fn + ": bad pool sizes");
  MLLM_REQUIRE(r->pool != MLLM_POOL_FP8 || (r->k_scale > 0.f && r->v_scale > 0.f && r->k_scale < INFINITY && r->v_scale < INFINITY),
               MLLM_ERR_INVALID, fn + ": scales must be positive and finite");
  if (r->num_tokens == 0) return MLLM_OK;
  MLLM_REQUIRE(r->q && r->k && r->v && r->cos && r->sin && r->q_out && r->k_cache && r->v_cache && r->slot_mapping &&
                   (!scaled || (r->k_scales && r->v_scales)),
               MLLM_ERR_INVALID, fn + ": null pointer");
  const uintptr_t ptrs = (uintptr_t)r->q | (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)r->cos | (uintptr_t)r->sin |
                         (uintptr_t)r->q_out | (uintptr_t)r->k_cache | (uintptr_t)r->v_cache | (uintptr_t)q_norm | (uintptr_t)k_norm;
  const int64_t strides = r->q_stride_tok | r->q_stride_head | r->k_stride_tok | r->k_stride_head | r->v_stride_tok |
                          r->v_stride_head | r->cs_stride_tok | r->q_out_stride_tok | r->q_out_stride_head;
  MLLM_REQUIRE(ptrs % 16 == 0 && strides % 8 == 0, MLLM_ERR_UNSUPPORTED, fn + ": rows must be 16-byte aligned");
  if (r->pool == MLLM_POOL_FP8_BLOCKS) return rope_append_fp8_blocks(fn, *r, q_norm, k_norm, eps, stream);
  QkArgs a{};
  a.q = (const char*)r->q, a.q_st = 2 * r->q_stride_tok, a.q_sh = 2 * r->q_stride_head;
  a.k = (const char*)r->k, a.k_st = 2 * r->k_stride_tok, a.k_sh = 2 * r->k_stride_head;
  a.v = (const char*)r->v, a.v_st = 2 * r->v_stride_tok, a.v_sh = 2 * r->v_stride_head;
  a.cos = (const char*)r->cos, a.sin = (const char*)r->sin, a.cs_st = 2 * r->cs_stride_tok;
  a.wq = (const char*)q_norm, a.wk = (const char*)k_norm, a.eps = eps;
  a.q_out = (char*)r->q_out, a.qo_st = 2 * r->q_out_stride_tok, a.qo_sh = 2 * r->q_out_stride_head;
  a.kp = {(char*)r->k_cache, (uint8_t*)r->k_scales};
  a.vp = {(char*)r->v_cache, (uint8_t*)r->v_scales};
  if (r->pool == MLLM_POOL_FP8) a.k_inv = 1.f / r->k_scale, a.v_inv = 1.f / r->v_scale;
  a.num_slots = r->num_blocks * r->block_size;
  a.slots = r->slot_mapping;
  a.tokens = a.T = (unsigned)r->num_tokens;
  a.H = r->num_heads, a.Hkv = r->num_kv_heads, a.dh = r->head_dim, a.bs = r->block_size;
  return launch_qk(fn, a, r->dtype, r->pool == MLLM_POOL_16BIT ? kPool16 : (fp4 ? kPoolFp4 : kPoolFp8),
                   reinterpret_cast<hipStream_t>(stream));
}

extern "C" int mllm_qk_norm_rope(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb,
                                 int64_t k_sh, int64_t k_st, const void* cos, const void* sin, int64_t cs_sb,
                                 int64_t cs_st, const void* q_norm, const void* k_norm, float eps, int32_t batch,
                                 int32_t seq, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                                 void* q_out, void* k_out, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_qk_norm_rope";
  MLLM_REQUIRE(batch >= 0 && seq >= 0, MLLM_ERR_INVALID, fn + ": bad sizes");
  const int rc = check_qk(fn, dtype, (int64_t)batch * seq, num_heads, num_kv_heads, head_dim, eps);
  if (rc != MLLM_OK) return rc;
  if (batch == 0 || seq == 0) return MLLM_OK;
  MLLM_REQUIRE(q && k && cos && sin && q_norm && k_norm && q_out && k_out, MLLM_ERR_INVALID, fn + ": null pointer");
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_norm | (uintptr_t)k_norm |
                         (uintptr_t)q_out | (uintptr_t)k_out;
  MLLM_REQUIRE(ptrs % 16 == 0 && (q_sb | q_sh | q_st | k_sb | k_sh | k_st | cs_sb | cs_st) % 8 == 0, MLLM_ERR_UNSUPPORTED,
               fn + ": rows must be 16-byte aligned");
  QkArgs a{};
  a.q = (const char*)q, a.q_sb = 2 * q_sb, a.q_st = 2 * q_st, a.q_sh = 2 * q_sh;
  a.k = (const char*)k, a.k_sb = 2 * k_sb, a.k_st = 2 * k_st, a.k_sh = 2 * k_sh;
  a.cos = (const char*)cos, a.sin = (const char*)sin, a.cs_sb = 2 * cs_sb, a.cs_st = 2 * cs_st;
  a.wq = (const char*)q_norm, a.wk = (const char*)k_norm, a.eps = eps;
  const int64_t row = 2ll * head_dim;  // outputs [B, heads, T, Dh], contiguous
  a.q_out = (char*)q_out, a.qo_st = row, a.qo_sh = row * seq, a.qo_sb = row * seq * num_heads;
  a.k_out = (char*)k_out, a.ko_st = row, a.ko_sh = row * seq, a.ko_sb = row * seq * num_kv_heads;
  a.tokens = (unsigned)((int64_t)batch * seq), a.T = (unsigned)seq;
  a.H = num_heads, a.Hkv = num_kv_heads, a.dh = head_dim, a.bs = 1;
  return launch_qk(fn, a, dtype, kRows, reinterpret_cast<hipStream_t>(stream));
}
