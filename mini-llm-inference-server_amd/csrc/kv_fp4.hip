// 4-bit KV pool: append a step's K and V rows, and read rows back (no counterpart in the reference; see common.h for the
// codes and scales).
//
// Layout: codes [num_blocks, block_size, Hkv, Dh / 2] bytes, as the other pools.  Scales lie as the decode kernel's lanes
// read them: K scales [num_blocks, block_size, Dh / 32, Hkv], because a lane multiplies with one dim block of one token's keys
// of adjacent heads; V scales [num_blocks, Hkv, Dh / 32, block_size], because a lane holds consecutive tokens of one dim block.
// Either way a lane's scales are one load.
//
// One thread moves eight dims: 16 bytes of a 16-bit row, four bytes of codes.  A block's largest magnitude is the
// maximum over its four threads of the 16-bit patterns without their sign, which order as the magnitudes do and put
// infinities and NaN on top.  Bound by the launch up to some hundred tokens (8 tokens: 2.8 us),
// by memory above: 8191 tokens of 8 heads of 128 dims, 42 MB, appended in 10.1 us, read back in 10.1 (4.2 TB/s).
#include "kv_common.h"

namespace mllm {
namespace {

// blockIdx.y: 0 K, 1 V.  A row's eight-dim chunks are consecutive threads (chunks a multiple of four), so the four lanes
// of a block stay together; a lane past the end or of a token without a slot has no partner that needs its value.
template <typename T>
__global__ __launch_bounds__(256) void append_fp4_kernel(const char* __restrict__ k, int64_t k_st, int64_t k_sh,
                                                        const char* __restrict__ v, int64_t v_st, int64_t v_sh,
                                                        Fp4Pool kp, Fp4Pool vp, int64_t num_slots, int hkv, int chunks,
                                                        int bs, const int64_t* __restrict__ slots, int64_t num_tokens) {
  const unsigned per_tok = (unsigned)(hkv * chunks);
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  const unsigned t = i / per_tok, rem = i - t * per_tok;
  if (t >= num_tokens) return;
  const int h = (int)(rem / (unsigned)chunks), ch = (int)(rem - (unsigned)h * (unsigned)chunks);
  const bool is_v = blockIdx.y != 0;
  const u32x4 x = ld16((is_v ? v + t * v_st + h * v_sh : k + t * k_st + h * k_sh) + 16 * (int64_t)ch);
  const int64_t slot = slots[t];
  const uint32_t e = block_exp<T>(x);
  if (slot < 0 || slot >= num_slots) return;
  const Fp4Pool p = is_v ? vp : kp;
  *reinterpret_cast<uint32_t*>(p.codes + 4 * (slot * per_tok + rem)) = fp4x8_from<T>(x, e8m0_to_f32(e));
  const int nblk = chunks / 4;
  if ((ch & 3) == 0)
    p.scales[is_v ? v_scale_at(slot, h, ch >> 2, hkv, nblk, bs) : k_scale_at(slot, h, ch >> 2, hkv, nblk)] = (uint8_t)e;
}

// Rows `slots` of the pools as 16-bit values [n, Hkv, Dh]; a slot outside the pool reads as zeros.
template <typename T>
__global__ __launch_bounds__(256) void read_fp4_kernel(Fp4Pool kp, Fp4Pool vp, int64_t num_slots, int hkv, int chunks,
                                                      int bs, const int64_t* __restrict__ slots, int64_t n,
                                                      char* __restrict__ k_out, char* __restrict__ v_out) {
  const unsigned per_tok = (unsigned)(hkv * chunks);
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  const unsigned t = i / per_tok, rem = i - t * per_tok;
  if (t >= n) return;
  const int h = (int)(rem / (unsigned)chunks), ch = (int)(rem - (unsigned)h * (unsigned)chunks), nblk = chunks / 4;
  const bool is_v = blockIdx.y != 0;
  const Fp4Pool p = is_v ? vp : kp;
  const int64_t slot = slots[t];
  u32x4 x = {0, 0, 0, 0};
  if (slot >= 0 && slot < num_slots) {
    const uint32_t e =
        p.scales[is_v ? v_scale_at(slot, h, ch >> 2, hkv, nblk, bs) : k_scale_at(slot, h, ch >> 2, hkv, nblk)];
    x = fp4x8_to<T>(*reinterpret_cast<const uint32_t*>(p.codes + 4 * (slot * per_tok + rem)), e8m0_to_f32(e));
  }
  st16((is_v ? v_out : k_out) + 16 * (int64_t)i, x);
}

// The checks both entry points share; `groups` receives the launch's workgroups.
int check_fp4(const std::string& fn, int32_t dtype, int64_t num_tokens, int64_t num_blocks, int32_t block_size,
              int32_t num_kv_heads, int32_t head_dim, int64_t* groups) {
  MLLM_REQUIRE(dtype == MLLM_DTYPE_BF16 || dtype == MLLM_DTYPE_F16, MLLM_ERR_UNSUPPORTED,
               fn + ": dtype must be bfloat16 or float16");
  MLLM_REQUIRE(num_tokens >= 0 && num_blocks >= 0 && block_size > 0 && num_kv_heads > 0 && head_dim > 0, MLLM_ERR_INVALID,
               fn + ": bad sizes");
  MLLM_REQUIRE(head_dim % kFp4Block == 0, MLLM_ERR_UNSUPPORTED, fn + ": head_dim must be a multiple of 32");
  MLLM_REQUIRE((int64_t)num_kv_heads * head_dim < (1 << 24), MLLM_ERR_UNSUPPORTED, fn + ": rows too long");
  const int64_t per_tok = (int64_t)num_kv_heads * (head_dim / 8);
  MLLM_REQUIRE(num_tokens <= kMaxGroups256 * 256 / per_tok, MLLM_ERR_UNSUPPORTED, fn + ": too many tokens");
  *groups = (num_tokens * per_tok + 255) / 256;
  return MLLM_OK;
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_kv_append_fp4(const void* k, int64_t k_stride_tok, int64_t k_stride_head, const void* v,
                                  int64_t v_stride_tok, int64_t v_stride_head, int32_t src_dtype, void* k_cache,
                                  void* v_cache, void* k_scales, void* v_scales, int64_t num_blocks,
                                  int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                                  const int64_t* slot_mapping, int64_t num_tokens, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_kv_append_fp4";
  int64_t groups = 0;
  const int rc = check_fp4(fn, src_dtype, num_tokens, num_blocks, block_size, num_kv_heads, head_dim, &groups);
  if (rc != MLLM_OK) return rc;
  if (num_tokens == 0) return MLLM_OK;
  MLLM_REQUIRE(k && v && k_cache && v_cache && k_scales && v_scales && slot_mapping, MLLM_ERR_INVALID,
               fn + ": null pointer");
  MLLM_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0 && ((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 &&
                   (k_stride_tok | k_stride_head | v_stride_tok | v_stride_head) % 8 == 0,
               MLLM_ERR_UNSUPPORTED, fn + ": rows must be 16-byte aligned");
  const dim3 grid((unsigned)groups, 2);
  const Fp4Pool kp{(char*)k_cache, (uint8_t*)k_scales}, vp{(char*)v_cache, (uint8_t*)v_scales};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto launch = [&](auto tag) {
    append_fp4_kernel<decltype(tag)><<<grid, 256, 0, st>>>(
        (const char*)k, 2 * k_stride_tok, 2 * k_stride_head, (const char*)v, 2 * v_stride_tok, 2 * v_stride_head, kp, vp,
        num_blocks * block_size, num_kv_heads, head_dim / 8, block_size, slot_mapping, num_tokens);
  };
  if (src_dtype == MLLM_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return check_launch(fn.c_str());
}

extern "C" int mllm_kv_read_fp4(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                                int64_t num_blocks, int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                                const int64_t* slots, int64_t num_slots, int32_t dtype, void* k_out, void* v_out,
                                void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_kv_read_fp4";
  int64_t groups = 0;
  const int rc = check_fp4(fn, dtype, num_slots, num_blocks, block_size, num_kv_heads, head_dim, &groups);
  if (rc != MLLM_OK) return rc;
  if (num_slots == 0) return MLLM_OK;
  MLLM_REQUIRE(k_cache && v_cache && k_scales && v_scales && slots && k_out && v_out, MLLM_ERR_INVALID,
               fn + ": null pointer");
  MLLM_REQUIRE(((uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0,
               MLLM_ERR_UNSUPPORTED, fn + ": rows must be 16-byte aligned");
  const dim3 grid((unsigned)groups, 2);
  const Fp4Pool kp{(char*)k_cache, (uint8_t*)k_scales}, vp{(char*)v_cache, (uint8_t*)v_scales};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto launch = [&](auto tag) {
    read_fp4_kernel<decltype(tag)><<<grid, 256, 0, st>>>(kp, vp, num_blocks * block_size, num_kv_heads, head_dim / 8,
                                                         block_size, slots, num_slots, (char*)k_out, (char*)v_out);
  };
  if (dtype == MLLM_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return check_launch(fn.c_str());
}
