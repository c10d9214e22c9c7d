// Rotation of queries and keys by their positions, in the forms that long contexts and other checkpoints use (the reference has
// the half-split rotation of whole heads, src/minillm/model/llama.py:58-72, with tables in the model's type):
//   out[a] = f (x[a] cos t - x[b] sin t),  out[b] = f (x[b] cos t + x[a] sin t),  t = position inv_freq[i]
// for the pairs i of the first `rot` dims of each head: (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved; dims behind them
// are copied.  Angles are products in 64 bits, reduced to a part of a turn there: in 32 bits a position of 10^6 is off by
// up to 0.06 rad.  The rest is fp32 with one rounding at the end.
//
// A workgroup takes a few tokens: it computes their cosines and sines once, into LDS, and turns all heads' rows with them.  Bound
// by memory: each row is read once and written once.
#include "kv_common.h"

namespace mllm {
namespace {

struct RotaryArgs {
  const char *q, *k;  // strides in bytes: batch, token, head
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh;
  const int64_t* positions;
  int64_t p_sb, p_st;
  const float* inv_freq;
  float factor;
  char *q_out, *k_out;  // [B, T, heads, Dh], contiguous
  unsigned tokens, T;
  int H, Hkv, dh, half, per_group;  // half: pairs; per_group: tokens of a workgroup
};

constexpr int kMaxPairs = 512;  // of a workgroup's tokens together

template <typename T, int VEC>
struct Vals {
  float f[VEC];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (VEC == 8) {
      Chunk c;
      c.v = ld16(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(c.e[i]);
    } else {
      f[0] = to_f32<T>(*reinterpret_cast<const uint16_t*>(p));
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (VEC == 8)
      st16(p, u32x4{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])});
    else
      *reinterpret_cast<uint16_t*>(p) = cvt1<T>(f[0]);
  }
};

// VEC 8: 16-byte pieces; 1: element by element, for other alignments and dims.
template <typename T, bool INTER, int VEC>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[kMaxPairs], sn[kMaxPairs];
  const unsigned t0 = blockIdx.x * (unsigned)a.per_group;
  const unsigned n = min((unsigned)a.per_group, a.tokens - t0);
  for (unsigned i = threadIdx.x; i < n * (unsigned)a.half; i += 256) {
    const unsigned u = i / (unsigned)a.half, d = i - u * (unsigned)a.half, t = t0 + u, b = t / a.T;
    const double turns = (double)a.positions[b * a.p_sb + (t - b * a.T) * a.p_st] * (double)a.inv_freq[d] * 0.15915494309189535;
    const float part = (float)(turns - __builtin_rint(turns));  // of a turn, as v_sin and v_cos take it
    cs[i] = a.factor * __builtin_amdgcn_cosf(part);
    sn[i] = a.factor * __builtin_amdgcn_sinf(part);
  }
  __syncthreads();
  // items of a head: the turned pieces (with their partners, where those lie apart), then the copied ones
  const unsigned turned = (unsigned)(INTER ? 2 * a.half / (VEC == 1 ? 2 : VEC) : a.half / VEC);
  const unsigned per_head = turned + (unsigned)(a.dh - 2 * a.half) / VEC, heads = (unsigned)(a.H + a.Hkv);
  const unsigned per_token = per_head * heads;
  for (unsigned i = threadIdx.x; i < n * per_token; i += 256) {
    const unsigned u = i / per_token, r = i - u * per_token, head = r / per_head, it = r - head * per_head;
    const unsigned t = t0 + u, b = t / a.T;
    const int64_t tt = t - b * a.T;
    const bool is_q = head < (unsigned)a.H;
    const int64_t h = is_q ? head : head - (unsigned)a.H;
    const char* src = is_q ? a.q + b * a.q_sb + tt * a.q_st + h * a.q_sh : a.k + b * a.k_sb + tt * a.k_st + h * a.k_sh;
    char* dst = (is_q ? a.q_out + ((int64_t)t * a.H + h) * a.dh * 2 : a.k_out + ((int64_t)t * a.Hkv + h) * a.dh * 2);
    Vals<T, VEC> x, y;
    if (it >= turned) {
      const unsigned at = 2 * (2 * a.half + (it - turned) * VEC);
      x.load(src + at);
      x.store(dst + at);
      continue;
    }
    const float *c = cs + u * a.half, *s = sn + u * a.half;
    if constexpr (INTER && VEC == 8) {
      x.load(src + 16 * it);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float cc = c[4 * it + e], ss = s[4 * it + e];
        y.f[2 * e] = x.f[2 * e] * cc - x.f[2 * e + 1] * ss;
        y.f[2 * e + 1] = x.f[2 * e + 1] * cc + x.f[2 * e] * ss;
      }
      y.store(dst + 16 * it);
    } else {
      const unsigned lo = 2 * (INTER ? 2 * it : it * VEC), hi = lo + 2 * (unsigned)(INTER ? 1 : a.half);
      x.load(src + lo);
      y.load(src + hi);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float cc = c[it * VEC + e], ss = s[it * VEC + e], p = x.f[e], q = y.f[e];
        x.f[e] = p * cc - q * ss;
        y.f[e] = q * cc + p * ss;
      }
      x.store(dst + lo);
      y.store(dst + hi);
    }
  }
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_rotary(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                           int64_t k_st, const int64_t* positions, int64_t p_sb, int64_t p_st, const float* inv_freq,
                           int32_t pairs, int32_t interleaved, float factor, int32_t batch, int32_t seq, int32_t num_heads,
                           int32_t num_kv_heads, int32_t head_dim, int32_t dtype, void* q_out, void* k_out, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_rotary";
  MLLM_REQUIRE(dtype == MLLM_DTYPE_BF16 || dtype == MLLM_DTYPE_F16, MLLM_ERR_UNSUPPORTED,
               fn + ": dtype must be bfloat16 or float16");
  const int64_t tokens = (int64_t)batch * seq;
  MLLM_REQUIRE(batch >= 0 && seq >= 0 && tokens < (1ll << 31) && num_heads > 0 && num_kv_heads > 0 && head_dim > 0 &&
                   num_heads < (1 << 16) && num_kv_heads < (1 << 16),
               MLLM_ERR_INVALID, fn + ": bad sizes");
  MLLM_REQUIRE(pairs > 0 && 2 * (int64_t)pairs <= head_dim, MLLM_ERR_INVALID, fn + ": at most head_dim / 2 pairs, and one at least");
  MLLM_REQUIRE(pairs <= kMaxPairs && head_dim <= 4096, MLLM_ERR_UNSUPPORTED, fn + ": head too long");
  if (tokens == 0) return MLLM_OK;
  MLLM_REQUIRE(q && k && positions && inv_freq && q_out && k_out, MLLM_ERR_INVALID, fn + ": null pointer");
  MLLM_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out) % 2 == 0, MLLM_ERR_UNSUPPORTED,
               fn + ": misaligned");
  RotaryArgs a{};
  a.q = (const char*)q, a.q_sb = 2 * q_sb, a.q_st = 2 * q_st, a.q_sh = 2 * q_sh;
  a.k = (const char*)k, a.k_sb = 2 * k_sb, a.k_st = 2 * k_st, a.k_sh = 2 * k_sh;
  a.positions = positions, a.p_sb = p_sb, a.p_st = p_st;
  a.inv_freq = inv_freq, a.factor = factor;
  a.q_out = (char*)q_out, a.k_out = (char*)k_out;
  a.tokens = (unsigned)tokens, a.T = (unsigned)seq;
  a.H = num_heads, a.Hkv = num_kv_heads, a.dh = head_dim, a.half = pairs;
  // several tokens to a workgroup once that leaves each CU workgroups to overlap
  int per = 1;
  while (per < 4 && 2 * per * pairs <= kMaxPairs && tokens >= 8ll * device_cus() * 2 * per) per *= 2;
  a.per_group = per;
  const int64_t groups = (tokens + per - 1) / per;
  MLLM_REQUIRE(groups <= kMaxGroups256, MLLM_ERR_UNSUPPORTED, fn + ": too many tokens");
  const bool whole = (interleaved ? 2 * pairs : pairs) % 8 == 0 && (head_dim - 2 * pairs) % 8 == 0 &&
                     ((uintptr_t)q | (uintptr_t)k | (uintptr_t)q_out | (uintptr_t)k_out) % 16 == 0 &&
                     (q_sb | q_sh | q_st | k_sb | k_sh | k_st) % 8 == 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto launch = [&](auto tag, auto inter) {
    using T = decltype(tag);
    constexpr bool INTER = decltype(inter)::value;
    if (whole)
      rotary_kernel<T, INTER, 8><<<(unsigned)groups, 256, 0, st>>>(a);
    else
      rotary_kernel<T, INTER, 1><<<(unsigned)groups, 256, 0, st>>>(a);
  };
  auto of_type = [&](auto tag) {
    if (interleaved)
      launch(tag, std::true_type{});
    else
      launch(tag, std::false_type{});
  };
  if (dtype == MLLM_DTYPE_BF16)
    of_type(BF16{});
  else
    of_type(F16{});
  return check_launch(fn.c_str());
}
