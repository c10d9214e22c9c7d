// Rotation of queries and keys by their positions, in the forms that long contexts and other checkpoints use (the reference has
// the half-split rotation of whole heads, src/minillm/model/llama.py:58-72, with tables in the model's type):
//   out[a] = f (x[a] cos t - x[b] sin t),  out[b] = f (x[b] cos t + x[a] sin t),  t = position inv_freq[i]
// for the pairs i of the first `rot` dims of each head: (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved; dims behind them
// are copied.  Angles are products in 64 bits, reduced to a part of a turn there: in 32 bits a position of 10^6 is off by
// up to 0.06 rad.  The rest is fp32 with one rounding at the end.
//
// Each thread takes one piece of a row, its workgroup the cosines and sines of the tokens that its pieces lie in, once, through
// LDS, while the rows are on their way.  Bound by memory: each row is read once and written once.  4 x 2,049 tokens of 40 heads
// of 128 dims in 16 bits, 168 MB: 29 us, 5.8 TB/s; with a token a workgroup 35, with persistent workgroups four pieces ahead
// 39.5.  A decode step's 32 tokens: 3 us, a launch.
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
  char *q_out, *k_out;
  int64_t qo_sb, qo_st, qo_sh, ko_sb, ko_st, ko_sh;
  unsigned tokens, T;
  int H, Hkv, dh, half;  // half: pairs
};

constexpr int kMaxPairs = 512;
// Cosines a workgroup may need: those of the tokens that 256 pieces lie in.  Two heads at least, a piece turns eight pairs at most:
// whole tokens take 4 pairs a piece, and the first and the last may be cut.
constexpr int kTable = 4 * 256 + 2 * kMaxPairs;

template <typename T, int VEC>
struct Vals {
  float f[VEC];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (VEC == 8) {
      Chunk c;
      c.v = ld16(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(c.e[i]);
    } else if constexpr (VEC == 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
      f[0] = to_f32<T>((uint16_t)w), f[1] = to_f32<T>((uint16_t)(w >> 16));
    } else {
      f[0] = to_f32<T>(*reinterpret_cast<const uint16_t*>(p));
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (VEC == 8)
      st16(p, u32x4{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])});
    else if constexpr (VEC == 2)
      *reinterpret_cast<uint32_t*>(p) = pack2<T>(f[0], f[1]);
    else
      *reinterpret_cast<uint16_t*>(p) = cvt1<T>(f[0]);
  }
};

// VEC: elements of a piece, 16 bytes of them or as many as sizes and alignment allow (launch).
template <typename T, bool INTER, int VEC>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  __shared__ __attribute__((aligned(16))) float cs[kTable], sn[kTable];
  // pieces of a head: the turned ones (with their partners, where those lie apart), then the copied ones
  constexpr bool kTwo = !(INTER && VEC > 1);  // a piece's partner is a piece of its own
  const unsigned turned = (unsigned)(kTwo && INTER ? a.half : (kTwo ? a.half : 2 * a.half) / VEC);
  const unsigned per_head = turned + (unsigned)(a.dh - 2 * a.half) / VEC, per_token = per_head * (unsigned)(a.H + a.Hkv);
  const uint64_t first = (uint64_t)blockIdx.x * 256u;
  const unsigned t0 = (unsigned)(first / per_token), r0 = (unsigned)(first - (uint64_t)t0 * per_token);  // its first token and piece of it
  const unsigned i = r0 + threadIdx.x, u = i / per_token, r = i - u * per_token, head = r / per_head, it = r - head * per_head;
  const unsigned t = t0 + u;
  const bool in = t < a.tokens, copied = it >= turned;
  Vals<T, VEC> x, y;
  char* dst = nullptr;
  if (in) {
    const unsigned b = t / a.T;
    const int64_t tt = t - b * a.T;
    const bool is_q = head < (unsigned)a.H;
    const int64_t h = is_q ? head : head - (unsigned)a.H;
    const unsigned lo = 2 * (copied ? 2 * a.half + (it - turned) * VEC : (kTwo && INTER ? 2 * it : it * VEC));
    const char* src = (is_q ? a.q + b * a.q_sb + tt * a.q_st + h * a.q_sh : a.k + b * a.k_sb + tt * a.k_st + h * a.k_sh) + lo;
    dst = (is_q ? a.q_out + b * a.qo_sb + tt * a.qo_st + h * a.qo_sh : a.k_out + b * a.ko_sb + tt * a.ko_st + h * a.ko_sh) + lo;
    x.load(src);
    if (kTwo && !copied) y.load(src + 2 * (INTER ? 1 : a.half));
  }
  const unsigned n = min((r0 + 255) / per_token + 1, a.tokens - t0);  // tokens of this workgroup
  for (unsigned c = threadIdx.x; c < n * (unsigned)a.half; c += 256) {
    const unsigned w = c / (unsigned)a.half, d = c - w * (unsigned)a.half, tok = t0 + w, b = tok / a.T;
    const double turns = (double)a.positions[b * a.p_sb + (tok - b * a.T) * a.p_st] * (double)a.inv_freq[d] * 0.15915494309189535;
    const float part = (float)(turns - __builtin_rint(turns));  // of a turn, as v_sin and v_cos take it
    cs[c] = a.factor * __builtin_amdgcn_cosf(part);
    sn[c] = a.factor * __builtin_amdgcn_sinf(part);
  }
  __syncthreads();
  if (!in) return;
  if (copied) {
    x.store(dst);
    return;
  }
  const unsigned at = u * (unsigned)a.half + it * (kTwo ? VEC : VEC / 2);
  const float *c = cs + at, *s = sn + at;
  if constexpr (!kTwo) {
    Vals<T, VEC> z;
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      z.f[2 * e] = x.f[2 * e] * c[e] - x.f[2 * e + 1] * s[e];
      z.f[2 * e + 1] = x.f[2 * e + 1] * c[e] + x.f[2 * e] * s[e];
    }
    z.store(dst);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float p = x.f[e], q = y.f[e];
      x.f[e] = p * c[e] - q * s[e];
      y.f[e] = q * c[e] + p * s[e];
    }
    x.store(dst);
    y.store(dst + 2 * (INTER ? 1 : a.half));
  }
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_rotary(const mllm_rotary_args* args, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_rotary";
  MLLM_REQUIRE(args, MLLM_ERR_INVALID, fn + ": null arguments");
  const mllm_rotary_args& r = *args;
  const int32_t batch = r.batch, seq = r.seq, num_heads = r.num_heads, num_kv_heads = r.num_kv_heads, head_dim = r.head_dim;
  const int32_t pairs = r.pairs, dtype = r.dtype;
  MLLM_REQUIRE(dtype == MLLM_DTYPE_BF16 || dtype == MLLM_DTYPE_F16, MLLM_ERR_UNSUPPORTED,
               fn + ": dtype must be bfloat16 or float16");
  const int64_t tokens = (int64_t)batch * seq;
  MLLM_REQUIRE(batch >= 0 && seq >= 0 && tokens < (1ll << 31) && num_heads > 0 && num_kv_heads > 0 && head_dim > 0 &&
                   num_heads < (1 << 16) && num_kv_heads < (1 << 16),
               MLLM_ERR_INVALID, fn + ": bad sizes");
  MLLM_REQUIRE(pairs > 0 && 2 * (int64_t)pairs <= head_dim, MLLM_ERR_INVALID, fn + ": at most head_dim / 2 pairs, and one at least");
  MLLM_REQUIRE(pairs <= kMaxPairs && head_dim <= 4096, MLLM_ERR_UNSUPPORTED, fn + ": head too long");
  if (tokens == 0) return MLLM_OK;
  MLLM_REQUIRE(r.q && r.k && r.positions && r.inv_freq && r.q_out && r.k_out, MLLM_ERR_INVALID, fn + ": null pointer");
  const uintptr_t ptrs = (uintptr_t)r.q | (uintptr_t)r.k | (uintptr_t)r.q_out | (uintptr_t)r.k_out;
  MLLM_REQUIRE(ptrs % 2 == 0, MLLM_ERR_UNSUPPORTED, fn + ": misaligned");
  RotaryArgs a{};
  a.q = (const char*)r.q, a.q_sb = 2 * r.q_sb, a.q_st = 2 * r.q_st, a.q_sh = 2 * r.q_sh;
  a.k = (const char*)r.k, a.k_sb = 2 * r.k_sb, a.k_st = 2 * r.k_st, a.k_sh = 2 * r.k_sh;
  a.positions = r.positions, a.p_sb = r.p_sb, a.p_st = r.p_st;
  a.inv_freq = r.inv_freq, a.factor = r.factor;
  a.q_out = (char*)r.q_out, a.qo_sb = 2 * r.qo_sb, a.qo_st = 2 * r.qo_st, a.qo_sh = 2 * r.qo_sh;
  a.k_out = (char*)r.k_out, a.ko_sb = 2 * r.ko_sb, a.ko_st = 2 * r.ko_st, a.ko_sh = 2 * r.ko_sh;
  a.tokens = (unsigned)tokens, a.T = (unsigned)seq;
  a.H = num_heads, a.Hkv = num_kv_heads, a.dh = head_dim, a.half = pairs;
  const int64_t strides = r.q_sb | r.q_sh | r.q_st | r.k_sb | r.k_sh | r.k_st | r.qo_sb | r.qo_sh | r.qo_st | r.ko_sb | r.ko_sh | r.ko_st;
  // 16 bytes a piece where every piece is whole and aligned, else 4, else single elements: 4 x 2,049 tokens of 40 heads of 128
  // dims take 28-30 us, 48 (adjacent pairs 82) and 85-89.
  auto fits = [&](int v) {
    return (r.interleaved ? 2 * pairs : pairs) % v == 0 && (head_dim - 2 * pairs) % v == 0 && ptrs % (2 * v) == 0 && strides % v == 0;
  };
  const int vec = fits(8) ? 8 : fits(2) ? 2 : 1;
  const int turned = r.interleaved ? (vec == 1 ? pairs : 2 * pairs / vec) : pairs / vec;
  const int64_t per_token = (int64_t)(turned + (head_dim - 2 * pairs) / vec) * (num_heads + num_kv_heads);
  const int64_t groups = (tokens * per_token + 255) / 256;
  MLLM_REQUIRE(groups <= kMaxGroups256, MLLM_ERR_UNSUPPORTED, fn + ": too many tokens");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto launch = [&](auto tag, auto inter) {
    using T = decltype(tag);
    constexpr bool INTER = decltype(inter)::value;
    if (vec == 8)
      rotary_kernel<T, INTER, 8><<<(unsigned)groups, 256, 0, st>>>(a);
    else if (vec == 2)
      rotary_kernel<T, INTER, 2><<<(unsigned)groups, 256, 0, st>>>(a);
    else
      rotary_kernel<T, INTER, 1><<<(unsigned)groups, 256, 0, st>>>(a);
  };
  auto of_type = [&](auto tag) {
    if (r.interleaved)
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
