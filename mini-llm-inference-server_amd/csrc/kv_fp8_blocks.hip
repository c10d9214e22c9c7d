// 8-bit KV pool with a scale for each block of tokens and head: append a step's K and V rows (optionally with the rotation and
// the head norms), and read rows back (no counterpart in the reference, whose planned fp8 cache has a scale per tensor).
//
// Layout: codes e4m3 [num_blocks, block_size, Hkv, 128], as the fp8 pool; scales e8m0 [num_blocks, Hkv] for K and for V, one
// byte for a page and head.  value = code 2^(scale - 127).
//
// A page's tokens share their scale, and tokens come a step at a time.  A run is a step's consecutive tokens at consecutive
// slots of one page.  With amax the largest finite magnitude of a run (and head), its exponent is the least e with
// amax <= 448 2^(e - 127).  A run at the page's first slot begins a new block under e, whatever the page held.  A run
// behind earlier tokens takes max(e, the block's exponent), and where that grows, the codes before the run are rounded again to
// it.  The scales are powers of two because that rounding is then exact for every code that stays normal: a page holds
// the same values however its tokens came in, but for those below 2^-6 of the scale, which round twice.  An infinity or a
// NaN becomes the code of NaN in its own place and takes no part in amax.
//
// A wavefront takes a few tokens of one head's K or V: 16 lanes hold a token's 128 dims, 16 bytes each, four tokens side by
// side.  In steps of many tokens it takes the runs that begin in its window of 16 tokens, whole: a page's 16 tokens stay in
// registers between their amax and their codes.  In small steps it takes four tokens (four decode rows at once) and reads what
// else their runs hold for its amax alone, so no wavefront waits for another.  The wavefront of a run's first token writes
// the scale and rounds the codes before it; the others read the old scale or the new one and get the same maximum from either.
//
// Bound by launch latency for few tokens (32 rows of 8 heads: 3.6 us, their read back 2.9) and by memory for many: 8,200 tokens
// of 8 heads, 50 MB, are appended in 12.1 us (4.2 TB/s; 20.9 with windows of 16 tokens that read what else their runs hold again,
// 14.4 with one routine for all runs, whose registers halve the wavefronts on a CU) and read back in 9.5 (5.3 TB/s).  With the
// rotation and 32 heads of q: 32 rows 3.4 us, with the norms 3.3; 8,200 tokens, 189 MB, 43.5 and 35.7 (4.3 and 5.3 TB/s: the
// rotation alone rounds each product and sum as torch does), where the same into a 16-bit pool, 206 MB, takes 36.
#include "kv_common.h"

namespace mllm {
namespace {

constexpr int kDh = 128;

// Patterns of the 16-bit type without sign: infinity, the largest magnitude the scales reach (448 times the largest);
// and the scale exponents whose values, 2^-9 to 448 of them, the type holds.
template <typename T>
struct Fp8Range;
template <>
struct Fp8Range<BF16> {
  static constexpr uint32_t inf = 0x7f80, top = 0x7f60;
  static constexpr int lo = 10, hi = 246;
};
template <>
struct Fp8Range<F16> {
  static constexpr uint32_t inf = 0x7c00, top = 0x7b00;
  static constexpr int lo = 112, hi = 134;
};

__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140, kRotate8 = 0x128;  // within rows of 16 lanes

// The largest of 16 lanes, in each of them.
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, dpp<kXor1>(x));
  x = max(x, dpp<kXor2>(x));
  x = max(x, dpp<kHalfMirror>(x));
  return max(x, dpp<kMirror>(x));
}
__device__ __forceinline__ float sum16(float x) {
  x += __uint_as_float(dpp<kXor1>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kXor2>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kHalfMirror>(__float_as_uint(x)));
  return x + __uint_as_float(dpp<kMirror>(__float_as_uint(x)));
}

// The largest magnitude (pattern) of eight values, past infinity's for a NaN.
__device__ __forceinline__ uint32_t max8(u32x4 x) {
  constexpr uint32_t kSign = 0x7fff7fffu;
  const uint32_t m = max_u16x2(max_u16x2(x[0] & kSign, x[1] & kSign), max_u16x2(x[2] & kSign, x[3] & kSign));
  return max(m & 0xffffu, m >> 16);
}
// The largest finite one.
template <typename T>
__device__ __forceinline__ uint32_t finite_max8(u32x4 x) {
  uint32_t a = max8(x);
  if (a >= Fp8Range<T>::inf) {
    a = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = x[i] & 0x7fffu, hi = (x[i] >> 16) & 0x7fffu;
      if (lo < Fp8Range<T>::inf) a = max(a, lo);
      if (hi < Fp8Range<T>::inf) a = max(a, hi);
    }
  }
  return a;
}

// The exponent for a finite magnitude: floor(log2 amax) - 8 puts it in [256, 512) of the scale; adding just under a quarter of
// the mantissa carries where it is past 448.
template <typename T>
__device__ __forceinline__ int block_exp8(uint32_t amax) {
  const uint32_t u = __float_as_uint(to_f32<T>((uint16_t)amax));
  return min(max((int)((u + 0x1fffffu) >> 23) - 8, Fp8Range<T>::lo), Fp8Range<T>::hi);
}

template <typename T>
__device__ __forceinline__ uint32_t pk4(uint32_t a, uint32_t b, float scale) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same<T, BF16>::value) {
    const i16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(i16x2{0, 0}, __builtin_bit_cast(bf16x2, a), scale, false);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, b), scale, true));
  } else {
    const i16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(i16x2{0, 0}, __builtin_bit_cast(f16x2, a), scale, false);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, b), scale, true));
  }
}

// Eight values -> eight codes of x / 2^(e - 127), to nearest with ties to even, at most 448; not finite (where `bad` says that
// there may be some): NaN.
template <typename T>
__device__ __forceinline__ u32x2 codes8(u32x4 x, int e, bool bad) {
  constexpr uint32_t kTop = Fp8Range<T>::top * 0x10001u;
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = min_u16x2(x[i] & 0x7fff7fffu, kTop) | (x[i] & 0x80008000u);
  const float scale = e8m0_to_f32((uint32_t)e);
  u32x2 c = {pk4<T>(y[0], y[1], scale), pk4<T>(y[2], y[3], scale)};
  if (bad) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (((x[i >> 1] >> (16 * (i & 1))) & 0x7fffu) >= Fp8Range<T>::inf) c[i >> 2] |= 0x7fu << (8 * (i & 3));
  }
  return c;
}

// Four codes rounded again to a scale 2^d times theirs, d <= 0 as the exponent of a float: through bf16, which holds them.
__device__ __forceinline__ uint32_t again4(uint32_t w, float two_d) {
  const u32x2 v = fp8x4_to<BF16>(w, two_d);
  return pk4<BF16>(v[0], v[1], 1.f);
}

enum Form { kPlain = 0, kRope = 1, kNormRope = 2 };

struct BlocksArgs {
  const char *k, *v;  // strides in bytes
  int64_t k_st, k_sh, v_st, v_sh;
  char *kc, *vc;
  uint8_t *ks, *vs;
  int64_t num_slots;
  const int64_t* slots;
  int hkv, bs, bs_shift;
  unsigned n;           // tokens
  unsigned pool_waves;  // wavefronts that append; those behind them turn q
  const char *q, *cos, *sin, *wq, *wk;
  int64_t q_st, q_sh, cs_st, qo_st, qo_sh;
  char* q_out;
  float eps;
  int H;
};

// Lane ln's 16 bytes of a row of 128 dims, normed and turned: dims 8 ln .. + 7, whose partners are lane ln ^ 8's.
template <typename T, int FORM>
__device__ __forceinline__ u32x4 turned(u32x4 x, const char* cr, const char* sr, const char* w, float eps, int ln) {
  Chunk c, s, v, p, o;
  c.v = ld16(cr + 16 * ln);
  s.v = ld16(sr + 16 * ln);
  v.v = x;
  if constexpr (FORM == kRope) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p.v[i] = dpp<kRotate8>(x[i]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = to_f32<T>(p.e[i]);
      o.e[i] = rot1<T>(v.e[i], c.e[i], ln < 8 ? -r : r, s.e[i]);
    }
  } else {
    Chunk wc;
    wc.v = ld16(w + 16 * ln);
    float y[8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = to_f32<T>(v.e[i]);
      ss += y[i] * y[i];
    }
    const float rs = rsqrtf(sum16(ss) / (float)kDh + eps);
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = y[i] * rs * to_f32<T>(wc.e[i]);
      const float r = __uint_as_float(dpp<kRotate8>(__float_as_uint(y[i])));
      f[i] = y[i] * to_f32<T>(c.e[i]) + (ln < 8 ? -r : r) * to_f32<T>(s.e[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
  }
  return o.v;
}

// One head's K or V of a pool, and its rows of the step, as a wavefront (lanes 16 j + ln) goes through them.
template <typename T, int FORM>
struct Appender {
  const BlocksArgs& a;
  const char* src;
  int64_t st;
  char* codes;
  uint8_t* scales;
  int64_t row_bytes;
  int lane, ln, j, mask;
  bool is_v;

  __device__ __forceinline__ Appender(const BlocksArgs& args, int h, bool v, int l)
      : a(args), src(v ? args.v + h * args.v_sh : args.k + h * args.k_sh), st(v ? args.v_st : args.k_st),
        codes((v ? args.vc : args.kc) + (int64_t)h * kDh), scales((v ? args.vs : args.ks) + h), row_bytes((int64_t)args.hkv * kDh),
        lane(l), ln(l & 15), j(l >> 4), mask(args.bs - 1), is_v(v) {}

  // lane ln's part of token t's row, as it goes into the pool
  __device__ __forceinline__ u32x4 row(int64_t t) const {
    const u32x4 x = ld16(src + t * st + 16 * ln);
    if constexpr (FORM == kPlain) {
      return x;
    } else {
      if (is_v) return x;
      return turned<T, FORM == kPlain ? kRope : FORM>(x, a.cos + t * a.cs_st, a.sin + t * a.cs_st, a.wk, a.eps, ln);
    }
  }

  // the largest finite magnitude of a wavefront's lanes
  static __device__ __forceinline__ uint32_t max64(uint32_t m) {
    m = max16(m);
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    return (uint32_t)__builtin_amdgcn_readfirstlane(max(m, (uint32_t)__shfl_xor((int)m, 32, 64)));
  }

  // of n tokens from t on
  __device__ __forceinline__ uint32_t top_of(int64_t t, int n) const {
    uint32_t m = 0;
    for (int i = 0; i < n; i += 4) m = max(m, finite_max8<T>(row(t + min(i + j, n - 1))));
    return max64(m);
  }

  // the first `rows` codes of a page, to a scale 2^-d times theirs
  __device__ __forceinline__ void round_again(int64_t page, int rows, int d) const {
    const float two_d = e8m0_to_f32((uint32_t)max(127 + d, 1));  // what 2^-126 leaves rounds to zero as well
    for (int r = lane >> 3; r < rows; r += 8) {
      char* c = codes + ((page << a.bs_shift) + r) * row_bytes + 16 * (lane & 7);
      u32x4 w = ld16(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = again4(w[i], two_d);
      st16(c, w);
    }
  }

  // One whole run of n tokens from t on, at slot s0: up to 16 rows stay in registers, longer runs are read twice.
  __device__ __forceinline__ void one_run(int64_t t, int n, int64_t s0) const {
    constexpr int W = 4;
    const int64_t page = s0 >> a.bs_shift;
    const int before = (int)(s0 & mask);
    int old = 0;
    if (before) old = scales[page * a.hkv];
    u32x4 x[W];
    auto load = [&](int i0) {
#pragma unroll
      for (int p = 0; p < W; ++p) {
        x[p] = u32x4{0, 0, 0, 0};
        if (i0 + 4 * p < n) x[p] = row(t + min(i0 + 4 * p + j, n - 1));
      }
    };
    load(0);
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < W; ++p) m = max(m, max8(x[p]));
    bool bad = __any(m >= Fp8Range<T>::inf);
    if (bad) {
      m = 0;
#pragma unroll
      for (int p = 0; p < W; ++p) m = max(m, finite_max8<T>(x[p]));
    }
    m = max64(m);
    if (n > 4 * W) m = max(m, top_of(t + 4 * W, n - 4 * W)), bad = true;  // (codes8 then looks for itself)
    const int e = before ? max(block_exp8<T>(m), __builtin_amdgcn_readfirstlane(old)) : block_exp8<T>(m);
    char* to = codes + (s0 + j) * row_bytes + 8 * ln;
    for (int i0 = 0; i0 < n; i0 += 4 * W) {
      if (i0) load(i0);
#pragma unroll
      for (int p = 0; p < W; ++p)
        if (i0 + 4 * p + j < n) st8(to + (i0 + 4 * p) * row_bytes, codes8<T>(x[p], e, bad));
    }
    if (lane == 0) scales[page * a.hkv] = (uint8_t)e;
    if (before && e > old) round_again(page, before, old - e);
  }

  // Up to four tokens from t0 on, of any runs: token t0 + j is lanes 16 j ..
  __device__ __forceinline__ void four_tokens(int64_t t0, int count) const {
    const int64_t last = t0 + count - 1, t = t0 + j, at = min(t, last);
    const int64_t s = a.slots[at], s_before = at > 0 ? a.slots[at - 1] : -1, s0 = a.slots[t0], sl = a.slots[last];
    const u32x4 x = row(at);
    const bool in = t <= last && s >= 0 && s < a.num_slots;
    const bool first = !in || s_before != s - 1 || (s & mask) == 0;  // begins a run, or has no slot
    // tokens before and behind these on a chain of slots of one page
    const int64_t tb = t0 - 1 - lane, ta = last + 1 + lane;
    const bool chain_b = s0 >= 0 && s0 < a.num_slots && lane < (int)(s0 & mask) && tb >= 0 &&
                         a.slots[max(tb, (int64_t)0)] == s0 - 1 - lane;
    const bool chain_a = sl >= 0 && sl < a.num_slots && (int)(sl & mask) + 1 + lane < a.bs && ta < a.n &&
                         a.slots[min(ta, (int64_t)a.n - 1)] == sl + 1 + lane;
    const int nb = __builtin_ctzll(~__ballot(chain_b)), na = __builtin_ctzll(~__ballot(chain_a));  // at most bs - 1 of 64 lanes
    const uint32_t own = finite_max8<T>(x), top = max16(own);
    const bool bad = __any(own != max8(x));
    const uint32_t top_b = nb ? top_of(t0 - nb, nb) : 0u, top_a = na ? top_of(last + 1, na) : 0u;

    // each token's run, [from u to v) of these tokens: its largest magnitude over them and what lies beyond
    const uint64_t f = __ballot(first);
    const uint32_t begins = (uint32_t)((f & 1) | (f >> 15 & 2) | (f >> 30 & 4) | (f >> 45 & 8));
    const uint32_t below = begins & ((2u << j) - 1), above = begins >> (j + 1);
    const int u = below ? 31 - __builtin_clz(below) : -nb, v = above ? j + 1 + __builtin_ctz(above) : 4;
    uint32_t m = max(below ? 0u : top_b, t0 + v > last ? top_a : 0u);
#pragma unroll
    for (int k = 0; k < 4; ++k) m = max(m, k >= u && k < v ? (uint32_t)__builtin_amdgcn_readlane((int)top, 16 * k) : 0u);

    const int64_t slot = in ? s : 0, page = slot >> a.bs_shift;
    const int before = (int)(slot & mask) - (j - u);  // slots of the page before the run
    int e = block_exp8<T>(m), old = e;
    if (in && before > 0) {
      old = scales[page * a.hkv];
      e = max(e, old);
    }
    const bool owner = in && first;
    if (in) st8(codes + slot * row_bytes + 8 * ln, codes8<T>(x, e, bad));
    if (owner && ln == 0 && (before == 0 || e != old)) scales[page * a.hkv] = (uint8_t)e;
    for (uint64_t grow = __ballot(owner && ln == 0 && e > old); grow; grow &= grow - 1) {
      const int of = __builtin_ctzll(grow);
      round_again(__builtin_amdgcn_readlane((int)page, of), __builtin_amdgcn_readlane(before, of), __builtin_amdgcn_readlane(old - e, of));
    }
  }
};

constexpr int kWindow = 16;  // tokens in whose window a wavefront's runs begin (WHOLE)

// WHOLE: the runs that begin in 16 tokens, each of them whole; without, four tokens and what their runs take.
template <typename T, int FORM, bool WHOLE>
__global__ __launch_bounds__(256) void append_fp8_blocks_kernel(const BlocksArgs a) {
  const int lane = threadIdx.x & 63, ln = lane & 15, j = lane >> 4;
  const unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
  if (FORM != kPlain && wave >= a.pool_waves) {  // four rows of q
    const unsigned r = (wave - a.pool_waves) * 4u + (unsigned)j, t = r / (unsigned)a.H;
    const bool in = t < a.n;
    const unsigned tt = in ? t : 0u, h = in ? r - t * (unsigned)a.H : 0u;
    const u32x4 x = ld16(a.q + tt * a.q_st + h * a.q_sh + 16 * ln);
    const u32x4 y = turned<T, FORM == kPlain ? kRope : FORM>(x, a.cos + tt * a.cs_st, a.sin + tt * a.cs_st, a.wq, a.eps, ln);
    if (in) st16(a.q_out + tt * a.qo_st + h * a.qo_sh + 16 * ln, y);
    return;
  }
  const unsigned per_window = 2u * (unsigned)a.hkv, window = wave / per_window;
  const int hv = (int)(wave - window * per_window);
  const Appender<T, FORM> to(a, hv >> 1, hv & 1, lane);
  if constexpr (!WHOLE) {
    const int64_t t0 = (int64_t)window * 4;
    if (t0 < a.n) to.four_tokens(t0, (int)min((int64_t)4, a.n - t0));
  } else {
    const int64_t t_window = (int64_t)window * kWindow;
    if (t_window >= a.n) return;
    // where runs begin (or tokens have no slot) among 64 tokens from `t` on; those past the last count too
    int64_t slot = -1;
    auto starts_from = [&](int64_t t) {
      const int64_t at = min(t, (int64_t)a.n - 1), s = a.slots[at], s_before = a.slots[max(at - 1, (int64_t)0)];
      const bool in = t < a.n && s >= 0 && s < a.num_slots;
      slot = in ? s : -1;
      return __ballot(!in || (s & to.mask) == 0 || t == 0 || s_before != s - 1);
    };
    const uint64_t starts = starts_from(t_window + lane);
    const int64_t slots16 = slot;
    for (int at = starts ? __builtin_ctzll(starts) : 64; at < kWindow;) {
      const uint64_t behind = starts >> (at + 1);
      // the next run begins at most bs tokens on: of as many on a chain one lies at a page's first slot
      int next = behind ? at + 1 + __builtin_ctzll(behind) : 64 + __builtin_ctzll(starts_from(t_window + 64 + lane));
      const int64_t t0 = t_window + at;
      if (t0 >= a.n) return;
      const int64_t s0 = ((int64_t)__builtin_amdgcn_readlane((int)(slots16 >> 32), at) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)slots16, at);
      if (next - at > 4) {
        if (s0 >= 0) to.one_run(t0, next - at, s0);
      } else {  // with the short ones behind it that fit and begin in the window
        while (next < kWindow) {
          const int end = next + 1 + __builtin_ctzll(starts >> (next + 1) | 1ull << 62);
          if (end - at > 4) break;
          next = end;
        }
        to.four_tokens(t0, (int)min((int64_t)(next - at), a.n - t0));
      }
      at = next;
    }
  }
}

// Rows `slots` of the pools as 16-bit values [n, Hkv, 128]; a slot outside the pool reads as zeros.  A thread takes 16 dims.
template <typename T>
__global__ __launch_bounds__(256) void read_fp8_blocks_kernel(const char* __restrict__ kc, const char* __restrict__ vc,
                                                             const uint8_t* __restrict__ ks, const uint8_t* __restrict__ vs,
                                                             int64_t num_slots, int hkv, int bs_shift,
                                                             const int64_t* __restrict__ slots, int64_t n,
                                                             char* __restrict__ k_out, char* __restrict__ v_out) {
  constexpr int kChunks = kDh / 16;
  const unsigned per_tok = (unsigned)(hkv * kChunks);
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  const unsigned t = i / per_tok, rem = i - t * per_tok;
  if (t >= n) return;
  const bool is_v = blockIdx.y != 0;
  const int64_t slot = slots[t];
  u32x4 lo = {0, 0, 0, 0}, hi = lo;
  if (slot >= 0 && slot < num_slots) {
    const float scale = e8m0_to_f32((is_v ? vs : ks)[(slot >> bs_shift) * hkv + rem / kChunks]);
    const u32x4 c = ld16((is_v ? vc : kc) + 16 * (slot * per_tok + rem));
    lo = fp8x8_to<T>(c[0], c[1], scale);
    hi = fp8x8_to<T>(c[2], c[3], scale);
  }
  char* out = (is_v ? v_out : k_out) + 32 * (int64_t)i;
  // past the caches: 8,200 tokens 9.5 against 11.0 us, 60,000 67.4 against 71.9
  __builtin_nontemporal_store(lo, reinterpret_cast<u32x4*>(out));
  __builtin_nontemporal_store(hi, reinterpret_cast<u32x4*>(out + 16));
}

// Up to so many tokens a wavefront takes four: few tokens are bound by the latency of a wavefront's chain, many by its
// instructions and by what is read again.  Of 8 heads, four tokens a wavefront against whole runs: 64 rows of one token 3.0 us
// against 7.2, 1,024 rows 3.9 against 7.9; 64 tokens in runs of 16 3.5 against 3.4, 1,024 4.7 against 3.8, 8,200 20.5 against
// 10.9.  With rotation and 32 heads of q, which four tokens a wavefront turn up to four times: 1,024 rows 8.8 against 11.9 (with
// norms 7.1 against 11.0), 1,024 in runs of 16 11.7 against 8.5 (8.5 against 6.6), 4,096 rows 26.7 against 27.9, 8,200 in runs
// of 16 66 against 44.  A step of up to 1,024 tokens may be decode rows throughout, one of more is prompts for the most part; the
// number of tokens alone loses up to 3 us to the better split on steps of 512-1,024 prompt tokens.
constexpr int64_t kSmallStep = 1024;

int check_blocks(const std::string& fn, int32_t dtype, int64_t num_tokens, int64_t num_blocks, int32_t block_size,
                 int32_t num_kv_heads, int32_t head_dim) {
  MLLM_REQUIRE(dtype == MLLM_DTYPE_BF16 || dtype == MLLM_DTYPE_F16, MLLM_ERR_UNSUPPORTED,
               fn + ": dtype must be bfloat16 or float16");
  MLLM_REQUIRE(num_tokens >= 0 && num_blocks >= 0 && num_kv_heads > 0, MLLM_ERR_INVALID, fn + ": bad sizes");
  MLLM_REQUIRE(head_dim == kDh, MLLM_ERR_UNSUPPORTED, fn + ": head_dim must be 128");
  MLLM_REQUIRE(block_size >= 16 && block_size <= 64 && (block_size & (block_size - 1)) == 0, MLLM_ERR_UNSUPPORTED,
               fn + ": block_size must be 16, 32 or 64");
  MLLM_REQUIRE(num_kv_heads < (1 << 16) && num_blocks < (1ll << 31), MLLM_ERR_UNSUPPORTED, fn + ": pool too large");
  MLLM_REQUIRE(num_tokens <= kMaxGroups256 * 4 / (2 * num_kv_heads), MLLM_ERR_UNSUPPORTED, fn + ": too many tokens");
  return MLLM_OK;
}

int launch_append(const std::string& fn, BlocksArgs a, int form, int dtype, hipStream_t st) {
  const bool small = a.n <= kSmallStep;
  const int64_t window = small ? 4 : kWindow;
  const int64_t pool = (a.n + window - 1) / window * 2 * a.hkv;
  const int64_t waves = pool + (form == kPlain ? 0 : ((int64_t)a.n * a.H + 3) / 4);
  MLLM_REQUIRE((waves + 3) / 4 <= kMaxGroups256, MLLM_ERR_UNSUPPORTED, fn + ": too many tokens");
  a.pool_waves = (unsigned)pool;
  const unsigned grid = (unsigned)((waves + 3) / 4);
  auto of_window = [&](auto tag, auto kind) {
    using T = decltype(tag);
    constexpr int FORM = decltype(kind)::value;
    if (small)
      append_fp8_blocks_kernel<T, FORM, false><<<grid, 256, 0, st>>>(a);
    else
      append_fp8_blocks_kernel<T, FORM, true><<<grid, 256, 0, st>>>(a);
  };
  auto of_form = [&](auto tag) {
    if (form == kPlain)
      of_window(tag, std::integral_constant<int, kPlain>{});
    else if (form == kRope)
      of_window(tag, std::integral_constant<int, kRope>{});
    else
      of_window(tag, std::integral_constant<int, kNormRope>{});
  };
  if (dtype == MLLM_DTYPE_BF16)
    of_form(BF16{});
  else
    of_form(F16{});
  return check_launch(fn.c_str());
}

}  // namespace

// mllm_qk_norm_rope_kv_append's part for this pool: its checks are that entry point's.
int rope_append_fp8_blocks(const std::string& fn, const mllm_rope_append& r, const void* q_norm, const void* k_norm, float eps,
                           void* stream) {
  const int rc = check_blocks(fn, r.dtype, r.num_tokens, r.num_blocks, r.block_size, r.num_kv_heads, r.head_dim);
  if (rc != MLLM_OK) return rc;
  BlocksArgs a{};
  a.k = (const char*)r.k, a.k_st = 2 * r.k_stride_tok, a.k_sh = 2 * r.k_stride_head;
  a.v = (const char*)r.v, a.v_st = 2 * r.v_stride_tok, a.v_sh = 2 * r.v_stride_head;
  a.kc = (char*)r.k_cache, a.vc = (char*)r.v_cache;
  a.ks = (uint8_t*)r.k_scales, a.vs = (uint8_t*)r.v_scales;
  a.num_slots = r.num_blocks * r.block_size;
  a.slots = r.slot_mapping;
  a.hkv = r.num_kv_heads, a.bs = r.block_size, a.bs_shift = __builtin_ctz((unsigned)r.block_size);
  a.n = (unsigned)r.num_tokens;
  a.q = (const char*)r.q, a.q_st = 2 * r.q_stride_tok, a.q_sh = 2 * r.q_stride_head;
  a.cos = (const char*)r.cos, a.sin = (const char*)r.sin, a.cs_st = 2 * r.cs_stride_tok;
  a.wq = (const char*)q_norm, a.wk = (const char*)k_norm, a.eps = eps;
  a.q_out = (char*)r.q_out, a.qo_st = 2 * r.q_out_stride_tok, a.qo_sh = 2 * r.q_out_stride_head;
  a.H = r.num_heads;
  return launch_append(fn, a, q_norm ? kNormRope : kRope, r.dtype, reinterpret_cast<hipStream_t>(stream));
}

}  // namespace mllm

extern "C" int mllm_kv_append_fp8_blocks(const void* k, int64_t k_stride_tok, int64_t k_stride_head, const void* v,
                                         int64_t v_stride_tok, int64_t v_stride_head, int32_t src_dtype, void* k_cache,
                                         void* v_cache, void* k_scales, void* v_scales, int64_t num_blocks,
                                         int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                                         const int64_t* slot_mapping, int64_t num_tokens, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_kv_append_fp8_blocks";
  const int rc = check_blocks(fn, src_dtype, num_tokens, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != MLLM_OK) return rc;
  if (num_tokens == 0) return MLLM_OK;
  MLLM_REQUIRE(k && v && k_cache && v_cache && k_scales && v_scales && slot_mapping, MLLM_ERR_INVALID,
               fn + ": null pointer");
  MLLM_REQUIRE(((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 &&
                   (k_stride_tok | k_stride_head | v_stride_tok | v_stride_head) % 8 == 0,
               MLLM_ERR_UNSUPPORTED, fn + ": rows must be 16-byte aligned");
  BlocksArgs a{};
  a.k = (const char*)k, a.k_st = 2 * k_stride_tok, a.k_sh = 2 * k_stride_head;
  a.v = (const char*)v, a.v_st = 2 * v_stride_tok, a.v_sh = 2 * v_stride_head;
  a.kc = (char*)k_cache, a.vc = (char*)v_cache;
  a.ks = (uint8_t*)k_scales, a.vs = (uint8_t*)v_scales;
  a.num_slots = num_blocks * block_size;
  a.slots = slot_mapping;
  a.hkv = num_kv_heads, a.bs = block_size, a.bs_shift = __builtin_ctz((unsigned)block_size);
  a.n = (unsigned)num_tokens;
  return launch_append(fn, a, kPlain, src_dtype, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int mllm_kv_read_fp8_blocks(const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                                       int64_t num_blocks, int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                                       const int64_t* slots, int64_t num_slots, int32_t dtype, void* k_out, void* v_out,
                                       void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_kv_read_fp8_blocks";
  const int rc = check_blocks(fn, dtype, num_slots, num_blocks, block_size, num_kv_heads, head_dim);
  if (rc != MLLM_OK) return rc;
  if (num_slots == 0) return MLLM_OK;
  MLLM_REQUIRE(k_cache && v_cache && k_scales && v_scales && slots && k_out && v_out, MLLM_ERR_INVALID,
               fn + ": null pointer");
  MLLM_REQUIRE(((uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0,
               MLLM_ERR_UNSUPPORTED, fn + ": rows must be 16-byte aligned");
  const int64_t groups = (num_slots * num_kv_heads * (kDh / 16) + 255) / 256;
  MLLM_REQUIRE(groups <= kMaxGroups256, MLLM_ERR_UNSUPPORTED, fn + ": too many slots");
  const dim3 grid((unsigned)groups, 2);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto launch = [&](auto tag) {
    read_fp8_blocks_kernel<decltype(tag)><<<grid, 256, 0, st>>>(
        (const char*)k_cache, (const char*)v_cache, (const uint8_t*)k_scales, (const uint8_t*)v_scales,
        num_blocks * block_size, num_kv_heads, __builtin_ctz((unsigned)block_size), slots, num_slots, (char*)k_out,
        (char*)v_out);
  };
  if (dtype == MLLM_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  return check_launch(fn.c_str());
}
