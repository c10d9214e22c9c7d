// Split-KV paged decode attention over an 8-bit pool with a scale for each block of tokens and head (kv_fp8_blocks.hip has its
// layout): the kernel of decode_slices.h, with K and V widened to 16 bits in registers.
//
// A wavefront takes NH adjacent KV heads (two where their query heads fit 16 MFMA columns, else one), so that one softmax
// serves the columns of both.  Column c is query head c of the NH G; lane l is (c, g) = (l % 16, l / 16).
//   S^T[16 tok x 16] = K_h . Q^T[128 x 16] for each head h: 4 x v_mfma_f32_16x16x32.  A lane holds 16 bytes of row c in each
//     64-byte half: half p at dims 64 p + 16 g, of which k-step 2 p + t takes eight, so a load reads 64 bytes of a row together.
//     All columns are multiplied with each head and a column keeps its own head's.
//   O^T += V^T . P^T: lane (c, g) loads tokens 4 g .. + 3 at bytes 8 NH c .. of the heads' joint row, D = 8 NH dims of one head.
//     Product m is element m of those: row r of it is dim D r + m of the joint row, and a column keeps the rows of its own head.
// A tile lies in one page, so its scales are one byte for each of the heads: read through the scalar cache and applied by the
// conversions.  Every code times its scale is exact in the 16-bit type.  P goes into
// the products in two 16-bit parts, 16 or 22 bits together: one part would round it to 8 bits in bf16, 40% more error in the
// output than its own rounding, and save 0.3% of a large step (190.5 against 191.1 us).
//
// Bound by HBM reads on large steps: 256 rows of 128-4,096 tokens, 1.18 GB, 185-190 us (6.3 TB/s).  Three rows of 50,000-120,000
// tokens over 2 KV heads in fp16, 126 MB: 24.4 us (5.2 TB/s).  Small steps are a chain of dependent reads (plan, page ids, tile):
// 4 rows of 100-700 tokens 8.3 us, the merge 2.6.
#include "decode_slices.h"

namespace mllm {
namespace {

constexpr int kRowBytes8 = kHeadDim;

template <int N>
struct Row {  // 8 N codes of a V row
  uint32_t w[2 * N];
};
template <int N>
__device__ __forceinline__ Row<N> ldrow(const char* p) {
  Row<N> r;
  if constexpr (N == 2) {
    const u32x4 v = ld16_nt(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = v[i];
  } else {
    const u32x2 v = ldkv8<true>(p);
    r.w[0] = v[0], r.w[1] = v[1];
  }
  return r;
}

template <int NH>
struct Fp8Pages {
  // A tile of 16 tokens, as the pool stores it.
  struct Tile {
    u32x4 k[2 * NH];  // token c, head h, dims 64 p + 16 g .. + 15: k[2 h + p]
    Row<NH> v[4];     // token 4 g + i, D dims of the joint row
    uint32_t ks, vs;  // the heads' scales, a byte each (uniform)
  };
  // What a lane adds to a sub-tile's uniform addresses, in bytes.
  struct Lane {
    unsigned k, v;
  };
  static __device__ __forceinline__ Lane lane(const SlicesArgs& a, int c, int g) {
    const unsigned st = (unsigned)(a.Hkv * kRowBytes8);
    return {(unsigned)c * st + 16u * g, (unsigned)(4 * g) * st + 8u * NH * c};
  }
  // First of the eight dims a lane holds at k-step kk.
  static __device__ __forceinline__ int q_dim(int kk, int g) { return 64 * (kk >> 1) + 16 * g + 8 * (kk & 1); }

  // The scale bytes from (block, head) on, in the low bits; NH of them lie in one dword (an even head of an even count).
  static __device__ __forceinline__ uint32_t scale_word(const uint8_t* s, int64_t at) {
    typedef const __attribute__((address_space(4))) uint32_t ConstU32;
    return ((ConstU32*)s)[at >> 2] >> (8 * (int)(at & 3));
  }
  // A scale byte at bits 7:0 where the conversions read it (bits 30:23 of their operand; they ignore the others).
  static __device__ __forceinline__ float scale_of(uint32_t w) { return __uint_as_float(w << 23); }

  static __device__ __forceinline__ void load(const SlicesArgs& a, int kvh0, const Lane& at, int blk, int sub, Tile& r) {
    const int64_t tok = (int64_t)blk * a.bs + 16 * sub;  // the tile's first slot
    const char* kp = a.kc + (tok * a.Hkv + kvh0) * kRowBytes8;
    const char* vp = a.vc + (tok * a.Hkv + kvh0) * kRowBytes8;
    const unsigned st = (unsigned)(a.Hkv * kRowBytes8);
#pragma unroll
    for (int p = 0; p < 2 * NH; ++p) r.k[p] = ld16_nt(kp + (64 * p + at.k));
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = ldrow<NH>(vp + (i * st + at.v));
    const int64_t s = (int64_t)blk * a.Hkv + kvh0;
    r.ks = scale_word(a.ks, s);
    r.vs = scale_word(a.vs, s);
  }

  // One 16-token tile: scores, online-softmax update, PV.  `q`: this lane's Q^T operands in LDS.
  template <typename T>
  static __device__ __forceinline__ void consume(Tile& r, const u32x4* q, int myhead, float scale_log2, int tpos0, int len, int c,
                                                 int g, float& m_run, float& l_run, f32x4 (&o)[8 * NH]) {
    f32x4 d[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) d[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const u32x4 qk = q[64 * kk];
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const u32x4& k = r.k[2 * h + (kk >> 1)];
        d[h] = Mfma<T>::m16x16x32(fp8x8_to<T>(k[2 * (kk & 1)], k[2 * (kk & 1) + 1], scale_of(r.ks >> (8 * h))), qk, d[h]);
      }
    }
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = d[0][i];
#pragma unroll
      for (int h = 1; h < NH; ++h) x = myhead == h ? d[h][i] : x;
      s[i] = x * scale_log2;
    }
    if (tpos0 + 16 > len) {  // the row's last, partly filled tile: mask the keys past its end, zero their V
      const int tpos = tpos0 + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (tpos + i >= len) {
          s[i] = -INFINITY;
#pragma unroll
          for (int w = 0; w < 2 * NH; ++w) r.v[i].w[w] = 0;
        }
      }
    }
    const auto pt = softmax_tile<T, true>(s, m_run, l_run, o);
    const float vs = scale_of(NH == 2 ? r.vs >> (c & 8) : r.vs);  // of the head whose dims the lane holds
#pragma unroll
    for (int j = 0; j < 2 * NH; ++j) {  // dword j of the four V rows, widened just in time
      u32x2 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = fp8x4_to<T>(r.v[i].w[j], vs);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int dw = e >> 1, hf = e & 1;
        add_pv(u32x2{pick_halves(w[0][dw], hf, w[1][dw], hf), pick_halves(w[2][dw], hf, w[3][dw], hf)}, pt, o[4 * j + e]);
      }
    }
  }
};

}  // namespace
}  // namespace mllm

extern "C" int mllm_paged_decode_fp8_blocks(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
                                     const void* v_cache, const void* k_scales, const void* v_scales,
                                     int64_t num_blocks, int32_t block_size, int32_t num_heads, int32_t num_kv_heads,
                                     int32_t head_dim, const int32_t* qo_indptr, const int32_t* kv_indices,
                                     const int32_t* decode_work, int32_t num_decode_work, const int32_t* merge_work,
                                     int32_t num_merge_work, int32_t pages_per_split,
                                     float softmax_scale, int32_t dtype, void* out, int64_t out_stride_tok,
                                     int64_t out_stride_head, void* workspace, int64_t workspace_bytes, void* stream) {
  return mllm::paged_decode_slices<mllm::Fp8Pages, 4>(
      "mllm_paged_decode_fp8_blocks", mllm::kRowBytes8, q, q_stride_tok, q_stride_head, k_cache, v_cache, k_scales, v_scales,
      num_blocks, block_size, num_heads, num_kv_heads, head_dim, qo_indptr, kv_indices, decode_work, num_decode_work,
      merge_work, num_merge_work, pages_per_split, softmax_scale, dtype, out, out_stride_tok, out_stride_head, workspace,
      workspace_bytes, stream);
}
