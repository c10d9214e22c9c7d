// Split-KV paged decode attention over a 4-bit pool (kv_fp4.hip has its layout): the plan, the segments and the online
// softmax of decode.hip's kernels, with K and V widened to 16 bits in registers.
//
// A wavefront takes NH adjacent KV heads (two where their query heads fit 16 MFMA columns, else one), so that one softmax
// serves the columns of both.  Column c is query head c of the NH G; lane l is (c, g) = (l % 16, l / 16).
//   S^T[16 tok x 16] = K_h . Q^T[128 x 16] for each head h: 4 x v_mfma_f32_16x16x32, k-step kk at dims 32 g + 8 kk .. +7, so a
//     lane's 16 bytes of K row c are the dim block g of token c, under one scale.  All columns are multiplied with each
//     head and a column keeps its own head's: no masked copies of Q.
//   O^T += V^T . P^T: lane (c, g) loads tokens 4 g .. + 3 at bytes 4 NH c .. of the heads' joint row, D = 8 NH dims under
//     one scale (a dword holds the four tokens').  Product m is element m of those: row r of it is dim D r + m of the joint
//     row, and a column keeps the rows of its own head, those of the lanes with g NH / 4 = its head.
// K and V are exact in the 16-bit type, the accumulators, the maximum and the sum are fp32.  P is rounded to bf16, half a
// step as the output's own rounding (the sum l takes the unrounded P); in fp16, whose output keeps three more bits, P goes
// in two parts, 22 bits together.
//
// Bound by memory and the vector pipes together.  Measured on 256 rows of 128-4,096 tokens (32 heads on 8, 630 MB), the
// pass with its merge, us: 114 at 5.5 TB/s; the same loads without arithmetic 108; the arithmetic without loads 90.  With
// four heads a wavefront the accumulators spill: 130; one wavefront a bin and head pair instead of workgroups that share
// a bin: 155; 32-token tiles with one set of registers: 140; two tiles ahead 116; three wavefronts a SIMD 119; P in two parts
// for bf16 too 3 - 4% more, also as one product of depth 32 over V taken twice.  A small step is a chain of dependent reads (plan,
// block ids, tile, partials): four rows of 100-700 tokens 10.8 us from a graph, in bins of 2 pages; of 4 pages 12.1, of 8 13.6.
#include "decode_slices.h"

namespace mllm {
namespace {

template <int N>
struct Words {  // N dwords loaded together
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> ldw(const char* p) {
  Words<N> r;
  if constexpr (N == 2) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.w[0] = v[0], r.w[1] = v[1];
  } else {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}

constexpr int kRowBytes4 = kHeadDim / 2, kBlocks4 = kHeadDim / kFp4Block;

// Byte h of a scale word where the conversions read it (bits 30:23 of their operand; they ignore the others).
__device__ __forceinline__ float scale_of(uint32_t w, int h) {
  return __uint_as_float(h < 3 ? w << (23 - 8 * h) : w >> 1);
}

template <int NH>
struct Fp4Pages {
  // A tile of 16 tokens, as the pool stores it.
  struct Tile {
    u32x4 k[NH];     // token c, head h, dims 32 g .. + 31
    Words<NH> v[4];  // token 4 g + i, D dims of the joint row
    uint32_t ks;     // token c, dim block g: the scales of the NH heads
    uint32_t vs;     // tokens 4 g .. + 3: their scales, a byte each
  };
  // What a lane adds to a sub-tile's uniform addresses, in bytes.
  struct Lane {
    unsigned k, ks, v, vs;
  };
  static __device__ __forceinline__ Lane lane(const SlicesArgs& a, int c, int g) {
    const unsigned st = (unsigned)(a.Hkv * kRowBytes4);
    return {(unsigned)c * st + 16u * g, (unsigned)((c * kBlocks4 + g) * a.Hkv), (unsigned)(4 * g) * st + 4u * NH * c,
            (unsigned)((8 * NH * c / kFp4Block) * a.bs + 4 * g)};
  }
  // First of the eight dims a lane holds at k-step kk.
  static __device__ __forceinline__ int q_dim(int kk, int g) { return 32 * g + 8 * kk; }

  static __device__ __forceinline__ void load(const SlicesArgs& a, int kvh0, const Lane& at, int blk, int sub, Tile& r) {
    const int64_t tok = (int64_t)blk * a.bs + 16 * sub;  // the tile's first slot
    const char* kp = a.kc + (tok * a.Hkv + kvh0) * kRowBytes4;
    const char* vp = a.vc + (tok * a.Hkv + kvh0) * kRowBytes4;
    const unsigned st = (unsigned)(a.Hkv * kRowBytes4);
#pragma unroll
    for (int h = 0; h < NH; ++h) r.k[h] = ld16_nt(kp + (h * kRowBytes4 + at.k));
    const uint8_t* sp = a.ks + tok * a.Hkv * kBlocks4 + kvh0;
    if constexpr (NH == 2)
      r.ks = *reinterpret_cast<const uint16_t*>(sp + at.ks);
    else
      r.ks = sp[at.ks];
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = ldw<NH>(vp + (i * st + at.v));
    r.vs = *reinterpret_cast<const uint32_t*>(a.vs + ((int64_t)blk * a.Hkv + kvh0) * kBlocks4 * a.bs + 16 * sub + at.vs);
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
      for (int h = 0; h < NH; ++h) d[h] = Mfma<T>::m16x16x32(fp4x8_to<T>(r.k[h][kk], scale_of(r.ks, h)), qk, d[h]);
    }
    float s[4], vs[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x = d[0][i];
#pragma unroll
      for (int h = 1; h < NH; ++h) x = myhead == h ? d[h][i] : x;
      s[i] = x * scale_log2;
      vs[i] = scale_of(r.vs, i);
    }
    if (tpos0 + 16 > len) {  // the row's last, partly filled tile: mask the keys past its end, zero their V
      const int tpos = tpos0 + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (tpos + i >= len) {
          s[i] = -INFINITY;
          vs[i] = 1.f;  // whatever the slot's scale says, NaN included
#pragma unroll
          for (int h = 0; h < NH; ++h) r.v[i].w[h] = 0;
        }
      }
    }
    const auto pt = softmax_tile<T, std::is_same<T, F16>::value>(s, m_run, l_run, o);
#pragma unroll
    for (int j = 0; j < NH; ++j)  // dword j of the four V rows, widened just in time
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = fp4x2_to<T>(r.v[i].w[j], vs[i], e);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const u32x2 vf = u32x2{pick_halves(w[0], hf, w[1], hf), pick_halves(w[2], hf, w[3], hf)};
          const int m = 8 * j + 2 * e + hf;
          add_pv(vf, pt, o[m]);
        }
      }
  }
};

}  // namespace
}  // namespace mllm

extern "C" int mllm_paged_decode_fp4(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
                                     const void* v_cache, const void* k_scales, const void* v_scales,
                                     int64_t num_blocks, int32_t block_size, int32_t num_heads, int32_t num_kv_heads,
                                     int32_t head_dim, const int32_t* qo_indptr, const int32_t* kv_indices,
                                     const int32_t* decode_work, int32_t num_decode_work, const int32_t* merge_work,
                                     int32_t num_merge_work, int32_t pages_per_split,
                                     float softmax_scale, int32_t dtype, void* out, int64_t out_stride_tok,
                                     int64_t out_stride_head, void* workspace, int64_t workspace_bytes, void* stream) {
  return mllm::paged_decode_slices<mllm::Fp4Pages, 16>(
      "mllm_paged_decode_fp4", mllm::kRowBytes4, q, q_stride_tok, q_stride_head, k_cache, v_cache, k_scales, v_scales,
      num_blocks, block_size, num_heads, num_kv_heads, head_dim, qo_indptr, kv_indices, decode_work, num_decode_work,
      merge_work, num_merge_work, pages_per_split, softmax_scale, dtype, out, out_stride_tok, out_stride_head, workspace,
      workspace_bytes, stream);
}
