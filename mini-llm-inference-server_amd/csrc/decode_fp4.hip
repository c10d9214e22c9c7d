// Split-KV paged decode attention over a 4-bit pool (kv_fp4.hip has its layout): the plan, the segments and the online
// softmax of decode.hip's kernels, with K and V widened to 16 bits in registers.
//
// A page of 4-bit keys is a quarter of a 16-bit one, so a wavefront takes NH adjacent KV heads (4, 2 or 1, with at most
// 16 query heads together): a 16-token tile of four heads is then 8.5 KB in the same load shapes as one 16-bit head's
// 8 KB, and one softmax serves the 16 MFMA columns of all its heads.  Column c is query head c of the NH G; lane l is
// (c, g) = (l % 16, l / 16).
//   S^T[16 tok x 16] = K_h . Q^T for each head h: 4 x v_mfma_f32_16x16x32, k-step kk at dims 32 g + 8 kk .. +7, so a
//     lane's 16 bytes of K row c are the dim block g of token c, under one scale.  All columns are multiplied with each
//     head and a column keeps its own head's: no masked copies of Q.
//   O^T += V^T . P^T: lane (c, g) loads tokens 4 g .. + 3 at bytes 4 NH c .. of the heads' joint row, D = 8 NH dims under
//     one scale (a dword holds the four tokens').  Product m is element m of those: row r of it is dim D r + m of the joint
//     row, and a column keeps the rows of its own head, those of the lanes with g NH / 4 = its head.
// K and V are exact in the 16-bit type; P is rounded to it (the sum l takes the unrounded P), the accumulators, the maximum
// and the sum are fp32.
#include <math.h>

#include "decode_common.h"

namespace mllm {
namespace {

struct DecodeFp4Args {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const char *kc, *vc;        // codes
  const uint8_t *ks, *vs;     // scales
  int64_t num_blocks;
  int bs, H, Hkv, G, HG;
  const int32_t* kv_indices;
  const int4* work;
  float scale_log2;  // softmax scale x log2(e)
  uint16_t* out;
  int64_t o_st, o_sh;
  float* part_o;
  float2* part_ml;
};

template <int N>
struct Words {  // N dwords loaded together
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> ldw(const char* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const u32x4 v = ld16_nt(p);
    r.w[0] = v[0], r.w[1] = v[1], r.w[2] = v[2], r.w[3] = v[3];
  } else if constexpr (N == 2) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.w[0] = v[0], r.w[1] = v[1];
  } else {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}

template <int NH>
struct Fp4Tile {
  u32x4 k[NH];     // token c, head h, dims 32 g .. + 31
  Words<NH> ks;    // token c: the four dim blocks' scales of each head
  Words<NH> v[4];  // token 4 g + i, D dims of the joint row
  uint32_t vs;     // their scales, one byte per token
};

constexpr int kRowBytes4 = kHeadDim / 2, kBlocks4 = kHeadDim / kFp4Block;

// What a lane adds to a tile's uniform addresses, in bytes.
struct Fp4Lane {
  unsigned k, ks, v, vs;
};

template <int NH>
__device__ __forceinline__ void load_tile4(const DecodeFp4Args& a, int kvh0, const Fp4Lane& at, const PageIds& pages,
                                           LoadCursor cur, Fp4Tile<NH>& r) {
  int blk = page_id(pages, cur.page);
  if ((unsigned)blk >= (unsigned)a.num_blocks) blk = 0;  // never taken with valid metadata; keeps reads in the pool
  const int64_t tok = (int64_t)blk * a.bs + 16 * cur.sub;  // the tile's first slot
  const int64_t row = tok * a.Hkv + kvh0;                  // (slot, head) rows
  const char* kp = a.kc + row * kRowBytes4;
  const char* vp = a.vc + row * kRowBytes4;
  const unsigned st = (unsigned)(a.Hkv * kRowBytes4);
#pragma unroll
  for (int h = 0; h < NH; ++h) r.k[h] = ld16_nt(kp + h * kRowBytes4 + at.k);
  r.ks = ldw<NH>(reinterpret_cast<const char*>(a.ks) + row * kBlocks4 + at.ks);
#pragma unroll
  for (int i = 0; i < 4; ++i) r.v[i] = ldw<NH>(vp + (i * st + at.v));
  r.vs = *reinterpret_cast<const uint32_t*>(a.vs + ((int64_t)blk * a.Hkv + kvh0) * kBlocks4 * a.bs + 16 * cur.sub + at.vs);
}

template <typename T, int NH>
__device__ __forceinline__ void consume_tile4(Fp4Tile<NH>& r, const u32x4 (&qf)[4], int myhead, float scale_log2, int tpos0,
                                              int len, int g, float& m_run, float& l_run, f32x4 (&o)[8 * NH]) {
  f32x4 d[NH];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    const float ks = e8m0_to_f32((r.ks.w[h] >> (8 * g)) & 0xffu);
    d[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) d[h] = Mfma<T>::m16x16x32(fp4x8_to<T>(r.k[h][kk], ks), qf[kk], d[h]);
  }
  float s[4], vs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = d[0][i];
#pragma unroll
    for (int h = 1; h < NH; ++h) x = myhead == h ? d[h][i] : x;
    s[i] = x * scale_log2;
    vs[i] = e8m0_to_f32((r.vs >> (8 * i)) & 0xffu);
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
  const float mx = maximum_xor32(maximum_xor16(maximum(maximum(s[0], s[1]), maximum(s[2], s[3]))));
  if (__any(mx > m_run + 8.f)) {  // lazy rescale, as in decode.hip
    const float m_new = fmaxf(m_run, mx);
    const float alpha = fast_exp2(m_run - m_new);
    l_run *= alpha;
#pragma unroll
    for (int m = 0; m < 8 * NH; ++m) o[m] *= alpha;
    m_run = m_new;
  }
  float p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = fast_exp2(s[i] - m_run);
  l_run += sum_xor32(sum_xor16((p[0] + p[1]) + (p[2] + p[3])));
  const u32x2 pfrag = u32x2{pack2<T>(p[0], p[1]), pack2<T>(p[2], p[3])};
#pragma unroll
  for (int j = 0; j < NH; ++j) {  // dword j of the four V rows, widened just in time
    u32x4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = fp4x8_to<T>(r.v[i].w[j], vs[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int dw = e >> 1, hf = e & 1;
      const u32x2 vfrag = u32x2{pick_halves(w[0][dw], hf, w[1][dw], hf), pick_halves(w[2][dw], hf, w[3][dw], hf)};
      o[8 * j + e] = Mfma<T>::m16x16x16(vfrag, pfrag, o[8 * j + e]);
    }
  }
}

template <typename T, int NH, int W, int OCC>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void decode_fp4_kernel(
    const DecodeFp4Args a) {
  constexpr int D = 8 * NH;
  const int lane = threadIdx.x & 63;
  const int hg = blockIdx.x % a.HG, bin = blockIdx.x / a.HG;
  const int kvh0 = NH * (hg * W + (threadIdx.x >> 6));
  if (kvh0 >= a.Hkv) return;  // wave-uniform
  const int nbins = plan_rec(a.work, 0).x;
  const int4 bw = plan_rec(a.work, 1 + bin);
  if (bin >= nbins) return;
  const int4* segs = a.work + bw.z;
  const int tpp = a.bs >> 4;
  const int c = lane & 15, g = lane >> 4;
  const bool qvalid = c < NH * a.G;
  const int myhead = qvalid ? c / a.G : 0;
  const int qhead = kvh0 * a.G + (qvalid ? c : 0);
  const int flat = D * c;  // first dim of this lane's part of the joint V row
  const unsigned st = (unsigned)(a.Hkv * kRowBytes4);
  const Fp4Lane at{(unsigned)c * st + 16u * g, (unsigned)(c * a.Hkv * kBlocks4), (unsigned)(4 * g) * st + 4u * NH * c,
                   (unsigned)((flat / kFp4Block) * a.bs + 4 * g)};

  auto load_q = [&](int qrow, u32x4 (&qf)[4]) {
    const char* qp = reinterpret_cast<const char*>(a.q + (int64_t)qrow * a.q_st + (int64_t)qhead * a.q_sh);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const u32x4 v = ld16(qp + 2 * (32 * g + 8 * kk));
      qf[kk] = qvalid ? v : u32x4{0, 0, 0, 0};
    }
  };

  const int glast = bw.y - 1;  // next-segment loads as in decode_kernel: unconditional
  int gi = bw.x;
  SegRec cur = seg_rec(segs, gi);
  SegRec nxt = seg_rec(segs, min(gi + 1, glast));
  PageIds pages = load_page_ids(a.kv_indices, cur.r0, lane);
  u32x4 qf[4];
  load_q(cur.r1.x, qf);
  Fp4Tile<NH> tile, ahead;
  LoadCursor pos;
  load_tile4<NH>(a, kvh0, at, pages, pos, tile);
  pos.advance(tpp);

  while (true) {
    gi = __builtin_amdgcn_readfirstlane(gi);
    const bool has_next = gi < glast;
    const int tok0 = cur.r0.z * a.bs, len = cur.r0.w;
    const int ntiles = max(min(len, tok0 + cur.r0.y * a.bs) - tok0 + 15, 0) >> 4;
    const PageIds next_pages = load_page_ids(a.kv_indices, nxt.r0, lane);
    u32x4 next_q[4];
    load_q(nxt.r1.x, next_q);
    const SegRec after = seg_rec(segs, min(gi + 2, glast));
    float m_run = -INFINITY, l_run = 0.f;
    f32x4 o[D];
#pragma unroll
    for (int m = 0; m < D; ++m) o[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool next_loaded = false;
    for (int t = 0; t < ntiles; ++t) {
      if (t + 1 < ntiles) {
        load_tile4<NH>(a, kvh0, at, pages, pos, ahead);
        pos.advance(tpp);
      } else if (has_next) {
        load_tile4<NH>(a, kvh0, at, next_pages, LoadCursor{}, ahead);
        next_loaded = true;
      }
      consume_tile4<T, NH>(tile, qf, myhead, a.scale_log2, tok0 + t * 16, len, g, m_run, l_run, o);
      tile = ahead;
    }

    // lane (c, g): o[m][i] is dim D (4 g + i) + m of the joint row; kept where that is the column's own head
    if (qvalid && g * NH / 4 == myhead) {
      const int head = kvh0 * a.G + c, d0 = (4 * D * g) % kHeadDim, slot = cur.r1.y;
      if (slot < 0) {
        const float inv = 1.f / l_run;
        char* op = reinterpret_cast<char*>(a.out + (int64_t)cur.r1.x * a.o_st + (int64_t)head * a.o_sh + d0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int m = 0; m < D; m += 8)
            st16(op + 2 * (D * i + m),
                 u32x4{pack2<T>(o[m][i] * inv, o[m + 1][i] * inv), pack2<T>(o[m + 2][i] * inv, o[m + 3][i] * inv),
                       pack2<T>(o[m + 4][i] * inv, o[m + 5][i] * inv), pack2<T>(o[m + 6][i] * inv, o[m + 7][i] * inv)});
      } else {
        const int64_t row = (int64_t)slot * a.H + head;
        float* po = a.part_o + row * kHeadDim + d0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int m = 0; m < D; m += 4)
            *reinterpret_cast<f32x4*>(po + D * i + m) = f32x4{o[m][i], o[m + 1][i], o[m + 2][i], o[m + 3][i]};
        if (d0 == 0) a.part_ml[row] = make_float2(m_run, l_run);
      }
    }
    if (!has_next) break;
    ++gi;
    cur = nxt;
    nxt = after;
    pages = next_pages;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[kk] = next_q[kk];
    pos = LoadCursor{};
    if (!next_loaded)  // this segment had no tile to load it behind
      load_tile4<NH>(a, kvh0, at, pages, pos, tile);
    pos.advance(tpp);
  }
}

constexpr int kWavesFp4 = 2;  // wavefronts per workgroup: with four heads each, eight KV heads read whole pages
constexpr int kOccupancyFp4 = 2;

// KV heads per wavefront.
int fp4_heads(int num_kv_heads, int group) {
  if (num_kv_heads % 4 == 0 && 4 * group <= 16) return 4;
  return num_kv_heads % 2 == 0 && 2 * group <= 16 ? 2 : 1;
}

template <typename T>
int launch_fp4(DecodeFp4Args a, int n_work, hipStream_t st) {
  const unsigned bins = (unsigned)max_bins(n_work);
  if (bins == 0) return MLLM_OK;
  const int nh = fp4_heads(a.Hkv, a.G);
  a.HG = (a.Hkv + nh * kWavesFp4 - 1) / (nh * kWavesFp4);
  const unsigned grid = bins * (unsigned)a.HG;
  if (nh == 4)
    decode_fp4_kernel<T, 4, kWavesFp4, kOccupancyFp4><<<grid, 64 * kWavesFp4, 0, st>>>(a);
  else if (nh == 2)
    decode_fp4_kernel<T, 2, kWavesFp4, kOccupancyFp4><<<grid, 64 * kWavesFp4, 0, st>>>(a);
  else
    decode_fp4_kernel<T, 1, kWavesFp4, kOccupancyFp4><<<grid, 64 * kWavesFp4, 0, st>>>(a);
  return check_launch("mllm_paged_decode_fp4");
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_paged_decode_fp4(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
                                     const void* v_cache, const void* k_scales, const void* v_scales,
                                     int64_t num_blocks, int32_t block_size, int32_t num_heads, int32_t num_kv_heads,
                                     int32_t head_dim, const int32_t* kv_indices, const int32_t* decode_work,
                                     int32_t num_decode_work, int32_t num_merge_work, int32_t pages_per_split,
                                     float softmax_scale, int32_t dtype, void* out, int64_t out_stride_tok,
                                     int64_t out_stride_head, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_paged_decode_fp4";
  MLLM_REQUIRE(dtype == MLLM_DTYPE_BF16 || dtype == MLLM_DTYPE_F16, MLLM_ERR_UNSUPPORTED,
               fn + ": dtype must be bfloat16 or float16");
  MLLM_REQUIRE(head_dim == kHeadDim, MLLM_ERR_UNSUPPORTED, fn + ": head_dim must be 128");
  MLLM_REQUIRE(block_size > 0 && block_size % 16 == 0, MLLM_ERR_UNSUPPORTED,
               fn + ": block_size must be a multiple of 16");
  MLLM_REQUIRE(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0, MLLM_ERR_INVALID,
               fn + ": num_heads must be a multiple of num_kv_heads");
  MLLM_REQUIRE(num_heads / num_kv_heads <= 16, MLLM_ERR_UNSUPPORTED, fn + ": at most 16 query heads per KV head");
  MLLM_REQUIRE(pages_per_split >= 1 && pages_per_split <= kMaxSplitPages, MLLM_ERR_INVALID,
               fn + ": pages_per_split must be in [1, 192]");
  MLLM_REQUIRE((int64_t)block_size * num_kv_heads * kRowBytes4 < (1ll << 31), MLLM_ERR_UNSUPPORTED,
               fn + ": KV block too large");
  MLLM_REQUIRE(num_decode_work >= 0 && num_merge_work >= 0, MLLM_ERR_INVALID, fn + ": negative count");
  if (num_decode_work == 0) return MLLM_OK;
  MLLM_REQUIRE(q && k_cache && v_cache && k_scales && v_scales && out && kv_indices && decode_work, MLLM_ERR_INVALID,
               fn + ": null pointer");
  const int64_t need = num_merge_work ? mllm_decode_workspace_bytes(num_decode_work, num_heads, head_dim) : 0;
  MLLM_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), MLLM_ERR_INVALID, fn + ": workspace too small");
  MLLM_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)k_scales |
                (uintptr_t)v_scales) % 16 == 0 &&
                   (q_stride_tok | q_stride_head | out_stride_tok | out_stride_head) % 8 == 0,
               MLLM_ERR_UNSUPPORTED, fn + ": q, out and pools need 16-byte aligned rows");
  DecodeFp4Args a;
  a.q = static_cast<const uint16_t*>(q);
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.kc = static_cast<const char*>(k_cache);
  a.vc = static_cast<const char*>(v_cache);
  a.ks = static_cast<const uint8_t*>(k_scales);
  a.vs = static_cast<const uint8_t*>(v_scales);
  a.num_blocks = num_blocks;
  a.bs = block_size;
  a.H = num_heads;
  a.Hkv = num_kv_heads;
  a.G = num_heads / num_kv_heads;
  a.HG = 0;
  a.kv_indices = kv_indices;
  a.work = reinterpret_cast<const int4*>(decode_work);
  a.scale_log2 = softmax_scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.o_st = out_stride_tok;
  a.o_sh = out_stride_head;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) +
                                        (int64_t)partial_slots(num_decode_work) * num_heads * head_dim * 4);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == MLLM_DTYPE_BF16 ? launch_fp4<BF16>(a, num_decode_work, st) : launch_fp4<F16>(a, num_decode_work, st);
}
