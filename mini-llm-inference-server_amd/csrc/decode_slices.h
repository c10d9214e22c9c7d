// Split-KV paged decode over pools with block scales: the kernel that the 4-bit and the 8-bit pools share, its merge and its
// entry point's checks.  A pool comes in as `POOL<NH>` for wavefronts of NH KV heads: the registers of a 16-token tile
// (`Tile`), what a lane adds to a tile's uniform addresses (`Lane`, `lane`), the load (`load`), the dims of the Q^T operand
// (`q_dim`), and a tile's scores, softmax and P V (`consume`).
#pragma once

#include <math.h>

#include <string>
#include <type_traits>

#include "decode_common.h"

namespace mllm {
namespace {

struct SlicesArgs {
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

// What two 16-bit values (`hi`) leave of the floats they were rounded from, as such values.
template <typename T>
__device__ __forceinline__ uint32_t rest_of(float a, float b, uint32_t hi) {
  return pack2<T>(a - to_f32<T>((uint16_t)hi), b - to_f32<T>((uint16_t)(hi >> 16)));
}

// P of a tile for its products with V: one 16-bit value, or (SPLIT) two.
template <typename T, bool SPLIT>
struct TileP {
  u32x2 hi, lo;
};

// The online softmax over a tile's scores s (exp2 domain, masked): the running maximum, sum and accumulators brought up to
// it, and P.
template <typename T, bool SPLIT, int D>
__device__ __forceinline__ TileP<T, SPLIT> softmax_tile(float (&s)[4], float& m_run, float& l_run, f32x4 (&o)[D]) {
  const float mx = maximum_xor32(maximum_xor16(maximum(maximum(s[0], s[1]), maximum(s[2], s[3]))));
  if (__any(mx > m_run + 8.f)) {  // lazy rescale, as in decode.hip
    const float m_new = fmaxf(m_run, mx);
    const float alpha = fast_exp2(m_run - m_new);
    l_run *= alpha;
#pragma unroll
    for (int m = 0; m < D; ++m) o[m] *= alpha;
    m_run = m_new;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = fast_exp2(s[i] - m_run);
  l_run += sum_xor32(sum_xor16((s[0] + s[1]) + (s[2] + s[3])));
  TileP<T, SPLIT> p{u32x2{pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3])}, {0, 0}};
  if constexpr (SPLIT) p.lo = u32x2{rest_of<T>(s[0], s[1], p.hi[0]), rest_of<T>(s[2], s[3], p.hi[1])};
  return p;
}

// O += V P for one row m of products.
template <typename T, bool SPLIT>
__device__ __forceinline__ void add_pv(u32x2 v, const TileP<T, SPLIT>& p, f32x4& o) {
  o = Mfma<T>::m16x16x16(v, p.hi, o);
  if constexpr (SPLIT) o = Mfma<T>::m16x16x16(v, p.lo, o);
}

// A workgroup of eight wavefronts takes one bin and HGW groups of NH heads: wavefront w group w % HGW and the tiles w / HGW,
// + SL, .. of each segment, SL = 8 / HGW (bins then need be no shorter than one per CU, which keeps the partials few, and
// with four groups of two heads whole pages are read together).  Each wavefront has the next tile on its way while it works
// on one, across segment boundaries.  The slices' (m, l, O) of a segment meet in LDS, where each thread combines eight
// dims of one query head and writes the output, or the segment's partial when the row is cut.
constexpr int kWavesSlices = 8;
constexpr int kPartRow = kHeadDim + 4;  // floats of a slice's query head in LDS: O, then m and l

template <typename T, template <int> class POOL, int NH, int HGW>
__global__ __launch_bounds__(64 * kWavesSlices) __attribute__((amdgpu_waves_per_eu(kWavesSlices / 4, kWavesSlices / 4))) void decode_slices_kernel(
    const SlicesArgs a) {
  using P = POOL<NH>;
  constexpr int D = 8 * NH, SL = kWavesSlices / HGW, kRows = 16 * HGW;  // query heads' places in LDS
  __shared__ __attribute__((aligned(16))) float part[SL][kRows][kPartRow];
  __shared__ u32x4 qs[2][HGW][4][64];  // Q^T operands of this and the next segment, as their lanes read them
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hg = blockIdx.x % a.HG, bin = blockIdx.x / a.HG;
  const int slice = wave / HGW, grp = wave % HGW;
  const int kvh0 = NH * (hg * HGW + grp);
  const bool has_heads = kvh0 < a.Hkv;  // past the last group: the wavefront only joins the barriers
  const int nbins = plan_rec(a.work, 0).x;
  const int4 bw = plan_rec(a.work, 1 + bin);
  if (bin >= nbins) return;
  const int4* segs = a.work + bw.z;
  const int tpp = a.bs >> 4;
  const int c = lane & 15, g = lane >> 4;
  const bool qvalid = c < NH * a.G;
  const int myhead = qvalid ? c / a.G : 0;
  const int kvh = has_heads ? kvh0 : 0;
  const auto at = P::lane(a, c, g);

  u32x4 qv[4];  // the first slice's waves fetch a segment's q and put it into LDS
  auto fetch_q = [&](int qrow) {
    if (slice) return;
    const char* qp = reinterpret_cast<const char*>(a.q + (int64_t)qrow * a.q_st + (int64_t)(kvh * a.G + (qvalid ? c : 0)) * a.q_sh);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qv[kk] = ld16(qp + 2 * P::q_dim(kk, g));
  };
  auto put_q = [&](int b) {
    if (slice) return;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qs[b][grp][kk][lane] = qvalid ? qv[kk] : u32x4{0, 0, 0, 0};
  };
  // tiles of a segment: pages past the row's last token (a block table may hold pages ahead) have none
  auto tiles_of = [&](const int4& r0) { return max(min(r0.w, (r0.z + r0.y) * a.bs) - r0.z * a.bs + 15, 0) >> 4; };

  // This slice's tiles in the order they are consumed, one ahead: the segment, the tile and the block it lies in.
  typedef const __attribute__((address_space(4))) int ConstI32;
  ConstI32* indices = (ConstI32*)a.kv_indices;
  const int glast = bw.y - 1;
  int cg = bw.x, ct = slice, cblk, csub;
  bool more;  // the cursor is on a tile; behind the last one it stays there, without
  int4 cr = plan_rec(segs, 2 * cg);
  int cn = tiles_of(cr);
  auto settle = [&]() {  // to the slice's next tile at or behind (cg, ct), and its block
    while (ct >= cn && cg < glast) {
      ++cg;
      cr = plan_rec(segs, 2 * cg);
      cn = tiles_of(cr);
      ct = slice;
    }
    more = ct < cn;
    const int t = min(ct, max(cn - 1, 0));
    const int page = tpp == 1 ? t : t / tpp;
    csub = t - page * tpp;
    cblk = indices[cr.x + page];
  };
  auto load = [&](typename P::Tile& into) {
    const int blk = (unsigned)cblk < (unsigned)a.num_blocks ? cblk : 0;  // else-branch never taken with valid metadata
    P::load(a, kvh, at, blk, csub, into);
  };
  auto advance = [&]() {
    ct += SL;
    settle();
  };

  int gi = bw.x, buf = 0;
  SegRec cur = seg_rec(segs, gi), nxt = cur;
  typename P::Tile tile, ahead;
  settle();
  load(tile);
  fetch_q(cur.r1.x);
  if (gi < glast) nxt = seg_rec(segs, gi + 1);
  advance();
  put_q(0);
  __syncthreads();

  while (true) {
    gi = __builtin_amdgcn_readfirstlane(gi);
    const bool has_next = gi < glast;
    const int tok0 = cur.r0.z * a.bs, len = cur.r0.w;
    const int ntiles = tiles_of(cur.r0);
    SegRec after = nxt;
    if (gi + 2 <= glast) after = seg_rec(segs, gi + 2);
    if (has_next) fetch_q(nxt.r1.x);
    float m_run = -INFINITY, l_run = 0.f;
    f32x4 o[D];
#pragma unroll
    for (int m = 0; m < D; ++m) o[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    const bool runs = has_heads && slice < ntiles;
    if (has_heads) {
      auto consume = [&](int t) {
        P::template consume<T>(tile, &qs[buf][grp][0][lane], myhead, a.scale_log2, tok0 + t * 16, len, c, g, m_run, l_run, o);
      };
      int t = slice;
      for (; t < ntiles && more; t += SL) {
        load(ahead);
        advance();
        consume(t);
        tile = ahead;
      }
      if (t < ntiles) consume(t);  // the bin's last: a load behind it would only be waited for (0.4 us of a small step's 11)
    }

    if (has_next) put_q(buf ^ 1);

    // lane (c, g): o[m][i] is dim D (4 g + i) + m of the joint row; kept where that is the column's own head
    if (qvalid && has_heads && g * NH / 4 == myhead) {
      float* p = part[slice][16 * grp + c];
      const int d0 = (4 * D * g) % kHeadDim;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < D; m += 4)
          *reinterpret_cast<f32x4*>(p + d0 + D * i + m) = f32x4{o[m][i], o[m + 1][i], o[m + 2][i], o[m + 3][i]};
      if (d0 == 0) p[kHeadDim] = m_run, p[kHeadDim + 1] = runs ? l_run : -1.f;
    }
    __syncthreads();
    for (int r = threadIdx.x >> 4; r < kRows; r += 4 * kWavesSlices) {  // 16 threads per query head
      const int head0 = NH * (hg * HGW + r / 16), cc = r % 16, d = 8 * (threadIdx.x & 15);
      if (head0 >= a.Hkv || cc >= NH * a.G) continue;
      float m = -INFINITY, l = 0.f, acc[8] = {};
#pragma unroll
      for (int x = 0; x < SL; ++x) m = fmaxf(m, part[x][r][kHeadDim]);
#pragma unroll
      for (int x = 0; x < SL; ++x) {
        const float lx = part[x][r][kHeadDim + 1];
        const float w = lx == -1.f ? 0.f : fast_exp2(part[x][r][kHeadDim] - m);  // -1: a slice without tiles
        l += w * lx;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += w * part[x][r][d + e];
      }
      const int head = head0 * a.G + cc, slot = cur.r1.y;
      if (slot < 0) {
        const float inv = 1.f / l;
        st16(a.out + (int64_t)cur.r1.x * a.o_st + (int64_t)head * a.o_sh + d,
             u32x4{pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv),
                   pack2<T>(acc[4] * inv, acc[5] * inv), pack2<T>(acc[6] * inv, acc[7] * inv)});
      } else {
        const int64_t row = (int64_t)slot * a.H + head;
        float* po = a.part_o + row * kHeadDim + d;
        *reinterpret_cast<f32x4*>(po) = f32x4{acc[0], acc[1], acc[2], acc[3]};
        *reinterpret_cast<f32x4*>(po + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
        if (d == 0) a.part_ml[row] = make_float2(m, l);
      }
    }
    if (!has_next) break;
    __syncthreads();  // the slices' places are free again
    ++gi;
    buf ^= 1;
    cur = nxt;
    nxt = after;
  }
}

// Log-sum-exp merge of a cut row's partials, as decode.hip's merge_kernel.  Eight groups of 32 threads, four dims each: of a
// row with at most eight partials each group takes a head; of a row with more, all groups take one head, partials in
// turn, and meet in LDS (three rows of 85,000 tokens: 91 us with one group a head, 4.6 with eight).  The number of
// partials alone decides, so a row's result does not depend on the launch: WIDE, for steps whose rows have many, has a
// workgroup per head, of which every eighth serves the short rows; without it a workgroup serves eight heads of either.
constexpr int kFewPartials = 8;
// Up to this many workgroups a step is WIDE whatever its rows have: 40 rows of 256-8,192 tokens beside 8 prompt chunks 114 us
// against 120; for 256 rows of 128-4,096 tokens, where most have few partials, 8192 workgroups take 1 us more than 1024.
constexpr int kWideGroups = 2048;
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void merge_slices_kernel(const int4* __restrict__ merge, const float* __restrict__ part_o,
                                                       const float2* __restrict__ part_ml, int H,
                                                       const int32_t* __restrict__ qo_indptr, uint16_t* __restrict__ out,
                                                       int64_t o_st, int64_t o_sh) {
  __shared__ float red[8][kHeadDim + 4];
  const int4 mw = merge[blockIdx.x];
  const int first = mw.y, n = mw.z;
  if (mw.x < 0) return;  // the whole workgroup
  const int grp = threadIdx.x >> 5, d0 = 4 * (threadIdx.x & 31);
  uint16_t* row_out = out + (int64_t)qo_indptr[mw.x] * o_st + d0;
  auto store = [&](int head, f32x4 acc, float l) {
    const float inv = 1.f / l;
    st8(row_out + (int64_t)head * o_sh, u32x2{pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv)});
  };
  // partials j0, j0 + step, .. below n of a head, added to (m, l, acc); four in flight
  auto add = [&](int head, int j0, int step, float& m, float& l, f32x4& acc) {
    for (; j0 < n; j0 += 4 * step) {
      float2 ml[4];
      f32x4 o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // places past n read the first again and weigh it 0
        const int64_t row = (int64_t)(first + (j0 + u * step < n ? j0 + u * step : j0)) * H + head;
        ml[u] = part_ml[row];
        o[u] = *reinterpret_cast<const f32x4*>(part_o + row * kHeadDim + d0);
      }
      float mc = m;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (j0 + u * step >= n) ml[u].x = -INFINITY;
        mc = fmaxf(mc, ml[u].x);
      }
      // Maxima of -inf: segments without tiles, of l and O zero, or with a NaN among each tile's keys, whose l and O are NaN
      // and stay so under the weight 0 that either gets.
      const float ref = mc == -INFINITY ? 0.f : mc;
      const float sc = fast_exp2(m - ref);
      l *= sc;
      acc *= sc;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = fast_exp2(ml[u].x - ref);
        l += w * ml[u].y;
        acc += w * o[u];
      }
      m = mc;
    }
  };
  const int head0 = WIDE ? blockIdx.y & ~7 : 8 * blockIdx.y;
  if (n <= kFewPartials) {
    const int head = head0 + grp;
    if ((WIDE && (blockIdx.y & 7)) || head >= H) return;
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    add(head, 0, 1, m, l, acc);
    store(head, acc, l);
    return;
  }
  const int from = WIDE ? (int)blockIdx.y : head0, to = WIDE ? from + 1 : min(head0 + 8, H);
  for (int head = from; head < to; ++head) {
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    add(head, grp, 8, m, l, acc);
    float* r = red[grp];
    *reinterpret_cast<f32x4*>(r + d0) = acc;
    if (d0 == 0) r[kHeadDim] = m, r[kHeadDim + 1] = l;
    __syncthreads();
    if (grp == 0) {
      float mc = m;
#pragma unroll
      for (int s = 1; s < 8; ++s) mc = fmaxf(mc, red[s][kHeadDim]);
      float w = fast_exp2(m - mc);
      l *= w;
      acc *= w;
#pragma unroll
      for (int s = 1; s < 8; ++s) {
        w = fast_exp2(red[s][kHeadDim] - mc);
        l += w * red[s][kHeadDim + 1];
        acc += w * *reinterpret_cast<const f32x4*>(red[s] + d0);
      }
      store(head, acc, l);
    }
    __syncthreads();
  }
}

// KV heads per wavefront.
int slice_heads(int num_kv_heads, int group) { return num_kv_heads % 2 == 0 && 2 * group <= 16 ? 2 : 1; }

template <typename T>
int launch_merge_slices(const std::string& fn, const SlicesArgs& a, const int32_t* merge_work, int num_merge, int n_work, const int32_t* qo_indptr,
                     hipStream_t st) {
  const int4* merge = reinterpret_cast<const int4*>(merge_work);
  if (max_bins(n_work) >= kFewPartials * num_merge || (int64_t)num_merge * a.H <= kWideGroups)
    merge_slices_kernel<T, true><<<dim3(num_merge, a.H), 256, 0, st>>>(merge, a.part_o, a.part_ml, a.H, qo_indptr, a.out, a.o_st,
                                                                   a.o_sh);
  else
    merge_slices_kernel<T, false><<<dim3(num_merge, (a.H + 7) / 8), 256, 0, st>>>(merge, a.part_o, a.part_ml, a.H, qo_indptr,
                                                                              a.out, a.o_st, a.o_sh);
  return check_launch(fn.c_str());
}

template <typename T, template <int> class POOL>
int launch_slices(const std::string& fn, SlicesArgs a, int n_work, hipStream_t st) {
  const unsigned bins = (unsigned)max_bins(n_work);
  if (bins == 0) return MLLM_OK;
  const int nh = slice_heads(a.Hkv, a.G), groups = a.Hkv / nh, hgw = groups > 2 ? 4 : groups;
  a.HG = (groups + hgw - 1) / hgw;
  const unsigned grid = bins * (unsigned)a.HG;
  auto launch = [&](auto heads, auto side) {
    decode_slices_kernel<T, POOL, decltype(heads)::value, decltype(side)::value><<<grid, 64 * kWavesSlices, 0, st>>>(a);
  };
  auto of_heads = [&](auto heads) {
    if (hgw == 4)
      launch(heads, std::integral_constant<int, 4>{});
    else if (hgw == 2)
      launch(heads, std::integral_constant<int, 2>{});
    else
      launch(heads, std::integral_constant<int, 1>{});
  };
  if (nh == 2)
    of_heads(std::integral_constant<int, 2>{});
  else
    of_heads(std::integral_constant<int, 1>{});
  return check_launch(fn.c_str());
}


// What the pools' entry points do: their checks, the decode launch and, behind it, the merge of the cut rows.  row_bytes: of
// a token and head in the pool.
template <template <int> class POOL, int kScaleAlign>
int paged_decode_slices(const std::string& fn, int row_bytes, const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                        const void* k_cache, const void* v_cache, const void* k_scales, const void* v_scales,
                        int64_t num_blocks, int32_t block_size, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                        const int32_t* qo_indptr, const int32_t* kv_indices, const int32_t* decode_work,
                        int32_t num_decode_work, const int32_t* merge_work, int32_t num_merge_work, int32_t pages_per_split,
                        float softmax_scale, int32_t dtype, void* out, int64_t out_stride_tok, int64_t out_stride_head,
                        void* workspace, int64_t workspace_bytes, void* stream) {
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
  MLLM_REQUIRE((int64_t)block_size * num_kv_heads * row_bytes < (1ll << 31), MLLM_ERR_UNSUPPORTED,
               fn + ": KV block too large");
  MLLM_REQUIRE(num_decode_work >= 0 && num_merge_work >= 0, MLLM_ERR_INVALID, fn + ": negative count");
  if (num_decode_work == 0) return MLLM_OK;
  MLLM_REQUIRE(q && k_cache && v_cache && k_scales && v_scales && out && qo_indptr && kv_indices && decode_work &&
                   (num_merge_work == 0 || merge_work),
               MLLM_ERR_INVALID, fn + ": null pointer");
  MLLM_REQUIRE(num_heads <= 65535, MLLM_ERR_UNSUPPORTED, fn + ": too many heads");
  const int64_t need = num_merge_work ? mllm_decode_workspace_bytes(num_decode_work, num_heads, head_dim) : 0;
  MLLM_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), MLLM_ERR_INVALID, fn + ": workspace too small");
  MLLM_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 &&
                   ((uintptr_t)k_scales | (uintptr_t)v_scales) % kScaleAlign == 0 &&
                   (q_stride_tok | q_stride_head | out_stride_tok | out_stride_head) % 8 == 0,
               MLLM_ERR_UNSUPPORTED, fn + ": q, out and pools need 16-byte aligned rows");
  SlicesArgs a;
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
  const bool bf16 = dtype == MLLM_DTYPE_BF16;
  const int rc = bf16 ? launch_slices<BF16, POOL>(fn, a, num_decode_work, st) : launch_slices<F16, POOL>(fn, a, num_decode_work, st);
  if (rc != MLLM_OK || num_merge_work == 0) return rc;
  return bf16 ? launch_merge_slices<BF16>(fn, a, merge_work, num_merge_work, num_decode_work, qo_indptr, st)
              : launch_merge_slices<F16>(fn, a, merge_work, num_merge_work, num_decode_work, qo_indptr, st);
}

}  // namespace
}  // namespace mllm
