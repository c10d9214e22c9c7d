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
#include <math.h>

#include <type_traits>

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
  if constexpr (N == 2) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.w[0] = v[0], r.w[1] = v[1];
  } else {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
  return r;
}

constexpr int kRowBytes4 = kHeadDim / 2, kBlocks4 = kHeadDim / kFp4Block;

// A tile of 16 tokens, as the pool stores it.
template <int NH>
struct Fp4Tile {
  u32x4 k[NH];     // token c, head h, dims 32 g .. + 31
  Words<NH> v[4];  // token 4 g + i, D dims of the joint row
  uint32_t ks;     // token c, dim block g: the scales of the NH heads
  uint32_t vs;     // tokens 4 g .. + 3: their scales, a byte each
};
// Byte h of a scale word where the conversions read it (bits 30:23 of their operand; they ignore the others).
__device__ __forceinline__ float scale_of(uint32_t w, int h) {
  return __uint_as_float(h < 3 ? w << (23 - 8 * h) : w >> 1);
}

// What a lane adds to a sub-tile's uniform addresses, in bytes.
struct Fp4Lane {
  unsigned k, ks, v, vs;
};

template <int NH>
__device__ __forceinline__ void load_tile4(const DecodeFp4Args& a, int kvh0, const Fp4Lane& at, int blk, int sub, Fp4Tile<NH>& r) {
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

// What two fp16 values (`hi`) leave of the floats they were rounded from, as fp16.
__device__ __forceinline__ uint32_t f16_rest(float a, float b, uint32_t hi) {
  return pack2<F16>(a - f16_bits_to_f32((uint16_t)hi), b - f16_bits_to_f32((uint16_t)(hi >> 16)));
}

// One 16-token tile: scores, online-softmax update, PV.  `q`: this lane's Q^T operands in LDS.
template <typename T, int NH>
__device__ __forceinline__ void consume_tile4(Fp4Tile<NH>& r, const u32x4* q, int myhead, float scale_log2, int tpos0, int len,
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
  const float mx = maximum_xor32(maximum_xor16(maximum(maximum(s[0], s[1]), maximum(s[2], s[3]))));
  if (__any(mx > m_run + 8.f)) {  // lazy rescale, as in decode.hip
    const float m_new = fmaxf(m_run, mx);
    const float alpha = fast_exp2(m_run - m_new);
    l_run *= alpha;
#pragma unroll
    for (int m = 0; m < 8 * NH; ++m) o[m] *= alpha;
    m_run = m_new;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = fast_exp2(s[i] - m_run);
  l_run += sum_xor32(sum_xor16((s[0] + s[1]) + (s[2] + s[3])));
  constexpr bool kSplit = std::is_same<T, F16>::value;
  const u32x2 phi = u32x2{pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3])};
  u32x2 plo = {0, 0};
  if constexpr (kSplit) plo = u32x2{f16_rest(s[0], s[1], phi[0]), f16_rest(s[2], s[3], phi[1])};
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
        o[m] = Mfma<T>::m16x16x16(vf, phi, o[m]);
        if constexpr (kSplit) o[m] = Mfma<T>::m16x16x16(vf, plo, o[m]);
      }
    }
}

// A workgroup of eight wavefronts takes one bin and HGW groups of NH heads: wavefront w group w % HGW and the tiles w / HGW,
// + SL, .. of each segment, SL = 8 / HGW (bins then need be no shorter than one per CU, which keeps the partials few, and
// with four groups of two heads whole pages are read together).  Each wavefront has the next tile on its way while it works
// on one, across segment boundaries.  The slices' (m, l, O) of a segment meet in LDS, where each thread combines eight
// dims of one query head and writes the output, or the segment's partial when the row is cut.
constexpr int kWavesFp4 = 8;
constexpr int kPartRow = kHeadDim + 4;  // floats of a slice's query head in LDS: O, then m and l

template <typename T, int NH, int HGW>
__global__ __launch_bounds__(64 * kWavesFp4) __attribute__((amdgpu_waves_per_eu(kWavesFp4 / 4, kWavesFp4 / 4))) void decode_fp4_kernel(
    const DecodeFp4Args a) {
  constexpr int D = 8 * NH, SL = kWavesFp4 / HGW, kRows = 16 * HGW;  // query heads' places in LDS
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
  const unsigned st = (unsigned)(a.Hkv * kRowBytes4);
  const Fp4Lane at{(unsigned)c * st + 16u * g, (unsigned)((c * kBlocks4 + g) * a.Hkv), (unsigned)(4 * g) * st + 4u * NH * c,
                   (unsigned)((D * c / kFp4Block) * a.bs + 4 * g)};

  u32x4 qv[4];  // the first slice's waves fetch a segment's q and put it into LDS
  auto fetch_q = [&](int qrow) {
    if (slice) return;
    const char* qp = reinterpret_cast<const char*>(a.q + (int64_t)qrow * a.q_st + (int64_t)(kvh * a.G + (qvalid ? c : 0)) * a.q_sh);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qv[kk] = ld16(qp + 2 * (32 * g + 8 * kk));
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
  auto load = [&](Fp4Tile<NH>& into) {
    const int blk = (unsigned)cblk < (unsigned)a.num_blocks ? cblk : 0;  // else-branch never taken with valid metadata
    load_tile4<NH>(a, kvh, at, blk, csub, into);
  };
  auto advance = [&]() {
    ct += SL;
    settle();
  };

  int gi = bw.x, buf = 0;
  SegRec cur = seg_rec(segs, gi), nxt = cur;
  Fp4Tile<NH> tile, ahead;
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
        consume_tile4<T, NH>(tile, &qs[buf][grp][0][lane], myhead, a.scale_log2, tok0 + t * 16, len, g, m_run, l_run, o);
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
    for (int r = threadIdx.x >> 4; r < kRows; r += 4 * kWavesFp4) {  // 16 threads per query head
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
__global__ __launch_bounds__(256) void merge_fp4_kernel(const int4* __restrict__ merge, const float* __restrict__ part_o,
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
int fp4_heads(int num_kv_heads, int group) { return num_kv_heads % 2 == 0 && 2 * group <= 16 ? 2 : 1; }

template <typename T>
int launch_merge_fp4(const DecodeFp4Args& a, const int32_t* merge_work, int num_merge, int n_work, const int32_t* qo_indptr,
                     hipStream_t st) {
  const int4* merge = reinterpret_cast<const int4*>(merge_work);
  if (max_bins(n_work) >= kFewPartials * num_merge || (int64_t)num_merge * a.H <= kWideGroups)
    merge_fp4_kernel<T, true><<<dim3(num_merge, a.H), 256, 0, st>>>(merge, a.part_o, a.part_ml, a.H, qo_indptr, a.out, a.o_st,
                                                                   a.o_sh);
  else
    merge_fp4_kernel<T, false><<<dim3(num_merge, (a.H + 7) / 8), 256, 0, st>>>(merge, a.part_o, a.part_ml, a.H, qo_indptr,
                                                                              a.out, a.o_st, a.o_sh);
  return check_launch("mllm_paged_decode_fp4");
}

template <typename T>
int launch_fp4(DecodeFp4Args a, int n_work, hipStream_t st) {
  const unsigned bins = (unsigned)max_bins(n_work);
  if (bins == 0) return MLLM_OK;
  const int nh = fp4_heads(a.Hkv, a.G), groups = a.Hkv / nh, hgw = groups > 2 ? 4 : groups;
  a.HG = (groups + hgw - 1) / hgw;
  const unsigned grid = bins * (unsigned)a.HG;
  auto launch = [&](auto heads, auto side) {
    decode_fp4_kernel<T, decltype(heads)::value, decltype(side)::value><<<grid, 64 * kWavesFp4, 0, st>>>(a);
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
  return check_launch("mllm_paged_decode_fp4");
}

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
  MLLM_REQUIRE(q && k_cache && v_cache && k_scales && v_scales && out && qo_indptr && kv_indices && decode_work &&
                   (num_merge_work == 0 || merge_work),
               MLLM_ERR_INVALID, fn + ": null pointer");
  MLLM_REQUIRE(num_heads <= 65535, MLLM_ERR_UNSUPPORTED, fn + ": too many heads");
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
  const bool bf16 = dtype == MLLM_DTYPE_BF16;
  const int rc = bf16 ? launch_fp4<BF16>(a, num_decode_work, st) : launch_fp4<F16>(a, num_decode_work, st);
  if (rc != MLLM_OK || num_merge_work == 0) return rc;
  return bf16 ? launch_merge_fp4<BF16>(a, merge_work, num_merge_work, num_decode_work, qo_indptr, st)
              : launch_merge_fp4<F16>(a, merge_work, num_merge_work, num_decode_work, qo_indptr, st);
}
