// Linear layers of 8-bit blocks: y[M, N] = x[M, K] . w[N, K]^T with e4m3 codes and one power-of-two scale (e8m0) for
// 128 x 128 weights and for 128 columns of a row of x, which is quantised here (no counterpart in the reference).
//   sx = the least power of two with max|x_block| / sx <= 448, xq = e4m3(x / sx), to nearest with ties to even
//   y[m][n] = T( sum_b sx[m][b] sw[n / 128][b] sum_{k in block b} xq[m][k] wq[n][k] )
// Every step but the rounding to e4m3 and the sums is exact.  v_mfma_scale_f32_16x16x128_f8f6f4 takes a block per
// instruction and applies both scales, so the accumulators run through K without a vector instruction.  It adds the products
// of eight neighbouring k aligned to the largest of them and drops what lies below 2^-13 of that one's power of two, as
// measured on the card with products of chosen sizes (the eights and the accumulator add with 24 bits): at most 7 2^-13 of an
// eight's largest product, under the 2^-4 of its x's own rounding.  An infinity or a NaN in a block of x makes its scale,
// and the row's outputs, NaN.
//
// MFMA operands: lane (n, g) = (l % 16, l / 16) holds row n's bytes 16 g .. + 15 and 64 + 16 g .. + 15 of the block, of the
// weights and of x alike (any order of k within a block is a valid sum: one scale covers it).  Weights are the A operand, so
// a lane ends with four consecutive outputs of one row of y.
#include <math.h>

#include <type_traits>

#include "common.h"

namespace mllm {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 128;    // K per scale, and rows of weights
constexpr int kFewRows = 64;                    // rows of x up to which the weights are streamed,
constexpr int kInPlaceRows = 16;                // .. and of them those fp8_rows_kernel takes,
// with weights of up to this many bytes.  Measured with either kernel for every size (us from a graph at 1 / 8 / 16 rows,
// fp8_rows_kernel against fp8_chunk_kernel): 4096 x 4096, 16 MiB, 6.9 / 7.5 / 8.8 against 8.1 / 9.1 / 9.6; 4096 x 6144 8.9 / 9.7 /
// 11.6 against 10.0 / 10.9 / 11.5; 6144 x 4096 8.6 / 11.0 / 14.0 against 11.5 / 12.3 / 13.0; 5120 x 5120 9.9 / 13.1 / 16.8 against
// 11.5 / 12.4 / 13.0; 14336 x 4096 15.3 / 20.0 / 25.0 against 17.2 / 17.7 / 18.6.  From 24 MiB up the
// first falls behind at 8 or 16 rows; up to 16 MiB it is ahead at all of them.
constexpr int64_t kSmallWeights = 1 << 24;

__device__ __forceinline__ i32x8 join(u32x4 lo, u32x4 hi) {
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
template <int OPSEL_X>
__device__ __forceinline__ f32x4 mfma_fp8(i32x8 w, i32x8 x, f32x4 c, int sw, int sx) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 0, 0, 0, sw, OPSEL_X, sx);
}

// A byte at a uniform address, as a scalar load of the dword that holds it.
__device__ __forceinline__ int scalar_byte(const uint8_t* at) {
  typedef const __attribute__((address_space(4))) uint32_t ConstU32;
  const uintptr_t p = (uintptr_t)at;
  return (int)((*(ConstU32*)(p & ~(uintptr_t)3) >> (8 * (p & 3))) & 0xffu);
}

// ---------------------------------------------------------------- quantisation of x

// Largest of the 16-bit patterns without their sign (they order as the magnitudes do; infinities and NaN are on top).
__device__ __forceinline__ uint32_t max_abs16(u32x4 x, uint32_t m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
  return m;
}
// Scale exponent of a block whose largest 16-bit pattern is m: 448 = 1.75 2^8, so floor(log2) - 8, one more where the
// mantissa is above 1.75.
template <typename T>
__device__ __forceinline__ uint32_t x_scale_exp(uint32_t m);
template <>
__device__ __forceinline__ uint32_t x_scale_exp<BF16>(uint32_t m) {
  const uint32_t u = m << 16;
  if (u >= 0x7f800000u) return 255u;
  return (uint32_t)max((int)((u + 0x1fffffu) >> 23) - 8, 1);
}
template <>
__device__ __forceinline__ uint32_t x_scale_exp<F16>(uint32_t m) {
  const uint32_t u = __float_as_uint(f16_bits_to_f32((uint16_t)m));
  if (u >= 0x7f800000u) return 255u;
  return (uint32_t)max((int)((u + 0x1fffffu) >> 23) - 8, 1);
}
// Four 16-bit values (two dwords) -> four e4m3 codes of x / scale.
template <typename T>
__device__ __forceinline__ uint32_t quant4_e4m3(uint32_t a, uint32_t b, float scale);
template <>
__device__ __forceinline__ uint32_t quant4_e4m3<BF16>(uint32_t a, uint32_t b, float scale) {
  i16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(i16x2{0, 0}, __builtin_bit_cast(bf16x2, a), scale, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, b), scale, true));
}
template <>
__device__ __forceinline__ uint32_t quant4_e4m3<F16>(uint32_t a, uint32_t b, float scale) {
  i16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(i16x2{0, 0}, __builtin_bit_cast(f16x2, a), scale, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, b), scale, true));
}
template <typename T>
__device__ __forceinline__ u32x4 quant16_e4m3(u32x4 lo, u32x4 hi, uint32_t e) {
  const float s = __uint_as_float(e << 23);
  return u32x4{quant4_e4m3<T>(lo[0], lo[1], s), quant4_e4m3<T>(lo[2], lo[3], s), quant4_e4m3<T>(hi[0], hi[1], s),
               quant4_e4m3<T>(hi[2], hi[3], s)};
}

// ---------------------------------------------------------------- few rows: the weights streamed once

struct RowsArgs {
  const char* x;  // 16-bit rows
  int64_t x_st;   // row stride, bytes
  int M, K, N, blocks;
  const char* w;  // [N][128 blocks]
  const uint8_t* ws;
  uint16_t* y;
  int tiles, ksplit;
  float* part;  // ksplit > 1: [ksplit][M][N]
};

constexpr int kRowsWaves = 8;

// Largest over the lanes that hold one row's block: l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ uint32_t max_over_g(uint32_t v) {
  auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((uint32_t)a[0], (uint32_t)a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)b[0], (uint32_t)b[1]);
}
// The value of lane l ^ 8.
__device__ __forceinline__ uint32_t lane_xor8(uint32_t v) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true); }

// A wavefront's operand of x for one block: rows of up to 16 quantised in place.  With at most 8 rows, lanes n and n + 8 share
// row n: each loads and quantises half of the lane's columns and they swap codes (columns 8 .. 15 of the product are unused).
template <typename T, bool HALF>
struct RowsX {
  static constexpr int kLoads = HALF ? 2 : 4;
  u32x4 v[kLoads];
  static __device__ __forceinline__ int column(int k0, int j, bool second) { return k0 + (HALF ? (second ? 64 : 0) : 32 * j); }
  // columns past K (a multiple of 16: a lane's 16 are all there or none) read the last ones and are cleared before their use
  __device__ __forceinline__ void load(const char* row, int k0, int K, bool second) {
#pragma unroll
    for (int j = 0; j < kLoads; j += 2) {
      const char* at = row + 2 * min(column(k0, j, second), K - 16);
      v[j] = ld16(at);
      v[j + 1] = ld16(at + 16);
    }
  }
  __device__ __forceinline__ void clear_past(int k0, int K, bool second) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      if (column(k0, j & ~1, second) >= K) v[j] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ i32x8 operand(uint32_t& e) const {
    u16x2 m = {0, 0};
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[j][i] & 0x7fff7fffu));
    uint32_t top = max((uint32_t)m[0], (uint32_t)m[1]);
    if (HALF) top = max(top, lane_xor8(top));
    e = x_scale_exp<T>(max_over_g(top));
    const u32x4 lo = quant16_e4m3<T>(v[0], v[1], e);
    if constexpr (HALF) return join(lo, u32x4{lane_xor8(lo[0]), lane_xor8(lo[1]), lane_xor8(lo[2]), lane_xor8(lo[3])});
    else return join(lo, quant16_e4m3<T>(v[2], v[3], e));
  }
};

// Both kernels are bound by the weights, N K bytes read once, and at these sizes by what surrounds the reading.
// Up to 16 rows, small weights: one workgroup per 16 weight rows, eight wavefronts along K, x quantised by the wavefronts that
// use it.  One launch, no exchange but the eight partial sums in LDS.  4096 x 4096 (us, from a graph, weights from memory): 6.9
// at 1 row, 7.2 at 8, 8.3 at 16; the chunk kernel below with the launch that adds its parts 8.0, 8.7, 8.9.  What it cost to
// quantise x in every workgroup: 8.9 at 8 rows when each of the 16 operand columns loaded a row, with maxima by dword and
// through LDS.  Loads that bypass the cache (nt) are 5 - 10% slower in both kernels.
template <typename T, bool HALF>
__global__ __launch_bounds__(64 * kRowsWaves) void fp8_rows_kernel(const RowsArgs a) {
  __shared__ f32x4 red[kRowsWaves][64];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = 16 * blockIdx.x;
  const int first = a.blocks * wave / kRowsWaves, end = a.blocks * (wave + 1) / kRowsWaves;
  const char* wp = a.w + (int64_t)(n0 + n) * a.blocks * kBlock + 16 * g;
  const uint8_t* ws = a.ws + (int64_t)(n0 / kBlock) * a.blocks;
  const char* xp = a.x + min(HALF ? n & 7 : n, a.M - 1) * a.x_st;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int kAhead = 2;  // blocks in flight
  struct Stage {
    u32x4 w[2];
    RowsX<T, HALF> x;
    int sw;
  } ring[kAhead];
  auto load = [&](Stage& s, int b) {
    s.x.load(xp, b * kBlock + 16 * g, a.K, n >= 8);
    s.sw = ws[b];
    s.w[0] = ld16(wp + (int64_t)b * kBlock);
    s.w[1] = ld16(wp + (int64_t)b * kBlock + 64);
  };
  auto use = [&](Stage& s, int b) {
    if ((b + 1) * kBlock > a.K) s.x.clear_past(b * kBlock + 16 * g, a.K, n >= 8);
    uint32_t e;
    const i32x8 xv = s.x.operand(e);
    acc = mfma_fp8<0>(join(s.w[0], s.w[1]), xv, acc, s.sw, (int)e);
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (first + u < end) load(ring[u], first + u);
  int b = first;
  for (; b + 2 * kAhead <= end; b += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      use(ring[u], b + u);
      load(ring[u], b + u + kAhead);
    }
  }
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    if (b + u < end) use(ring[u], b + u);
    if (b + u + kAhead < end) load(ring[u], b + u + kAhead);
  }
#pragma unroll
  for (int u = 0; u < kAhead - 1; ++u)
    if (b + u + kAhead < end) use(ring[u], b + u + kAhead);
  red[wave][lane] = acc;
  __syncthreads();
  if (wave > 0) return;
  f32x4 s = red[0][lane];  // lane (n, g): row n of y, outputs 4 g .. + 3 of the tile
#pragma unroll
  for (int k = 1; k < kRowsWaves; ++k) s += red[k][lane];
  if (n < a.M && !(HALF && n >= 8)) st8(a.y + (int64_t)n * a.N + n0 + 4 * g, u32x2{pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3])});
}

// Up to 64 rows: a workgroup takes 128 weight rows, 16 a wavefront, and a part of K in chunks of kChunk blocks.  Its wavefronts
// quantise the chunk of x together, a block of 16 rows each, into LDS in operand order while weights load: x is read and
// quantised once per 128 weight rows.  Parts meet in fp32 (mllm_sum_partials): as many as leave no CU two workgroups, but
// of small weights always eight, the wavefronts' parts of fp8_rows_kernel, whose bits a row then keeps at any number of
// rows (a K of fewer than eight blocks leaves some of them empty: sums of zero that are written and added all the same).  Measured as above, 14336 x 4096 / 4096 x 14336, 8 rows 17.6 / 17.7 us (3.3 TB/s with both launches), 32
// rows 20.6, 64 rows 25.3 / 24.6.  Workgroups of 16 weight rows (fp8_rows_kernel's way) took 20.2 / 20.9 at 8 rows, 73 / 60 at 64; with x quantised
// once by another launch 26.9 / 30.6 at 64.  Two workgroups per CU: 22.1 / 18.4 at 8
// rows, but 29.8 against 32.8 for 13312 x 8192; with some CUs taking two (20480 x 4096 in two parts) 27.4 against 24.7.  Halves
// of K within a workgroup of 64 weight rows, which need no adding launch: no faster.
template <typename T, int MT, bool HALF>
__global__ __launch_bounds__(64 * kRowsWaves) void fp8_chunk_kernel(const RowsArgs a) {
  constexpr int kChunk = MT == 1 ? 8 : 4;
  constexpr int kTasks = MT * kChunk / kRowsWaves;  // blocks of 16 rows per wavefront
  __shared__ u32x4 codes[2][kChunk][MT][2][64];     // lane's 16-byte halves
  __shared__ uint8_t scales[2][kChunk][16][4];      // [row % 16][row / 16]
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % a.tiles, ks = blockIdx.x / a.tiles;
  const int n0 = kBlock * tile + 16 * wave;
  const int first = (int)((int64_t)a.blocks * ks / a.ksplit), end = (int)((int64_t)a.blocks * (ks + 1) / a.ksplit);
  const char* wp = a.w + (int64_t)min(n0 + n, a.N - 1) * a.blocks * kBlock + 16 * g;
  const uint8_t* ws = a.ws + (int64_t)tile * a.blocks;
  const char* xp[kTasks];
#pragma unroll
  for (int i = 0; i < kTasks; ++i) {
    const int m = 16 * ((wave + kRowsWaves * i) % MT) + (HALF ? n & 7 : n);
    xp[i] = a.x + min(m, a.M - 1) * a.x_st;
  }
  u32x4 w[kChunk][2];
  int sw[kChunk];
  RowsX<T, HALF> x[kTasks];
  auto task_block = [&](int i) { return (wave + kRowsWaves * i) / MT; };
  auto load_x = [&](int b0) {
#pragma unroll
    for (int i = 0; i < kTasks; ++i)
      if (b0 + task_block(i) < end) x[i].load(xp[i], (b0 + task_block(i)) * kBlock + 16 * g, a.K, n >= 8);
  };
  auto load_w = [&](int u, int b) {
    sw[u] = ws[b];
    w[u][0] = ld16(wp + (int64_t)b * kBlock);
    w[u][1] = ld16(wp + (int64_t)b * kBlock + 64);
  };
  auto quantise = [&](int b0, int buf) {
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      const int u = task_block(i), m = (wave + kRowsWaves * i) % MT;
      if (b0 + u >= end) continue;
      if ((b0 + u + 1) * kBlock > a.K) x[i].clear_past((b0 + u) * kBlock + 16 * g, a.K, n >= 8);
      uint32_t e;
      const i32x8 v = x[i].operand(e);
      codes[buf][u][m][0][lane] = u32x4{(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3]};
      codes[buf][u][m][1][lane] = u32x4{(uint32_t)v[4], (uint32_t)v[5], (uint32_t)v[6], (uint32_t)v[7]};
      if (g == 0) scales[buf][u][n][m] = (uint8_t)e;
    }
  };
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](int u, int buf) {
    const i32x8 wv = join(w[u][0], w[u][1]);
    const int sx = *reinterpret_cast<const int*>(scales[buf][u][n]);
    acc[0] = mfma_fp8<0>(wv, join(codes[buf][u][0][0][lane], codes[buf][u][0][1][lane]), acc[0], sw[u], sx);
    if constexpr (MT > 1) acc[1] = mfma_fp8<1>(wv, join(codes[buf][u][1][0][lane], codes[buf][u][1][1][lane]), acc[1], sw[u], sx);
    if constexpr (MT > 2) {
      acc[2] = mfma_fp8<2>(wv, join(codes[buf][u][2][0][lane], codes[buf][u][2][1][lane]), acc[2], sw[u], sx);
      acc[3] = mfma_fp8<3>(wv, join(codes[buf][u][3][0][lane], codes[buf][u][3][1][lane]), acc[3], sw[u], sx);
    }
  };
  load_x(first);
#pragma unroll
  for (int u = 0; u < kChunk; ++u)
    if (first + u < end) load_w(u, first + u);
  quantise(first, 0);
  barrier_lds();
  // a chunk: the next one's x loads, this one's products, each block's weights replaced by the next chunk's, the next one's codes
  for (int b0 = first, buf = 0; b0 < end; b0 += kChunk, buf ^= 1) {
    load_x(b0 + kChunk);
#pragma unroll
    for (int u = 0; u < kChunk; ++u) {
      if (b0 + u < end) multiply(u, buf);
      if (b0 + kChunk + u < end) load_w(u, b0 + kChunk + u);
    }
    quantise(b0 + kChunk, buf ^ 1);
    barrier_lds();
  }
  const int col = n0 + 4 * g;  // lane (n, g): row 16 m + n of y, outputs 4 g .. + 3 of the wavefront's
  if (col >= a.N) return;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int row = 16 * m + n;
    if (row >= a.M || (HALF && n >= 8)) continue;
    if (a.ksplit > 1)
      *reinterpret_cast<f32x4*>(a.part + ((int64_t)ks * a.M + row) * a.N + col) = acc[m];
    else
      st8(a.y + (int64_t)row * a.N + col, u32x2{pack2<T>(acc[m][0], acc[m][1]), pack2<T>(acc[m][2], acc[m][3])});
  }
}

// ---------------------------------------------------------------- many rows: x quantised once, then tiles

// xq [M][128 blocks] codes; scales as the tile kernel's lanes read them: sx[block][row / 64][row % 16] is a dword, byte
// (row / 16) % 4 of it the row's scale.
template <typename T>
__global__ __launch_bounds__(256) void fp8_quant_kernel(const char* __restrict__ x, int64_t x_st, unsigned M, int K, int blocks,
                                                       char* __restrict__ xq, uint8_t* __restrict__ sx, unsigned groups64) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;  // 16 columns each, eight threads a block
  const unsigned per_row = 8u * (unsigned)blocks;
  const unsigned m = i / per_row, c = i - m * per_row;
  if (m >= M) return;
  const int k0 = 16 * (int)c;
  u32x4 lo = {0, 0, 0, 0}, hi = lo;
  if (k0 < K) {
    lo = ld16(x + m * x_st + 2 * k0);
    hi = ld16(x + m * x_st + 2 * k0 + 16);
  }
  uint32_t top = max_abs16(hi, max_abs16(lo, 0u));
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
  const uint32_t e = x_scale_exp<T>(top);
  st16(xq + 16 * (int64_t)i, quant16_e4m3<T>(lo, hi, e));
  if ((c & 7) == 0) sx[((int64_t)(c >> 3) * groups64 + (m >> 6)) * 64 + 4 * (m & 15) + ((m >> 4) & 3)] = (uint8_t)e;
}

struct TileArgs {
  const char* xq;
  const uint8_t* sx;
  const char* w;
  const uint8_t* ws;
  int M, N, blocks, groups64;
  int tiles_n, tiles_m, ksplit;
  uint16_t* y;
  float* part;  // ksplit > 1: [ksplit][M][N]
};

// y tile of BN weight rows x BM rows of x per workgroup, WN x WM wavefronts of (BN / WN) x (BM / WM) each.  Codes go through
// LDS by DMA, a block of K (128 bytes a row) per step, STAGES - 1 steps ahead; 16-byte piece j of row r lies at j ^ (r % 8),
// so that eight lanes of an operand read hit distinct banks.
// Bound by the matrix instructions (4.4 PFLOP/s of them alone) and the DMA into LDS between them: a step of 256 x 256 takes
// 1.65 us, 1.35 without its DMA, 1.38 without its products; either tile takes 40 - 47 bytes/ns per CU into LDS, also when all
// read the same one.  8192 x 14336 x 4096: 366 us, 2.6 PFLOP/s (the library's product of
// fp8 matrices without blocks 2.7), and 59 us for quantising x, bound by memory (6 TB/s).  Measured slower there: reading a
// step's operands before a barrier, with the DMA two steps ahead, 435 us; the two wavefronts of a SIMD reading and multiplying
// in turn, 445; four wavefronts of 128 x 128.
// Tiles of 128 x 128, for products of fewer, go two workgroups to a CU with two stages each, or, where no CU gets two, with
// four: 256 rows on 14336 x 4096 32.1 us against 40.8 (all launches, from a graph), 777 on 4096 x 4096 29.0 against 39.3,
// 65 on 4096 x 14336 23.6 against 28.3.
template <typename T, int BN, int BM, int WN, int WM, int OCC, int STAGES>
__global__ __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(OCC, OCC))) void fp8_tile_kernel(const TileArgs a) {
  constexpr int kWaves = WN * WM;
  constexpr int kA = BN * kBlock, kB = BM * kBlock, kStage = kA + kB + 4 * 64 * (BM / 256 ? BM / 256 : 1);
  constexpr int FN = BN / WN / 16, FM = BM / WM / 16;  // 16-row operands per wavefront
  constexpr int kRowsX = BM / WM;                      // rows of x per wavefront
  static_assert(kRowsX % 64 == 0, "a dword of scales per lane serves 64 rows of x");
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * kStage];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;

  // workgroups are dealt round-robin to the 8 XCDs: each takes a contiguous run of the tiles, ordered in bands of kBand
  // tiles of weights, so that the workgroups of one L2 share both operands (bands of 4: 2 - 8% slower)
  constexpr int kBand = 8;
  const int tiles = a.tiles_n * a.tiles_m;
  const int ks = blockIdx.x / tiles, id = blockIdx.x % tiles;
  const int per = tiles / 8, rest = tiles % 8, xcd = id % 8;
  const int t = xcd * per + min(xcd, rest) + id / 8;
  const int band = t / (kBand * a.tiles_m), bn = min(kBand, a.tiles_n - kBand * band), in = t - kBand * a.tiles_m * band;
  // (divisions run on the vector unit: tell the compiler that the results are uniform)
  const int n0 = __builtin_amdgcn_readfirstlane(BN * (kBand * band + in % bn)), m0 = __builtin_amdgcn_readfirstlane(BM * (in / bn));
  const int first = __builtin_amdgcn_readfirstlane(a.blocks * ks / a.ksplit);
  const int steps = __builtin_amdgcn_readfirstlane(a.blocks * (ks + 1) / a.ksplit) - first;

  const int64_t row_bytes = (int64_t)a.blocks * kBlock;
  const char* wbase = a.w + n0 * row_bytes + (int64_t)first * kBlock;
  const char* xbase = a.xq + m0 * row_bytes + (int64_t)first * kBlock;
  // one DMA instruction fills 1 KB: 8 rows, lane l row l / 8, place l % 8
  constexpr int kDmaA = BN / 8 / kWaves, kDmaB = BM / 8 / kWaves;
  const int dr = lane >> 3, dc = (lane & 7) ^ dr;
  unsigned offa[kDmaA], offb[kDmaB];
#pragma unroll
  for (int i = 0; i < kDmaA; ++i)
    offa[i] = (unsigned)min(8 * (kDmaA * wave + i) + dr, a.N - 1 - n0) * (unsigned)row_bytes + 16u * dc;
#pragma unroll
  for (int i = 0; i < kDmaB; ++i)
    offb[i] = (unsigned)min(8 * (kDmaB * wave + i) + dr, a.M - 1 - m0) * (unsigned)row_bytes + 16u * dc;
  // scales of the tile's rows of x: BM bytes, 64 to a row group; groups past the last repeat it
  const unsigned offs = 64u * (unsigned)min(m0 / 64 + lane / 16, a.groups64 - 1) + 4u * (lane & 15);
  auto load = [&](int s) {
    char* st = lds + s % STAGES * kStage;
    const char* wb = wbase + (int64_t)s * kBlock;
    const char* xb = xbase + (int64_t)s * kBlock;
#pragma unroll
    for (int i = 0; i < kDmaA; ++i) dma16(wb, offa[i], lds_offset(st) + 1024 * (kDmaA * wave + i));
#pragma unroll
    for (int i = 0; i < kDmaB; ++i) dma16(xb, offb[i], lds_offset(st + kA) + 1024 * (kDmaB * wave + i));
    if (wave == 0) dma4(reinterpret_cast<const char*>(a.sx) + (int64_t)(first + s) * a.groups64 * 64, offs, lds_offset(st + kA + kB));
  };

  f32x4 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int nb0 = (n0 + wn * (BN / WN)) / kBlock;  // the wavefront's weights lie in one row of blocks (past N: repeated)
  const uint8_t* wsrow = a.ws + (int64_t)min(nb0, (a.N - 1) / kBlock) * a.blocks + first;
  const int rl = n & 7, c0 = 16 * (g ^ rl), c1 = 16 * ((4 + g) ^ rl);
  // all loads but those of the last STAGES - 2 steps have landed, in every wavefront
  auto landed = [&](bool more) {
    constexpr int kLoad = kDmaA + kDmaB;
    if (STAGES == 2 || !more)
      barrier_vm<0>();
    else if (wave == 0)
      barrier_vm<(STAGES - 2) * (kLoad + 1)>();
    else
      barrier_vm<(STAGES - 2) * kLoad>();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps) load(s);
  landed(steps >= STAGES - 1);
  for (int s = 0; s < steps; ++s) {
    if (s + STAGES - 1 < steps) load(s + STAGES - 1);
    const char* st = lds + s % STAGES * kStage;
    const char* pa = st + (wn * (BN / WN) + n) * kBlock;
    const char* pb = st + kA + (wm * kRowsX + n) * kBlock;
    int sx[kRowsX / 64];
#pragma unroll
    for (int j = 0; j < kRowsX / 64; ++j) sx[j] = *reinterpret_cast<const int*>(st + kA + kB + kRowsX * wm + 64 * j + 4 * n);
    const int sw = scalar_byte(wsrow + s);
    i32x8 xb[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) xb[j] = join(ld16(pb + 16 * j * kBlock + c0), ld16(pb + 16 * j * kBlock + c1));
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const i32x8 wv = join(ld16(pa + 16 * i * kBlock + c0), ld16(pa + 16 * i * kBlock + c1));
#pragma unroll
      for (int j = 0; j < FM; j += 4) {
        acc[i][j] = mfma_fp8<0>(wv, xb[j], acc[i][j], sw, sx[j / 4]);
        acc[i][j + 1] = mfma_fp8<1>(wv, xb[j + 1], acc[i][j + 1], sw, sx[j / 4]);
        acc[i][j + 2] = mfma_fp8<2>(wv, xb[j + 2], acc[i][j + 2], sw, sx[j / 4]);
        acc[i][j + 3] = mfma_fp8<3>(wv, xb[j + 3], acc[i][j + 3], sw, sx[j / 4]);
      }
    }
    landed(s + STAGES - 1 < steps);
  }
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int col = n0 + wn * (BN / WN) + 16 * i + 4 * g;
    if (col >= a.N) continue;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int m = m0 + wm * kRowsX + 16 * j + n;
      if (m >= a.M) continue;
      const f32x4 v = acc[i][j];
      if (a.ksplit > 1)
        *reinterpret_cast<f32x4*>(a.part + ((int64_t)ks * a.M + m) * a.N + col) = v;
      else
        st8(a.y + (int64_t)m * a.N + col, u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])});
    }
  }
}

// ---------------------------------------------------------------- launch rules

struct Plan {
  bool rows, chunk, large;
  int ksplit;
  int64_t xq_bytes, sx_bytes, part_bytes;
};
constexpr int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

Plan plan_linear(int64_t m, int64_t n, int64_t blocks, int cus) {
  Plan p{};
  p.ksplit = 1;
  p.rows = m <= kInPlaceRows && n * blocks * kBlock <= kSmallWeights;
  p.chunk = !p.rows && m <= kFewRows;
  if (p.rows) return p;
  if (p.chunk) {
    // the parts do not depend on m, and those of small weights are the wavefronts' of fp8_rows_kernel: neither does a row's result
    const int64_t tiles = (n + kBlock - 1) / kBlock, ks = cus / tiles;
    p.ksplit = n * blocks * kBlock <= kSmallWeights ? kRowsWaves : (int)(ks < 1 ? 1 : ks > blocks ? blocks : ks);
  } else {
    const int64_t large = ((n + 255) / 256) * ((m + 255) / 256), small = ((n + 127) / 128) * ((m + 127) / 128);
    p.large = large * 4 >= 3 * (int64_t)cus;
    if (!p.large && small < cus) {
      int64_t ks = cus / small;
      if (ks > 8) ks = 8;
      if (ks > blocks / 4) ks = blocks / 4;
      p.ksplit = ks < 1 ? 1 : (int)ks;
    }
    p.xq_bytes = align256(m * blocks * kBlock);
    p.sx_bytes = align256(blocks * ((m + 63) / 64) * 64);
  }
  p.part_bytes = p.ksplit > 1 ? align256(4 * p.ksplit * m * n) : 0;
  return p;
}

}  // namespace
}  // namespace mllm

extern "C" int64_t mllm_fp8_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, int32_t num_cus) {
  using namespace mllm;
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Plan p = plan_linear(m, n, (k + kBlock - 1) / kBlock, num_cus > 0 ? num_cus : device_cus());
  return p.xq_bytes + p.sx_bytes + p.part_bytes;
}

extern "C" int mllm_fp8_linear(const void* x, int64_t x_stride, int64_t m, int64_t k, const void* weight,
                               const void* weight_scales, int64_t n, int32_t dtype, void* workspace,
                               int64_t workspace_bytes, void* out, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_fp8_linear";
  MLLM_REQUIRE(dtype == MLLM_DTYPE_BF16 || dtype == MLLM_DTYPE_F16, MLLM_ERR_UNSUPPORTED,
               fn + ": dtype must be bfloat16 or float16");
  MLLM_REQUIRE(m >= 0 && n > 0 && k > 0, MLLM_ERR_INVALID, fn + ": bad sizes");
  MLLM_REQUIRE(k % 16 == 0 && n % 16 == 0, MLLM_ERR_UNSUPPORTED, fn + ": k and n must be multiples of 16");
  // 32-bit offsets within a tile of 256 rows; launches below 2^31 workgroups
  MLLM_REQUIRE(k <= (1 << 23) && n < (1 << 28) && m < (1ll << 31) - 256, MLLM_ERR_UNSUPPORTED, fn + ": sizes too large");
  if (m == 0) return MLLM_OK;
  MLLM_REQUIRE(x && weight && weight_scales && out, MLLM_ERR_INVALID, fn + ": null pointer");
  MLLM_REQUIRE(((uintptr_t)x | (uintptr_t)weight | (uintptr_t)out) % 16 == 0 && x_stride % 8 == 0 &&
                   (uintptr_t)weight_scales % 4 == 0,
               MLLM_ERR_UNSUPPORTED, fn + ": operands must be 16-byte aligned");
  const int blocks = (int)((k + kBlock - 1) / kBlock);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const Plan p = plan_linear(m, n, blocks, device_cus());
  const int64_t need = p.xq_bytes + p.sx_bytes + p.part_bytes;
  MLLM_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 256 == 0 && workspace_bytes >= need), MLLM_ERR_INVALID,
               fn + ": workspace too small or not 256-byte aligned");
  const int64_t quant_groups = (m * blocks * 8 + 255) / 256;
  const int64_t bn = p.large ? 256 : 128;
  const int64_t tiles_n = (n + bn - 1) / bn, tiles_m = (m + bn - 1) / bn, groups = tiles_n * tiles_m * p.ksplit;
  MLLM_REQUIRE(p.rows || p.chunk || (quant_groups <= kMaxGroups256 && groups <= kMaxGroups256 / 2), MLLM_ERR_UNSUPPORTED,
               fn + ": too many rows");
  char* base = static_cast<char*>(workspace);
  uint8_t* sx = (uint8_t*)base + p.xq_bytes;
  RowsArgs r{(const char*)x, 2 * x_stride, (int)m, (int)k, (int)n, blocks, (const char*)weight, (const uint8_t*)weight_scales,
             (uint16_t*)out, (int)((n + kBlock - 1) / kBlock), p.ksplit, (float*)(sx + p.sx_bytes)};
  TileArgs a{base, sx, (const char*)weight, (const uint8_t*)weight_scales, (int)m, (int)n, blocks, (int)((m + 63) / 64),
             (int)tiles_n, (int)tiles_m, p.ksplit, (uint16_t*)out, (float*)(sx + p.sx_bytes)};
  auto launch = [&](auto tag) {
    using T = decltype(tag);
    if (p.rows) {
      if (m <= 8) return fp8_rows_kernel<T, true><<<(unsigned)(n / 16), 64 * kRowsWaves, 0, st>>>(r);
      return fp8_rows_kernel<T, false><<<(unsigned)(n / 16), 64 * kRowsWaves, 0, st>>>(r);
    }
    if (p.chunk) {
      const unsigned grid = (unsigned)(r.tiles * r.ksplit);
      if (m <= 8) return fp8_chunk_kernel<T, 1, true><<<grid, 64 * kRowsWaves, 0, st>>>(r);
      if (m <= 16) return fp8_chunk_kernel<T, 1, false><<<grid, 64 * kRowsWaves, 0, st>>>(r);
      if (m <= 32) return fp8_chunk_kernel<T, 2, false><<<grid, 64 * kRowsWaves, 0, st>>>(r);
      return fp8_chunk_kernel<T, 4, false><<<grid, 64 * kRowsWaves, 0, st>>>(r);
    }
    fp8_quant_kernel<T><<<(unsigned)quant_groups, 256, 0, st>>>((const char*)x, 2 * x_stride, (unsigned)m, (int)k, blocks, base, sx,
                                                               (unsigned)a.groups64);
    if (p.large)
      fp8_tile_kernel<T, 256, 256, 2, 4, 2, 2><<<(unsigned)groups, 512, 0, st>>>(a);
    else if (groups <= device_cus())
      fp8_tile_kernel<T, 128, 128, 2, 2, 1, 4><<<(unsigned)groups, 256, 0, st>>>(a);
    else
      fp8_tile_kernel<T, 128, 128, 2, 2, 2, 2><<<(unsigned)groups, 256, 0, st>>>(a);
  };
  if (dtype == MLLM_DTYPE_BF16)
    launch(BF16{});
  else
    launch(F16{});
  const int rc = check_launch(fn.c_str());
  if (rc != MLLM_OK || p.ksplit <= 1) return rc;
  return mllm_sum_partials(r.part, p.ksplit, m, n, nullptr, dtype, out, stream);
}
