// What the split-KV decode kernels of all pool types share: streaming loads, the position within a bin's pages, the
// plan's records (mllm_plan) and the sizes that follow from them.
#pragma once

#include "common.h"

namespace mllm {
namespace {

constexpr int kHeadDim = 128;

template <bool NT>
__device__ __forceinline__ u32x4 ldkv(const char* p) {
  if constexpr (NT)
    return ld16_nt(p);
  else
    return ld16(p);
}
template <bool NT>
__device__ __forceinline__ u32x2 ldkv8(const char* p) {
  if constexpr (NT)
    return __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
  else
    return ld8(p);
}

// The next 16-token tile to load: its page within the segment and its 16-token slice of that page (tiles
// are loaded in order, once each, so a counter replaces a division by the tiles per page).
struct LoadCursor {
  int page = 0, sub = 0;
  __device__ __forceinline__ void advance(int tpp) {
    if (++sub == tpp) {
      sub = 0;
      ++page;
    }
  }
};

// A segment's page ids, one per lane in three registers: pages 0-63, 64-127 and 128-191 of the segment
// (a bin holds at most kMaxSplitPages pages).
constexpr int kMaxSplitPages = 192;
struct PageIds {
  int r[3];
};
__device__ __forceinline__ PageIds load_page_ids(const int32_t* kv_indices, const int4& r0, int lane) {
  PageIds p;
#pragma unroll
  for (int i = 0; i < 3; ++i) p.r[i] = lane + 64 * i < r0.y ? kv_indices[r0.x + 64 * i + lane] : 0;
  return p;
}
// Page `page` (wave-uniform) of the segment.
__device__ __forceinline__ int page_id(const PageIds& p, int page) {
  return __builtin_amdgcn_readlane(page < 64 ? p.r[0] : (page < 128 ? p.r[1] : p.r[2]), page & 63);
}

// The records of one segment of a bin (the plan's layout): r0 = {first page in kv_indices, pages, first
// page within the row, row length}, r1 = {q row, partial slot or -1, sequence, 0}.
struct SegRec {
  int4 r0, r1;
};
// The plan is read through the constant address space: it does not change during the launch, so its
// uniform records become scalar loads, which the wave waits for with lgkmcnt apart from the vector
// loads of K, V and q (read as global memory, a record would be a vector load, and waiting for it would
// wait for every vector load issued before it).
typedef const __attribute__((address_space(4))) int PlanInt;
__device__ __forceinline__ int4 plan_rec(const int4* work, int i) {
  const PlanInt* p = (const PlanInt*)(work + i);
  return make_int4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ SegRec seg_rec(const int4* segs, int g) {
  return SegRec{plan_rec(segs, 2 * g), plan_rec(segs, 2 * g + 1)};
}

// Bins a plan of n_work records can hold: a header, then per bin one record and at least one segment
// of two records.  The grid covers that many bins; the workgroups past the step's own exit at once.
constexpr int max_bins(int n_work) { return n_work >= 4 ? (n_work - 1) / 3 : 0; }
// Partial slots a plan of n_work records can use: a cut row takes one slot per segment, and the segments
// take two records each after the header, so slots <= segments <= (n_work - 1) / 2.  The workspace holds
// that many slots: acc[slot][head][Dh], then (m, l)[slot][head].
constexpr int partial_slots(int n_work) { return n_work >= 1 ? (n_work - 1) / 2 : 0; }

}  // namespace
}  // namespace mllm
