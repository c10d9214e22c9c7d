// Copies of pages within the pools, of every layer's keys, values and scales in one call (no counterpart in the reference,
// which shares whole blocks alone): what a fork of a sequence or a compaction of a pool moves.
//
// Bound by memory: a page is read once and written once.  A wavefront moves rows of 1 KB, 16 bytes a lane, kRows of them in
// flight: 2,999 pages of 16 KB in 16 tensors, 1.57 GB, 325 us (4.8 TB/s, what a large copy reaches); with four rows 334, with
// plain loads and stores 385, with plain stores alone 360.  Eight pages of 32 KB in 64 tensors: 5.5 us.  Pages that are no whole
// number of such rows (scales) go word by word, one a thread; the eight pages would take 9.4 us that way, and 256 of 16 KB in 16
// tensors 26.3 instead of 23.2.
#include <vector>

#include "common.h"

namespace mllm {
namespace {

// The ids and the tensors travel in the kernel's arguments: nothing is uploaded, and a captured launch keeps them.
constexpr int kPairs = 256, kTensors = 128;
struct PagesArgs {
  char* base[kTensors];
  uint32_t bytes[kTensors];  // of a page
  int32_t src[kPairs], dst[kPairs];
  uint32_t pairs;
};

constexpr uint32_t kRowBytes = 1024;
constexpr int kRows = 8;

template <typename W>
__device__ __forceinline__ void copy_words(const PagesArgs& a, char* base, uint32_t bytes) {
  const uint32_t per = bytes / (uint32_t)sizeof(W), total = per * a.pairs;
  for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < total; i += gridDim.x * 256u) {
    const uint32_t p = i / per, w = i - p * per;
    reinterpret_cast<W*>(base + (int64_t)a.dst[p] * bytes)[w] = reinterpret_cast<const W*>(base + (int64_t)a.src[p] * bytes)[w];
  }
}

__global__ __launch_bounds__(256) void copy_pages_kernel(const PagesArgs a) {
  char* base = a.base[blockIdx.y];
  const uint32_t bytes = a.bytes[blockIdx.y];
  if (bytes % kRowBytes == 0 && (uintptr_t)base % 16 == 0) {
    const uint32_t per = bytes / kRowBytes, total = per * a.pairs;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const uint32_t first = wave * kRows;
    if (first >= total) return;
    uint32_t p = first / per, r = first - p * per;
    u32x4 x[kRows];
    char* to[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const bool in = first + i < total;  // uniform
      to[i] = nullptr;
      if (in) {
        const int64_t at = (int64_t)r * kRowBytes + 16 * lane;
        x[i] = ld16_nt(base + (int64_t)a.src[p] * bytes + at);
        to[i] = base + (int64_t)a.dst[p] * bytes + at;
      }
      if (++r == per) r = 0, ++p;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (first + i < total) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(to[i]));
    return;
  }
  if (bytes % 16 == 0 && (uintptr_t)base % 16 == 0)
    copy_words<u32x4>(a, base, bytes);
  else if (bytes % 4 == 0 && (uintptr_t)base % 4 == 0)
    copy_words<uint32_t>(a, base, bytes);
  else
    copy_words<uint8_t>(a, base, bytes);
}

}  // namespace
}  // namespace mllm

extern "C" int mllm_copy_pages(const uint64_t* tensors, const int64_t* page_bytes, int32_t num_tensors, int64_t num_pages,
                               const int64_t* src, const int64_t* dst, int64_t num_pairs, void* stream) {
  using namespace mllm;
  const std::string fn = "mllm_copy_pages";
  MLLM_REQUIRE(num_tensors >= 0 && num_pages >= 0 && num_pairs >= 0, MLLM_ERR_INVALID, fn + ": bad sizes");
  MLLM_REQUIRE(num_pages < (1ll << 31), MLLM_ERR_UNSUPPORTED, fn + ": too many pages");
  if (num_pairs == 0 || num_tensors == 0) return MLLM_OK;
  MLLM_REQUIRE(tensors && page_bytes && src && dst, MLLM_ERR_INVALID, fn + ": null pointer");
  uint32_t most = 0;
  for (int t = 0; t < num_tensors; ++t) {
    MLLM_REQUIRE(tensors[t], MLLM_ERR_INVALID, fn + ": null pointer");
    MLLM_REQUIRE(page_bytes[t] > 0 && page_bytes[t] < (1ll << 23), MLLM_ERR_UNSUPPORTED, fn + ": page too large");
    most = page_bytes[t] > most ? (uint32_t)page_bytes[t] : most;
  }
  try {  // sources as they were before the call: no page may be written twice, or written and read
    std::vector<uint8_t> seen((size_t)num_pages, 0);
    for (int64_t i = 0; i < num_pairs; ++i) {
      MLLM_REQUIRE(src[i] >= 0 && src[i] < num_pages && dst[i] >= 0 && dst[i] < num_pages, MLLM_ERR_INVALID,
                   fn + ": block " + std::to_string(src[i] < 0 || src[i] >= num_pages ? src[i] : dst[i]) + " is outside the pool");
      MLLM_REQUIRE(!seen[(size_t)dst[i]], MLLM_ERR_INVALID, fn + ": block " + std::to_string(dst[i]) + " is written twice");
      seen[(size_t)dst[i]] = 1;
    }
    for (int64_t i = 0; i < num_pairs; ++i)
      MLLM_REQUIRE(!seen[(size_t)src[i]], MLLM_ERR_INVALID, fn + ": block " + std::to_string(src[i]) + " is read and written");
  } catch (const std::exception& e) {
    return fail(MLLM_ERR_HIP, fn + ": out of host memory");
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  for (int t0 = 0; t0 < num_tensors; t0 += kTensors) {
    const int nt = num_tensors - t0 < kTensors ? num_tensors - t0 : kTensors;
    for (int64_t p0 = 0; p0 < num_pairs; p0 += kPairs) {
      PagesArgs a = {};
      for (int t = 0; t < nt; ++t) a.base[t] = (char*)(uintptr_t)tensors[t0 + t], a.bytes[t] = (uint32_t)page_bytes[t0 + t];
      a.pairs = (uint32_t)(num_pairs - p0 < kPairs ? num_pairs - p0 : kPairs);
      for (uint32_t i = 0; i < a.pairs; ++i) a.src[i] = (int32_t)src[p0 + i], a.dst[i] = (int32_t)dst[p0 + i];
      const uint64_t rows = (uint64_t)a.pairs * ((most + kRowBytes - 1) / kRowBytes);
      copy_pages_kernel<<<dim3((unsigned)((rows + 4 * kRows - 1) / (4 * kRows)), nt), 256, 0, st>>>(a);
    }
  }
  return check_launch(fn.c_str());
}
