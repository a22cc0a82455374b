// Device helpers shared by the decode attention kernels: buffer resources of a
// page, the lazily moved softmax maximum, the flat (sequence, kv head, page)
// space.
#pragma once
#include "xv_common.h"

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kNontemporal = 2;  // buffer instruction cache-policy bits: nt

// base and bytes are wave uniform: readfirstlane lets the compiler keep the
// resource in SGPRs (otherwise it emits a per-lane "waterfall" loop).
XV_INLINE __amdgpu_buffer_rsrc_t page_rsrc(const bf16_t* base, uint32_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
  void* q = reinterpret_cast<void*>(((uint64_t)hi << 32) | lo);
  return __builtin_amdgcn_make_buffer_rsrc(q, (short)0, (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// How far (log2) a head's maximum may pass the one in use before the sums are rescaled to it.
constexpr float kLazy = 8.0f;

// Value of head (4g+RR)%G -- the head of O row 4g+RR -- for a per-head value
// that is equal across the four 16-lane rows: lane (4g+RR)%G of this row.
// G == 16 is the cascade prefix pass: 16 distinct query rows per tile, so
// row 4g+RR's value sits in lane 4g+RR of the 16-lane row, which depends on g.
template <int G, int RR>
XV_INLINE float head_of_row(float x, int g) {
  if constexpr (G == 16) return __shfl(x, 20 * g + RR);
  else if constexpr (G == 8) return (g & 1) ? row_bcast<(4 + RR) % 8>(x) : row_bcast<RR % 8>(x);
  else return row_bcast<RR % G>(x);
}

// Sequence holding flat page f: the largest b with hkv*pref[b] <= f.
XV_INLINE int seq_of(const int* pref, int batch, int hkv, int64_t f) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)hkv * pref[mid] <= f) lo = mid; else hi = mid - 1;
  }
  return lo;
}

}  // namespace
