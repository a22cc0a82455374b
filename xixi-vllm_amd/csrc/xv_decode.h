// Device helpers shared by the decode attention kernels: buffer resources of a
// page, the lazily moved softmax maximum, the flat (sequence, kv head, page)
// space, the merge of partial outputs.
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

// Weighted merge of n partials of one (sequence, query head) by one wave:
// lane j holds partial j's weight (j < 64, then j - 64, j - 128 in two more
// registers); four groups of 16 lanes take every fourth partial, 8 dims per
// lane, 32 partials per batch of loads with two batches in flight, and the
// groups are summed by lane swaps.  part_vals(j, i, lo, hi) loads values
// 8i .. 8i + 7 of partial j, part_lse(j) is its log2-sum-exp; n <= kMergeMaxParts.
constexpr int kMergeMaxParts = 192;
// lse_lane: partial `lane`'s log2-sum-exp when the caller loaded it already
// (HAVE_LANE), so that it need not wait for a load after learning n.
template <bool HAVE_LANE, typename PV, typename PL>
XV_INLINE void merge_general(int n, PV part_vals, PL part_lse, float lse_lane, bf16_t* orow, int lane) {
  const float la = lane < n ? (HAVE_LANE ? lse_lane : part_lse(lane)) : -INFINITY;
  const float lb = 64 + lane < n ? part_lse(64 + lane) : -INFINITY;
  const float lc = 128 + lane < n ? part_lse(128 + lane) : -INFINITY;
  const float mx = wave_max(fmaxf(la, fmaxf(lb, lc)));
  const float wa = lane < n ? __builtin_amdgcn_exp2f(la - mx) : 0.f;
  const float wb = 64 + lane < n ? __builtin_amdgcn_exp2f(lb - mx) : 0.f;
  const float wc = 128 + lane < n ? __builtin_amdgcn_exp2f(lc - mx) : 0.f;
  const float den = wave_sum(wa + wb + wc);
  const int g = lane >> 4, i = lane & 15;  // group g: partials g, g + 4, ...; dims 8i .. 8i + 7
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto load = [&](float4 (&v)[8][2], int j0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      part_vals(min(j0 + 4 * k + g, n - 1), i, v[k][0], v[k][1]);
    }
  };
  auto fold = [&](const float4 (&v)[8][2], int j0) {
    // partial j's weight sits in lane j mod 64 of the register of its
    // 64-block; a batch (32 partials from j0, a multiple of 32) lies in one
    // block, and group g's partial of step k is j0 + 4k + g: four lane reads
    // into scalars, one per group
    const float wsrc = j0 < 64 ? wa : j0 < 128 ? wb : wc;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int j = j0 + 4 * k + g;
      const int s0 = (j0 + 4 * k) & 63;
      const float w0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wsrc), s0));
      const float w1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wsrc), s0 + 1));
      const float w2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wsrc), s0 + 2));
      const float w3 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wsrc), s0 + 3));
      const float w = j < n ? (g == 0 ? w0 : g == 1 ? w1 : g == 2 ? w2 : w3) : 0.f;
      acc[0] += w * v[k][0].x; acc[1] += w * v[k][0].y; acc[2] += w * v[k][0].z; acc[3] += w * v[k][0].w;
      acc[4] += w * v[k][1].x; acc[5] += w * v[k][1].y; acc[6] += w * v[k][1].z; acc[7] += w * v[k][1].w;
    }
  };
  float4 va[8][2], vb[8][2];
  load(va, 0);
  for (int j0 = 0; j0 < n; j0 += 64) {
    if (j0 + 32 < n) load(vb, j0 + 32);
    fold(va, j0);
    if (j0 + 32 < n) {
      if (j0 + 64 < n) load(va, j0 + 64);
      fold(vb, j0 + 32);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = xor32_sum(xor16_sum(acc[e]));
  if (g == 0) {
    const float inv = 1.0f / den;
    uint32_t* o = reinterpret_cast<uint32_t*>(orow + 8 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
  }
}

}  // namespace
