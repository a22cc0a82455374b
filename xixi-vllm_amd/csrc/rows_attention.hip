// Paged attention of a few query rows per sequence for gfx950: decode with a
// sliding window and sinks (one row per query head), and trees of drafted
// tokens (one row per node and query head).
//
//   out[r] = sum_t softmax_t(scale * q[r] . K[t]) V[t] over the tokens t row r sees
//   window: row at position p = ctx - 1 sees t > p - window, and t < sinks
//   tree:   node i of n, token ctx - n + i, sees t < ctx - n and the nodes of its mask
//
// Work split: a sequence's visible 16-token pages in order (the sinks' pages,
// then the window's) make its units of two pages.  The (sequence, kv head,
// unit) space is flattened in that order and cut into equal contiguous ranges;
// a range cut inside a segment leaves partials (normalised fp32 rows and their
// log2-sum-exp) for a merge kernel, two partial slots per range at most.
// A wave takes NT tiles of 16 rows, 1 or 2; trees of more rows, and few ones of
// more than 16, are the matter of tree_tiles.hip.
//
// A unit (32 tokens), all on v_mfma_f32_16x16x32_bf16:
//   K and V rows go HBM -> LDS by LDS-DMA, two units in flight per wave.
//   S^T = K Q^T: operand A is K as stored, B the rows' q.  Lane (g, c) gets
//   row c's scores of tokens 4g .. 4g+3 of both pages, which are the k
//   indices that lane group supplies to the second product:
//   O^T = V^T P^T: A is V read transposed (ds_read_b64_tr_b16), B is P in
//   the lanes where the scores landed.  O^T has row c in lane c too, so the
//   softmax maximum, sum and rescale stay in the lane.
//
// Bound by the stream of pages where there is enough of it (a large copy
// reaches 6.5 TB/s): 64 sequences with a window of 2048 and 32 / 8 heads,
// 516 MB, 85 us (6.1 TB/s); 200 padded rows with a window of 1000 and 64 / 8
// heads, 750 MB, 131 us (5.7 TB/s).  One sequence with a window of 4096,
// 17 MB, takes 7.5 us, and its merge 5.6: four trips to memory one after the
// other (lengths, page ids, pages; partial counts and partials).
#include "xv_common.h"
#include "xv_kernels.h"
#include "xv_rows.h"
#include <math.h>

using namespace xv_rows;

namespace {

constexpr int kD = 128;
constexpr int kUnit = 32;          // tokens of a unit: two pages
constexpr int kWaves = 4;          // waves of a workgroup, one workgroup per CU
constexpr int kMaxGroups = 256;    // workgroups at most
constexpr int kHalf = 4096;        // a page's K (or V) rows in LDS
constexpr int kUnitLds = 4 * kHalf;  // page A: K, V; page B: K, V
constexpr int kUnitOps = 16;       // LDS-DMA instructions a unit
constexpr int kIdWindow = 32;      // units per half of the block-id table (2 ids each)
constexpr int kWaveLds = 2 * kUnitLds + 2 * kIdWindow * 8;

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

XV_INLINE u32x2_t lds_ids(const char* p) {
  u32x2_t v;
  __asm__ __volatile__("ds_read_b64 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                       : "=&v"(v)
                       : "v"((uint32_t)reinterpret_cast<uintptr_t>(p))
                       : "memory");
  return v;
}

// Which pages of a sequence its rows see: pages 0 .. sink - 1 and sink + skip ..,
// `list` of them in all.
struct Pages {
  int lo;    // first token of the window
  int sink, skip, list;
};
template <bool TREE>
XV_INLINE Pages pages_of(int ctx, int window, int sinks) {
  const int np = (ctx + kPage - 1) / kPage;
  if (TREE) return Pages{0, 0, 0, np};
  Pages p;
  p.lo = max(0, ctx - window);
  p.sink = (min(sinks, p.lo) + kPage - 1) / kPage;
  p.skip = max(0, p.lo / kPage - p.sink);
  p.list = np - p.skip;
  return p;
}
XV_INLINE int page_at(const Pages& p, int i) { return i < p.sink ? i : i + p.skip; }
template <bool TREE>
XV_INLINE int units_of(int ctx, int window, int sinks) {
  return (pages_of<TREE>(ctx, window, sinks).list + 1) / 2;
}

// LDS image of a page's K or V rows of one kv head: token t's 256-byte row at
// 256 t, its 16-byte chunk c in slot c ^ swz(t): conflict-free K reads (one
// chunk of 16 tokens) and transposed V reads.
XV_INLINE int swz(int t) { return ((t & 7) << 1) | (t >> 3); }

struct RowsLane {
  int g[4];        // global byte offset of load instruction s within a page
  uint32_t k[4];   // K operand of product step s
  uint32_t v[8];   // transposed V read of d-tile n
};
XV_INLINE RowsLane lane_offsets(int64_t tok_stride, int lane) {
  RowsLane o;
  const int i = lane & 15, g = lane >> 4;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int t = 4 * s + g;
    o.g[s] = (int)(t * tok_stride * 2) + ((i ^ swz(t)) << 4);
    o.k[s] = (uint32_t)(i * 256 + (((4 * s + g) ^ swz(i)) << 4));
  }
  const int t = 4 * g + (i >> 2);
#pragma unroll
  for (int n = 0; n < 8; ++n)
    o.v[n] = (uint32_t)(kHalf + t * 256 + (((2 * n + ((i & 3) >> 1)) ^ swz(t)) << 4) + 8 * (i & 1));
  return o;
}

struct UnitRegs {
  bf16x8_t k[2][4];   // K operands of the two pages
  short4_t v[2][8];   // transposed V of d-tile n: tokens 4g .. 4g+3
};
// A unit's operands out of its LDS image (its loads have arrived), in one asm block with one wait.
XV_INLINE void read_unit(UnitRegs& u, const char* buf, const RowsLane& lo) {
  const uint32_t b = (uint32_t)reinterpret_cast<uintptr_t>(buf);
  static_assert(2 * kHalf == 8192, "the offsets below");
  __asm__ __volatile__(
      "ds_read_b128 %0, %24\n\t"
      "ds_read_b128 %1, %25\n\t"
      "ds_read_b128 %2, %26\n\t"
      "ds_read_b128 %3, %27\n\t"
      "ds_read_b128 %4, %24 offset:8192\n\t"
      "ds_read_b128 %5, %25 offset:8192\n\t"
      "ds_read_b128 %6, %26 offset:8192\n\t"
      "ds_read_b128 %7, %27 offset:8192\n\t"
      "ds_read_b64_tr_b16 %8, %28\n\t"
      "ds_read_b64_tr_b16 %9, %29\n\t"
      "ds_read_b64_tr_b16 %10, %30\n\t"
      "ds_read_b64_tr_b16 %11, %31\n\t"
      "ds_read_b64_tr_b16 %12, %32\n\t"
      "ds_read_b64_tr_b16 %13, %33\n\t"
      "ds_read_b64_tr_b16 %14, %34\n\t"
      "ds_read_b64_tr_b16 %15, %35\n\t"
      "ds_read_b64_tr_b16 %16, %28 offset:8192\n\t"
      "ds_read_b64_tr_b16 %17, %29 offset:8192\n\t"
      "ds_read_b64_tr_b16 %18, %30 offset:8192\n\t"
      "ds_read_b64_tr_b16 %19, %31 offset:8192\n\t"
      "ds_read_b64_tr_b16 %20, %32 offset:8192\n\t"
      "ds_read_b64_tr_b16 %21, %33 offset:8192\n\t"
      "ds_read_b64_tr_b16 %22, %34 offset:8192\n\t"
      "ds_read_b64_tr_b16 %23, %35 offset:8192\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(u.k[0][0]), "=&v"(u.k[0][1]), "=&v"(u.k[0][2]), "=&v"(u.k[0][3]), "=&v"(u.k[1][0]), "=&v"(u.k[1][1]),
        "=&v"(u.k[1][2]), "=&v"(u.k[1][3]), "=&v"(u.v[0][0]), "=&v"(u.v[0][1]), "=&v"(u.v[0][2]), "=&v"(u.v[0][3]),
        "=&v"(u.v[0][4]), "=&v"(u.v[0][5]), "=&v"(u.v[0][6]), "=&v"(u.v[0][7]), "=&v"(u.v[1][0]), "=&v"(u.v[1][1]),
        "=&v"(u.v[1][2]), "=&v"(u.v[1][3]), "=&v"(u.v[1][4]), "=&v"(u.v[1][5]), "=&v"(u.v[1][6]), "=&v"(u.v[1][7])
      : "v"(b + lo.k[0]), "v"(b + lo.k[1]), "v"(b + lo.k[2]), "v"(b + lo.k[3]), "v"(b + lo.v[0]), "v"(b + lo.v[1]),
        "v"(b + lo.v[2]), "v"(b + lo.v[3]), "v"(b + lo.v[4]), "v"(b + lo.v[5]), "v"(b + lo.v[6]), "v"(b + lo.v[7])
      : "memory");
}

template <int NT>
struct RowsState {
  float m[NT];          // the softmax maximum in use (log2 domain) of row c of each tile, the same in the four lane rows
  float l[NT];          // sum of p over this lane's tokens
  floatx4_t o[NT][8];   // O^T of d-tile n: d = 16n + 4g + r, row c
};

// Scores, softmax update and O^T += V^T P^T of one unit.  EDGE: seen[t] has the tokens that row c of tile t sees.
template <int NT, bool EDGE>
XV_INLINE void unit_math(RowsState<NT>& st, const UnitRegs& u, const bf16x8_t (&qb)[NT][4], const uint32_t (&seen)[NT],
                         float scale_log2, int lane) {
  const int g = lane >> 4;
  floatx4_t a[NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) a[t][0] = a[t][1] = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int t = 0; t < NT; ++t) a[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u.k[p][s], qb[t][s], a[t][p], 0, 0, 0);
  bf16x8_t pb[NT];
  uint32_t any = 0;  // tokens that some row of the wave sees
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const uint32_t bits = seen[t] >> (4 * g);  // bit r: token 4g + r, bit 16 + r: the second page's
    any |= seen[t];
    if (EDGE) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) a[t][p][r] = (bits >> (16 * p + r)) & 1 ? a[t][p][r] : -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(a[t][0][0], a[t][0][1]), fmaxf(a[t][0][2], a[t][0][3])),
                     fmaxf(fmaxf(a[t][1][0], a[t][1][1]), fmaxf(a[t][1][2], a[t][1][3])));
    mx = xor32_max(xor16_max(mx)) * scale_log2;
    // the maximum in use moves only when some row's grew by more than kLazy
    const float m_new = fmaxf(st.m[t], mx);
    if (__any(m_new > st.m[t] + kLazy)) {
      const float alpha = st.m[t] == m_new ? 1.f : __builtin_amdgcn_exp2f(st.m[t] - m_new);
      st.m[t] = m_new;
      st.l[t] *= alpha;
#pragma unroll
      for (int n = 0; n < 8; ++n) st.o[t][n] *= alpha;
    }
    const float nm = EDGE && st.m[t] == -INFINITY ? 0.f : -st.m[t];  // a row that has seen nothing yet: p = 0
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = e >> 1, r = 2 * (e & 1);
      const float p0 = __builtin_amdgcn_exp2f(fmaf(a[t][p][r], scale_log2, nm));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(a[t][p][r + 1], scale_log2, nm));
      w[e] = pack_bf16x2(p0, p1);
      // the row sum takes the bf16 weights that the product multiplies: their rounding (2^-8 of a weight at most) moves
      // the output by that share of the values' spread only, and a row of one heavy token is exact
      st.l[t] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(xv_bf16x2, w[e]),
                                                (xv_bf16x2){(__bf16)1.0f, (__bf16)1.0f}, st.l[t], false);
    }
    __builtin_memcpy(&pb[t], w, 16);
  }
  uint32_t keep[4];
  if (EDGE) {  // V of tokens that no row sees may be anything, NaN included: read as zeros
    any |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)any, 0x128, 0xf, 0xf, false);
    any |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)any, 0x124, 0xf, 0xf, false);
    any |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)any, 0x4E, 0xf, 0xf, false);
    any |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)any, 0xB1, 0xf, 0xf, false);
    any >>= 4 * g;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t two = any >> (16 * (e >> 1) + 2 * (e & 1));
      keep[e] = (two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
    }
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    bf16x8_t v = __builtin_bit_cast(bf16x8_t, (short8_t)__builtin_shufflevector(u.v[0][n], u.v[1][n], 0, 1, 2, 3, 4, 5, 6, 7));
    if (EDGE) {
      u32x4_t w = __builtin_bit_cast(u32x4_t, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] &= keep[e];
      v = __builtin_bit_cast(bf16x8_t, w);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) st.o[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb[t], st.o[t][n], 0, 0, 0);
  }
}

template <int NT>
XV_INLINE void reset(RowsState<NT>& st) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    st.m[t] = -INFINITY;
    st.l[t] = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) st.o[t][n] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  }
}

// The finished segment's rows: bf16 output if the range covered the whole
// segment (slot < 0), else fp32 rows of partial slot `slot`.
template <int NT>
XV_INLINE void finish_rows(const RowsArgs& a, const RowsState<NT>& st, int tok0, int kvh, int nrows, int slot, int lane) {
  typedef u32x2_t __attribute__((aligned(4))) u32x2_a4;  // the caller's rows need not be 8-byte aligned
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = 16 * t + c;
    const float lsum = xor32_sum(xor16_sum(st.l[t]));
    const float inv = lsum == 0.f ? 0.f : 1.0f / lsum;  // a row that sees nothing: zeros; NaN stays NaN
    if (row >= nrows) continue;
    if (slot < 0) {
      const int node = row >> a.glog, h = (kvh << a.glog) + (row & ((1 << a.glog) - 1));
      bf16_t* dst = a.out + (int64_t)(tok0 + node) * a.out_st + (int64_t)h * kD + 4 * g;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const floatx4_t o = st.o[t][n];
        *reinterpret_cast<u32x2_a4*>(dst + 16 * n) = u32x2_t{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
      }
    } else {
      const int64_t at = (int64_t)slot * a.rows + row;
      float* dst = a.ws_o + at * kD + 4 * g;
#pragma unroll
      for (int n = 0; n < 8; ++n) *reinterpret_cast<floatx4_t*>(dst + 16 * n) = st.o[t][n] * inv;
      if (g == 0) a.ws_lse[at] = lsum == 0.f ? -INFINITY : st.m[t] + __log2f(lsum);
    }
  }
}

// Block ids of the range's units, two pages each, in a double-buffered LDS
// table filled by LDS-DMA from the block table.  Units past the range, and
// pages past a sequence's list, fetch an entry that exists.
template <bool TREE>
XV_INLINE void load_window(char* half, const RowsArgs& a, __amdgpu_buffer_rsrc_t rbt, const Sequences& s,
                           int64_t f0, int base, int n, int lane) {
  static_assert(kIdWindow * 2 == 64, "one id per lane");
  const int y = base + (lane >> 1);
  int off = 0;
  if (y < n) {
    const int64_t f = f0 + y;
    const int b = seq_of(s.pref, a.batch, a.hkv, f);
    const int nu = s.pref[b + 1] - s.pref[b];
    const int u = (int)(f - (int64_t)a.hkv * s.pref[b]) % nu;
    const Pages p = pages_of<TREE>(s.ctx[b], a.window, a.sinks);
    const int page = page_at(p, min(2 * u + (lane & 1), p.list - 1));
    off = (int)(((int64_t)b * a.bt_stride + page / a.nsub) * 4);
  }
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rbt, (lds_void*)half, 4, off, 0, 0, 0);
}

// Nodes of its sequence that lane's row of tile t sees, as bits of the unit whose first token is tok0 = P + at.
XV_INLINE uint32_t node_bits(const uint64_t* words, int n, int at) {
  if (at < 0) return (uint32_t)(words[0] << -at) | low_bits(-at);
  const int w = at >> 6, off = at & 63;
  uint64_t v = w < n ? words[w] >> off : 0;
  if (off > 32 && w + 1 < n) v |= words[w + 1] << (64 - off);
  return (uint32_t)v;
}

template <int NT, bool TREE>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(1, 1))) void rows_kernel(RowsArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kWaveLds];
  __shared__ Sequences seqs;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave == 0)
    load_sequences<TREE, false>(seqs, a, lane, [&](int ctx) { return units_of<TREE>(ctx, a.window, a.sinks); });
  __syncthreads();
  const Ranges rg = ranges_of<false>(seqs, a, gridDim.x * kWaves, lane);
  const int L = rg.len;
  const int id = wave * gridDim.x + blockIdx.x;  // short launches spread over the CUs first
  const int64_t f0 = (int64_t)id * L;
  const int n = (int)max((int64_t)0, min(f0 + L, rg.total) - f0);
  if (n == 0) return;
  char* const mine = lds + wave * kWaveLds;
  char* const idtab = mine + 2 * kUnitLds;
  const RowsLane offs = lane_offsets(a.ts, lane);

  Cursor ic = cursor_at<false>(seqs, a, f0), pc = ic;  // issue and process cursors
  const __amdgpu_buffer_rsrc_t rbt =
      page_rsrc(reinterpret_cast<const bf16_t*>(a.bt), (uint32_t)((int64_t)a.batch * a.bt_stride * 4));
  load_window<TREE>(idtab, a, rbt, seqs, f0, 0, n, lane);
  if (n > kIdWindow) load_window<TREE>(idtab + kIdWindow * 8, a, rbt, seqs, f0, kIdWindow, n, lane);
  __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");

  const uint32_t page_bytes = (uint32_t)((15 * a.ts + kD) * 2);
  // Unit y, whose cursor is ic, into its ring slot.  Whole pages: tokens that no row sees are masked later.
  auto issue = [&](int y) {
    char* buf = mine + (y & 1) * kUnitLds;
    if (y % kIdWindow == 0 && y > 0)  // entering window k (in place since window k - 1 began): request window k + 1
      load_window<TREE>(idtab + ((y / kIdWindow + 1) & 1) * (kIdWindow * 8), a, rbt, seqs, f0, y + kIdWindow, n, lane);
    const u32x2_t ids = lds_ids(idtab + ((y / kIdWindow) & 1) * (kIdWindow * 8) + (y % kIdWindow) * 8);
    const Pages p = pages_of<TREE>(ic.ctx, a.window, a.sinks);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int page = page_at(p, min(2 * ic.u + j, p.list - 1));
      const int64_t id = (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)ids[j]);
      const int64_t base = id * a.ps + (int64_t)(page % a.nsub) * kPage * a.ts + (int64_t)ic.kvh * a.hs;
      const __amdgpu_buffer_rsrc_t rk = page_rsrc(a.kc + base, page_bytes), rv = page_rsrc(a.vc + base, page_bytes);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(buf + 2 * kHalf * j + 1024 * s), 16, offs.g[s], 0, 0,
                                                 kNontemporal);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(buf + 2 * kHalf * j + kHalf + 1024 * s), 16, offs.g[s], 0, 0,
                                                 kNontemporal);
      }
    }
  };

  RowsState<NT> st;
  bf16x8_t qb[NT][4];
  int tok0 = 0, nrows = 0;  // the segment's first row of q, and its rows
  auto finish = [&](const Cursor& c) {
    finish_rows<NT>(a, st, tok0, c.kvh, nrows, finish_slot(seqs, a, c, f0, n, id, L, lane == 0), lane);
  };
  auto row_of = [&](int t) { return min(16 * t + (lane & 15), nrows - 1); };  // rows past the last: the last again
  auto begin = [&] {
    tok0 = lds_int(seqs.cq + pc.b);
    nrows = (TREE ? lds_int(seqs.cq + pc.b + 1) - tok0 : 1) << a.glog;
    reset(st);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = row_of(t);
      const bf16_t* src = a.q + (int64_t)(tok0 + (row >> a.glog)) * a.q_st +
                          (int64_t)((pc.kvh << a.glog) + (row & ((1 << a.glog) - 1))) * a.q_sh + 8 * (lane >> 4);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        Vec8 v = load_vec8(src + 32 * s);
#pragma unroll
        for (int e = 0; e < 4; ++e) v.w[e] = (v.w[e] & a.q_keep) ^ a.q_flip;
        __builtin_memcpy(&qb[t][s], &v, 16);
      }
    }
  };
  issue(0);
  if (n > 1) {
    advance<false>(ic, seqs, a);
    issue(1);
  }
  UnitRegs u;
  for (int x = 0; x < n; ++x) {
    const Cursor prev = pc;
    if (x > 0) advance<false>(pc, seqs, a);
    if (x == 0 || pc.u == 0) {
      if (x > 0) finish(prev);
      begin();
    }
    static_assert(kUnitOps == 16, "the wait below");
    if (x + 1 < n) __asm__ __volatile__("s_waitcnt vmcnt(16)" ::: "memory");
    else __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");
    read_unit(u, mine + (x & 1) * kUnitLds, offs);
    if (x + 2 < n) {
      advance<false>(ic, seqs, a);
      issue(x + 2);
    }
    const Pages p = pages_of<TREE>(pc.ctx, a.window, a.sinks);
    uint32_t seen[NT];
    bool edge;
    if (TREE) {
      const int t0 = pc.u * kUnit, nodes = nrows >> a.glog, at = t0 - (pc.ctx - nodes);
      edge = at + kUnit > 0;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        seen[t] = ~0u;
        if (edge) seen[t] = node_bits(a.mask + (int64_t)(tok0 + (row_of(t) >> a.glog)) * a.mask_st, a.words, at) & low_bits(pc.ctx - t0);
      }
    } else {
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int i = 2 * pc.u + j;
        if (i >= p.list) break;
        const int t0 = kPage * page_at(p, i);
        bits |= (low_bits(min(pc.ctx - t0, kPage)) & (low_bits(a.sinks - t0) | ~low_bits(p.lo - t0))) << (16 * j);
      }
      edge = bits != ~0u;
#pragma unroll
      for (int t = 0; t < NT; ++t) seen[t] = bits;
    }
    if (edge) unit_math<NT, true>(st, u, qb, seen, a.scale_log2, lane);
    else unit_math<NT, false>(st, u, qb, seen, a.scale_log2, lane);
  }
  finish(pc);
}

// One wave per row (node, query head) of sequence blockIdx.y, four a
// workgroup: zeros for an empty sequence, else the sum of its partials, each
// by its share of the segment's mass, where the segment was cut.  16 lanes
// hold a row (8 values each), the four lane rows take every fourth partial,
// four in flight each.
template <bool TREE>
__global__ __launch_bounds__(256) void rows_merge_kernel(RowsArgs a) {
  const int task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
  const int b = blockIdx.y;
  const int node = task / a.hq, h = task - node * a.hq;
  const int tok0 = TREE ? a.cu_q[b] : b;
  if (node >= (TREE ? min(a.max_nodes, a.cu_q[b + 1] - tok0) : 1)) return;
  const int kvh = h >> a.glog, r0 = (node << a.glog) + (h & ((1 << a.glog) - 1));
  const int ctx = a.seqlens[b];
  const int2 seg = a.ws_seg[seg_index(a, b, r0 / kPassRows, kvh)];  // stale when ctx <= 0: not used then
  bf16_t* orow = a.out + (int64_t)(tok0 + node) * a.out_st + (int64_t)h * kD;
  if (ctx <= 0) {
    *reinterpret_cast<uint32_t*>(orow + 2 * lane) = 0u;
    return;
  }
  const int n = seg.y;
  if (n <= 1) return;
  auto slot = [&](int j) { return (int64_t)(j == 0 ? 2 * seg.x + 1 : 2 * (seg.x + j)) * a.rows + r0 % kPassRows; };
  const int g = lane >> 4, i = lane & 15;
  constexpr int kAhead = 4;  // partials in flight per lane row
  floatx4_t r[kAhead][2];
  auto load = [&](int k, int j) {
    const floatx4_t* from = reinterpret_cast<const floatx4_t*>(a.ws_o + slot(min(j, n - 1)) * kD + 8 * i);
    r[k][0] = from[0];
    r[k][1] = from[1];
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (4 * k < n) load(k, 4 * k + g);
  // lane j: the log2-sum-exps of partials j, 64 + j, 128 + j
  const float la = lane < n ? a.ws_lse[slot(lane)] : -INFINITY;
  float lb = -INFINITY, lc = -INFINITY;
  if (n > 64) {
    if (64 + lane < n) lb = a.ws_lse[slot(64 + lane)];
    if (128 + lane < n) lc = a.ws_lse[slot(128 + lane)];
  }
  float mx = wave_max(fmaxf(la, fmaxf(lb, lc)));
  if (mx == -INFINITY) mx = 0.f;  // the row sees nothing: weights of 0
  float wa = __builtin_amdgcn_exp2f(la - mx), wb = __builtin_amdgcn_exp2f(lb - mx), wc = __builtin_amdgcn_exp2f(lc - mx);
  const float mass = wave_sum(wa + wb + wc);
  const float inv = mass == 0.f ? 0.f : 1.0f / mass;
  wa *= inv; wb *= inv; wc *= inv;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  auto fold = [&](floatx4_t lo, floatx4_t hi, int j) {  // partial j of this lane row (the four rows' lie in one block of 64)
    const float w = __shfl(j < 64 ? wa : j < 128 ? wb : wc, j & 63);
    if (j < n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[e] += w * lo[e];
        acc[4 + e] += w * hi[e];
      }
    }
  };
  for (int j0 = 0; j0 < n; j0 += 4 * kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int j = j0 + 4 * k;
      if (j >= n) break;
      const floatx4_t lo = r[k][0], hi = r[k][1];
      if (j + 4 * kAhead < n) load(k, j + 4 * kAhead + g);
      fold(lo, hi, j + g);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = xor32_sum(xor16_sum(acc[e]));
  if (g == 0) {
    uint32_t* o = reinterpret_cast<uint32_t*>(orow + 8 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(acc[2 * e], acc[2 * e + 1]);
  }
}

// The same for many rows of few partials: four rows a wave, 16 lanes each (8 values a lane), one partial after the
// other, four in flight.
__global__ __launch_bounds__(256) void rows_merge4_kernel(RowsArgs a) {
  const int lane = threadIdx.x & 63, i = lane & 15;
  const int task = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 4 + (lane >> 4), b = blockIdx.y;
  const int node = task / a.hq, h = task - node * a.hq;
  const int tok0 = a.cu_q[b];
  if (node >= min(a.max_nodes, a.cu_q[b + 1] - tok0)) return;
  const int kvh = h >> a.glog, r0 = (node << a.glog) + (h & ((1 << a.glog) - 1));
  const int ctx = a.seqlens[b];
  const int2 seg = a.ws_seg[seg_index(a, b, r0 / kPassRows, kvh)];  // stale when ctx <= 0: not used then
  uint32_t* orow = reinterpret_cast<uint32_t*>(a.out + (int64_t)(tok0 + node) * a.out_st + (int64_t)h * kD + 8 * i);
  if (ctx <= 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) orow[e] = 0u;
    return;
  }
  const int n = seg.y;
  if (n <= 1) return;
  auto slot = [&](int j) { return (int64_t)(j == 0 ? 2 * seg.x + 1 : 2 * (seg.x + j)) * a.rows + r0 % kPassRows; };
  float mx = -INFINITY;
  for (int j = i; j < n; j += 16) mx = fmaxf(mx, a.ws_lse[slot(j)]);
  mx = row16_max(mx);
  if (mx == -INFINITY) mx = 0.f;  // the row sees nothing: weights of 0
  float mass = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < n; j0 += 4) {
    float lse[4];
    floatx4_t lo[4], hi[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t at = slot(min(j0 + k, n - 1));
      const floatx4_t* from = reinterpret_cast<const floatx4_t*>(a.ws_o + at * kD + 8 * i);
      lse[k] = a.ws_lse[at];
      lo[k] = from[0];
      hi[k] = from[1];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = j0 + k < n ? __builtin_amdgcn_exp2f(lse[k] - mx) : 0.f;
      mass += w;
      if (j0 + k < n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[e] += w * lo[k][e];
          acc[4 + e] += w * hi[k][e];
        }
      }
    }
  }
  const float inv = mass == 0.f ? 0.f : 1.0f / mass;
#pragma unroll
  for (int e = 0; e < 4; ++e) orow[e] = pack_bf16x2(acc[2 * e] * inv, acc[2 * e + 1] * inv);
}

int rows_groups() {
  static int cached = 0;  // one GPU model per process
  if (!cached) {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      cus = kMaxGroups;
    cached = max(1, min(kMaxGroups, cus));
  }
  return cached;
}

// Trees of up to 16 rows per sequence and kv head (nodes times query heads per kv head) run here, a wave on its own; those
// of more than 32 share their tiles among the waves of a workgroup (tree_tiles.hip).  Between the two it goes by the
// (sequence, kv head) segments: no more than the workgroups there, and a segment is cut into more ranges here, which
// the merge then joins.  Captured calls of 32 rows, 8 kv heads (here, there, us):
//   sequences        1           4           32          64          128         256
//   300 tokens     9.6, 10.6  12.5, 11.6   28.4, 18.1  30.3, 27.5  36.8, 45.4   73, 92
//   1000          11.4, 11.1  21.7, 13.7   36.7, 31.8  57.7, 55.2    91, 113   186, 222
//   4000          24.6, 15.4  30.9, 24.9  103.2, 100.3  177, 192
//   16000         32.5, 25.0  59.6, 55.4
//   60000         59.3, 52.8   175, 194
// So up to 32 sequences of 8 kv heads go there (20 rows: as these).  What that costs is 5 to 11 % where they hold more than
// 100000 tokens together: the host knows the tables' width, not their lengths.
constexpr int kWaveRows = 32;
bool by_tiles(int batch, int hkv, int max_rows) {
  return max_rows > kWaveRows || (max_rows > 16 && (int64_t)batch * hkv <= kTileGroups);
}
// Rows of a tree call from which on the merge takes four rows a wave: enough waves then without spreading a row's partials.
// Four and one a wave, the whole call, captured: 2048 rows 37.9 and 34.8 us, 17.6 and 16.7; 4096 44.4 and 44.0, 25.5 and
// 25.8; 8192 35.8 and 37.6, 102.4 and 104.2 (60.8 and 59.3 in the one case that is the other way); 16384 48.0 and 49.4;
// 65536 34.2 and 41.0.
constexpr int kManyRows = 8192;
int slot_rows(int max_rows, bool tiles) { return tiles ? kPassRows : max_rows <= 16 ? 16 : 32; }
size_t slots(bool tiles) { return 2 * (size_t)(tiles ? kTileGroups : kMaxGroups * kWaves); }

size_t al256(size_t x) { return (x + 255) / 256 * 256; }
int row_passes(int max_rows) { return (max_rows + kPassRows - 1) / kPassRows; }
size_t seg_bytes(int batch, int hkv, int max_rows) {
  return al256((size_t)row_passes(max_rows) * min(batch, kMaxBatch) * hkv * sizeof(int2));
}
size_t lse_bytes(int max_rows, bool tiles) { return al256(slots(tiles) * slot_rows(max_rows, tiles) * sizeof(float)); }

bool valid_group(int hq, int hkv) {
  if (hkv <= 0 || hq <= 0 || hq % hkv) return false;
  const int g = hq / hkv;
  return g == 1 || g == 2 || g == 4 || g == 8;
}

template <bool TREE>
int launch_rows(RowsArgs a, const bf16_t* q, const int32_t* bt, const int32_t* seqlens, const int32_t* cu_q, bf16_t* out,
                int batch, int max_nodes, void* workspace, hipStream_t stream) {
  const int max_rows = max_nodes << a.glog;
  const bool tiles = TREE && by_tiles(batch, a.hkv, max_rows);
  a.rows = slot_rows(max_rows, tiles);
  a.max_nodes = max_nodes;
  a.passes = row_passes(max_rows);
  a.ws_seg = (int2*)workspace;
  a.ws_lse = (float*)((char*)workspace + seg_bytes(batch, a.hkv, max_rows));
  a.ws_o = (float*)((char*)a.ws_lse + lse_bytes(max_rows, tiles));
  // units that the widest visible list may hold
  const int64_t pages = TREE ? (a.max_ctx + kPage - 1) / kPage
                             : min((int64_t)(a.max_ctx + kPage - 1) / kPage,
                                   ((int64_t)a.window + kPage - 1) / kPage + ((int64_t)a.sinks + kPage - 1) / kPage + 1);
  for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {
    a.batch = min(kMaxBatch, batch - b0);
    a.q = TREE ? q : q + (int64_t)b0 * a.q_st;
    a.out = TREE ? out : out + (int64_t)b0 * a.out_st;
    a.cu_q = TREE ? cu_q + b0 : nullptr;
    a.bt = bt + (int64_t)b0 * a.bt_stride;
    a.seqlens = seqlens + b0;
    const int64_t units = (int64_t)a.batch * a.hkv * ((pages + 1) / 2);
    const unsigned groups = (unsigned)min((int64_t)rows_groups(), units);
    if (max_rows <= 16) {
      rows_kernel<1, TREE><<<groups, kWaves * 64, 0, stream>>>(a);
    } else if constexpr (TREE) {
      if (!tiles) {
        rows_kernel<2, TREE><<<groups, kWaves * 64, 0, stream>>>(a);
      } else {
        const int e = launch_tiles(a, stream);
        if (e) return e;
      }
    }
    XV_CHECK_LAUNCH();
    const int64_t per_seq = (int64_t)max_nodes * a.hq;
    if (TREE && per_seq * a.batch >= kManyRows)
      rows_merge4_kernel<<<dim3((unsigned)((per_seq + 15) / 16), (unsigned)a.batch), 256, 0, stream>>>(a);
    else
      rows_merge_kernel<TREE><<<dim3((unsigned)((per_seq + 3) / 4), (unsigned)a.batch), 256, 0, stream>>>(a);
    XV_CHECK_LAUNCH();
  }
  return 0;
}

// Checks shared by the two entries; fills the record's cache and table fields.
bool rows_args(RowsArgs& a, const void* q, int64_t q_st, int64_t q_sh, const void* kc, const void* vc, int64_t ps, int64_t ts,
               int64_t hs, int64_t bt_stride, const void* out, int64_t out_st, int batch, int hq, int hkv, int head_dim,
               int block_size, int max_blocks, int passes, float scale) {
  if (head_dim != kD || block_size <= 0 || block_size % kPage || batch < 0 || !valid_group(hq, hkv) || max_blocks <= 0) return false;
  const int64_t max_ctx = (int64_t)max_blocks * block_size;
  // 256M tokens per sequence, and the units (of 32 tokens, or of 64 as often as there are passes) of a launch's sequences,
  // and of a sequence's kv heads, in 31 bits
  if (max_ctx > (1 << 28) || max(hkv, min(batch, kMaxBatch)) * (max_ctx / 32 + 1) * max(1, (passes + 1) / 2) > INT32_MAX)
    return false;
  // rows move by 16-byte LDS-DMA at 32-bit offsets within a page
  if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc) & 15 || (q_st | q_sh | ps | ts | hs) & 7) return false;
  if (ts < kD || ts > (1 << 26) || ps < 0 || ps > UINT32_MAX || hs < 0 || bt_stride < max_blocks || min(batch, kMaxBatch) * bt_stride * 4 > INT32_MAX)
    return false;
  if ((uintptr_t)out & 3 || out_st & 1) return false;
  a.q_st = q_st; a.q_sh = q_sh;
  a.kc = (const bf16_t*)kc; a.vc = (const bf16_t*)vc; a.ps = ps; a.ts = ts; a.hs = hs;
  a.bt_stride = bt_stride; a.out_st = out_st;
  a.hq = hq; a.hkv = hkv;
  a.glog = __builtin_ctz(hq / hkv);
  a.nsub = block_size / kPage;
  a.max_ctx = (int)max_ctx;
  a.scale_log2 = scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f;
  a.q_keep = scale == 0.f ? 0u : ~0u;
  a.q_flip = scale < 0.f ? 0x80008000u : 0u;
  return true;
}

}  // namespace

extern "C" size_t xv_tree_attention_workspace_size(int batch, int max_nodes, int num_q_heads, int num_kv_heads) {
  if (batch <= 0 || max_nodes <= 0 || !valid_group(num_q_heads, num_kv_heads)) return 256;
  const int max_rows = max_nodes * (num_q_heads / num_kv_heads);
  const bool tiles = max_rows > 16;  // of either kernel, so that a smaller batch never needs more
  return seg_bytes(batch, num_kv_heads, max_rows) + lse_bytes(max_rows, tiles) + slots(tiles) * slot_rows(max_rows, tiles) * kD * sizeof(float);
}

extern "C" int xv_window_decode_attention(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
                                          const void* v_cache, int64_t page_stride, int64_t tok_stride, int64_t head_stride,
                                          const int32_t* block_tables, int64_t bt_stride, const int32_t* cache_seqlens,
                                          void* out, int64_t out_stride_tok, void* workspace, size_t workspace_bytes, int batch,
                                          int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                                          int max_blocks_per_seq, int window, int sink_tokens, float scale,
                                          hipStream_t stream) {
  RowsArgs a{};
  if (window < 1 || sink_tokens < 0 ||
      !rows_args(a, q, q_stride_tok, q_stride_head, k_cache, v_cache, page_stride, tok_stride, head_stride, bt_stride, out,
                 out_stride_tok, batch, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq, 1, scale))
    return (int)hipErrorInvalidValue;
  if (batch == 0) return 0;
  if (workspace == nullptr || (uintptr_t)workspace & 15 ||
      workspace_bytes < xv_tree_attention_workspace_size(batch, 1, num_q_heads, num_kv_heads))
    return (int)hipErrorInvalidValue;
  a.window = window;
  a.sinks = sink_tokens;
  return launch_rows<false>(a, (const bf16_t*)q, block_tables, cache_seqlens, nullptr, (bf16_t*)out, batch, 1, workspace, stream);
}

extern "C" int xv_tree_attention(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache,
                                 const void* v_cache, int64_t page_stride, int64_t tok_stride, int64_t head_stride,
                                 const int32_t* block_tables, int64_t bt_stride, const int32_t* cache_seqlens,
                                 const int32_t* cu_seqlens_q, const int64_t* tree_mask, int64_t mask_stride, int mask_words,
                                 void* out, int64_t out_stride_tok, void* workspace, size_t workspace_bytes, int batch,
                                 int max_nodes, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                                 int max_blocks_per_seq, float scale, hipStream_t stream) {
  RowsArgs a{};
  if (max_nodes < 0 || max_nodes > 1024 || mask_words < 1 || max_nodes > 64 * (int64_t)mask_words || mask_stride < mask_words ||
      !rows_args(a, q, q_stride_tok, q_stride_head, k_cache, v_cache, page_stride, tok_stride, head_stride, bt_stride, out,
                 out_stride_tok, batch, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                 valid_group(num_q_heads, num_kv_heads) ? row_passes(max_nodes * (num_q_heads / num_kv_heads)) : 1, scale))
    return (int)hipErrorInvalidValue;
  if (batch == 0 || max_nodes == 0) return 0;
  if (workspace == nullptr || (uintptr_t)workspace & 15 ||
      workspace_bytes < xv_tree_attention_workspace_size(batch, max_nodes, num_q_heads, num_kv_heads))
    return (int)hipErrorInvalidValue;
  a.mask = (const uint64_t*)tree_mask; a.mask_st = mask_stride; a.words = mask_words;
  return launch_rows<true>(a, (const bf16_t*)q, block_tables, cache_seqlens, cu_seqlens_q, (bf16_t*)out, batch, max_nodes,
                           workspace, stream);
}
