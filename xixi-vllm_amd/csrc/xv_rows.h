// What the kernels of paged attention over a few rows per sequence share: their
// arguments, and the flat (sequence, kv head, unit) space that is cut into
// ranges; a sequence of many rows is in it once per pass over up to 256 of them.  A range's segments that it does not hold whole leave partials:
// normalised fp32 rows and their log2-sum-exp, slot 2 * range for one that
// started before the range, 2 * range + 1 for one that ends after it.
#pragma once
#include "xv_decode.h"

namespace xv_rows {

constexpr int kPage = 16;
constexpr int kMaxBatch = 256;   // sequences per launch (larger batches are launched in chunks)
constexpr int kMaxParts = 192;   // partials of a segment at most

struct RowsArgs {
  const bf16_t* q; int64_t q_st, q_sh;
  const bf16_t* kc; const bf16_t* vc; int64_t ps, ts, hs;
  const int32_t* bt; int64_t bt_stride;
  const int32_t* seqlens;
  const int32_t* cu_q;                          // tree: first node of each sequence
  const uint64_t* mask; int64_t mask_st; int words;  // tree: visible nodes of each node
  bf16_t* out; int64_t out_st;
  int2* ws_seg;     // (first range, partials) per segment: seg_index
  float* ws_lse;    // log2-sum-exp of partial slot s, row r at s * rows + r
  float* ws_o;      // its rows, 128 values each
  int batch, hq, hkv, glog;  // query heads per kv head: 1 << glog
  int nsub;         // 16-token pages per cache block
  int max_ctx;      // tokens the block table has room for
  int window, sinks;
  int rows;         // rows of a partial slot
  int max_nodes;    // of a sequence; further ones are not looked at
  int passes;       // of a sequence, at most
  // scale * log2(e); q is taken as (q & q_keep) ^ q_flip, so that the scale is positive: the sign of a negative
  // one goes to q, and a scale of 0 is 1 over a q of zeros
  float scale_log2;
  uint32_t q_keep, q_flip;
};

// Passes are segments of the flat space: equal ranges over them balance a large tree among small ones (one of 1024 nodes
// among 31 of 20: 178 us, 1065 with the same number of workgroups for every pass).
constexpr int kPassRows = 256;
XV_INLINE int seg_index(const RowsArgs& a, int b, int pass, int kvh) { return (b * a.passes + pass) * a.hkv + kvh; }

// Sequences of a launch, in LDS.
struct Sequences {
  int pref[kMaxBatch + 1];  // units of sequences 0 .. b - 1, all their passes
  int ctx[kMaxBatch];       // their tokens (0: no rows)
  int cq[kMaxBatch + 1];    // their first rows of q
};

// LDS reads in asm: before a plain one the compiler waits for every LDS-DMA load in flight.
XV_INLINE int lds_int(const int* p) {
  int v;
  __asm__ __volatile__("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                       : "=&v"(v)
                       : "v"((uint32_t)reinterpret_cast<uintptr_t>(p))
                       : "memory");
  return __builtin_amdgcn_readfirstlane(v);
}

// Passes over n nodes, at least one.
template <bool PASSES>
XV_INLINE int passes_of(const RowsArgs& a, int n) {
  return PASSES ? max(1, min(a.passes, (int)((((int64_t)n << a.glog) + kPassRows - 1) / kPassRows))) : 1;
}

// Fills `s` by one wave; units(ctx) > 0 for ctx > 0.
template <bool TREE, bool PASSES, typename F>
XV_INLINE void load_sequences(Sequences& s, const RowsArgs& a, int lane, F units) {
  int carry = 0;
  for (int c = 0; c < a.batch; c += 64) {
    const int b = c + lane;
    int ctx = 0, q0 = b, q1 = b + 1;
    if (b < a.batch) {
      ctx = min(max(a.seqlens[b], 0), a.max_ctx);
      if (TREE) {
        q0 = a.cu_q[b];
        q1 = a.cu_q[b + 1];
        if (q1 <= q0) ctx = 0;  // no rows: no units
      }
    }
    int inc = ctx > 0 ? units(ctx) * passes_of<PASSES>(a, q1 - q0) : 0;
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x111, 0xf, 0xf, true);  // inclusive scan: row_shr 1, 2, 4, 8,
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x112, 0xf, 0xf, true);  // then the row sums across rows
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x114, 0xf, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x118, 0xf, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x142, 0xa, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x143, 0xc, 0xf, true);
    if (b < a.batch) {
      s.pref[b + 1] = carry + inc;
      s.ctx[b] = ctx;
      s.cq[b] = q0;
      s.cq[b + 1] = q1;  // the next lane writes the same value
    }
    carry += __builtin_amdgcn_readlane(inc, 63);
  }
  if (lane == 0) s.pref[0] = 0;
}

// Units of the flat space, and units per range: every range the same, and no
// segment in more than kMaxParts ranges.
struct Ranges {
  int64_t total;
  int len;
};
template <bool PASSES>
XV_INLINE Ranges ranges_of(const Sequences& s, const RowsArgs& a, int nranges, int lane) {
  int longest = 0;
  for (int b = lane; b < a.batch; b += 64) {
    const int nu = s.pref[b + 1] - s.pref[b];
    longest = max(longest, a.passes > 1 ? nu / passes_of<PASSES>(a, s.cq[b + 1] - s.cq[b]) : nu);
  }
  const int max_nu = __builtin_amdgcn_readfirstlane((int)wave_max((float)longest));  // exact in fp32 (below 2^24)
  Ranges r;
  r.total = (int64_t)a.hkv * __builtin_amdgcn_readfirstlane(s.pref[a.batch]);  // wave uniform, as all of this
  r.len = (int)max((int64_t)max(1, (max_nu + kMaxParts - 2) / (kMaxParts - 1)), (r.total + nranges - 1) / nranges);
  return r;
}

// A position in the flat space.
struct Cursor {
  int b, pass, kvh, u;  // sequence, pass over its rows, kv head, unit within the sequence
  int np, nu, ctx;      // passes, units of one and tokens of sequence b
};
template <bool PASSES>
XV_INLINE Cursor cursor_at(const Sequences& s, const RowsArgs& a, int64_t f) {
  Cursor c;
  c.b = __builtin_amdgcn_readfirstlane(seq_of(s.pref, a.batch, a.hkv, f));
  c.np = __builtin_amdgcn_readfirstlane(passes_of<PASSES>(a, s.cq[c.b + 1] - s.cq[c.b]));
  c.nu = __builtin_amdgcn_readfirstlane(s.pref[c.b + 1] - s.pref[c.b]);
  if (c.np > 1) c.nu /= c.np;
  c.ctx = __builtin_amdgcn_readfirstlane(s.ctx[c.b]);
  const int r = (int)(f - (int64_t)a.hkv * s.pref[c.b]);
  const int seg = __builtin_amdgcn_readfirstlane(r / c.nu);
  c.u = __builtin_amdgcn_readfirstlane(r - seg * c.nu);
  c.pass = PASSES && c.np > 1 ? seg / a.hkv : 0;
  c.kvh = seg - c.pass * a.hkv;
  return c;
}
// The next one.  Sequences without units are stepped over.
template <bool PASSES>
XV_INLINE void advance(Cursor& c, const Sequences& s, const RowsArgs& a) {
  if (++c.u < c.nu) return;
  c.u = 0;
  if (++c.kvh < a.hkv) return;
  c.kvh = 0;
  if (PASSES && ++c.pass < c.np) return;
  c.pass = 0;
  do {
    ++c.b;
    c.nu = lds_int(s.pref + c.b + 1) - lds_int(s.pref + c.b);
  } while (c.nu == 0 && c.b < a.batch - 1);
  if (PASSES) {
    c.np = passes_of<PASSES>(a, lds_int(s.cq + c.b + 1) - lds_int(s.cq + c.b));
    if (c.np > 1) c.nu /= c.np;
  }
  c.ctx = lds_int(s.ctx + c.b);
}

// Where the rows of the segment at c go, in the range of n units from f0 on:
// -1 the output (the range holds all of it), else a partial slot.  `record`:
// this caller also writes the segment's (first range, partials).
XV_INLINE int finish_slot(const Sequences& s, const RowsArgs& a, const Cursor& c, int64_t f0, int n, int id, int len, bool record) {
  const int64_t seg0 = (int64_t)a.hkv * lds_int(s.pref + c.b) + (int64_t)(c.pass * a.hkv + c.kvh) * c.nu;
  const bool first = seg0 >= f0, last = seg0 + c.nu <= f0 + n;
  if (last && record) {
    const int w0 = (int)(seg0 / len);
    a.ws_seg[seg_index(a, c.b, c.pass, c.kvh)] = make_int2(w0, id - w0 + 1);
  }
  return first && last ? -1 : 2 * id + (first ? 1 : 0);
}

// The lowest n bits (none below 0, all from 32 or 64 on).
XV_INLINE uint32_t low_bits(int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; }
XV_INLINE uint64_t low_bits64(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull; }

// Trees of more than 32 rows, and few of more than 16: tree_tiles.hip.  a: all but the workspace's slots, filled for `batch` sequences.
constexpr int kTileGroups = 256;   // ranges: as many as there are workgroups resident at once
int launch_tiles(const RowsArgs& a, hipStream_t stream);

}  // namespace xv_rows
