// Attention of trees of drafted tokens with more than 32 rows (nodes times query
// heads per kv head), or few trees with more than 16, over the paged cache, for
// gfx950.
//
// The work split, partials and merge are those of xv_rows.h with 64-key tiles
// as units and a workgroup per range: its waves take 32 rows each of the same
// (sequence, kv head), so a K / V tile that is staged in LDS once serves up
// to 256 rows (further ones are further passes over the tiles).
// Per tile and wave, on v_mfma_f32_32x32x16_bf16 as in prefill attention:
// S^T = K Q^T, the softmax of a row in its lane pair, O^T += V^T P^T with P
// straight from the scores' registers.  Tiles travel by LDS-DMA into a ring of
// kRing slots, one barrier per tile.
//
// Measured (a call with its merge): 32 trees of 5 to 64 nodes over up to 4096
// tokens, 32 / 8 heads, 317 MB and 37 GFLOP, 113 us (2.8 TB/s, 327 TFLOP/s); 4 of
// 40 to 90 over up to 90000, 16 / 8 heads, 1013 MB and 128 GFLOP, 257 us (3.9 TB/s,
// 500 TFLOP/s).  Under a profiler the kernel alone takes 111 and 321 us (medians;
// 109 and 249 at best).  Neither stream nor products alone bound it: without the
// products it takes two thirds of that, without the loads three quarters.  Of 3900 to 4700
// cycles a tile the first wave computes 2200 (the 32 products are 1056; the softmax
// between them waits for one and is waited for by the other), stands 580 at its
// LDS-DMA (all waves issue theirs behind the barrier), spends 350 on where the next
// tile is and 500 to 800 on the barrier and on data; a segment's ends take 6500.
// Above 128 rows some SIMDs have two waves of rows, and the others wait for them.
// Scores a tile ahead of the softmax, loads issued later or by four of the waves,
// two tiles a barrier, halves of a tile or a tile each on two waves where half of
// them have no rows: 0 to 10 % slower in all.
//
// Workgroups of four waves and a ring of two, two a CU, for up to 128 rows:
// slower on most (32 trees of 32 nodes over 2000 tokens 77 against 63 us, 16 of
// 24 over 8000 124 against 109, one of 32 over 4000 30 against 24), faster where
// segments are many and short (128 of 20 over 1000 118 against 131).
#include "xv_kernels.h"
#include "xv_rows.h"
#include "xv_tile.h"
#include <math.h>

using namespace xv_rows;

namespace {

constexpr int kWaves = 8;
constexpr int kRing = 4;                // tiles in LDS: 128 KB, a workgroup a CU
constexpr int kRows = kKeys / kWaves;   // rows of a tile that a wave loads
constexpr int kOps = 2 * (kRows / 4);   // LDS-DMA instructions it takes for K and V
static_assert(32 * kWaves == kPassRows);

const xv_bf16x2 kOnes = {(__bf16)1.0f, (__bf16)1.0f};
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

struct TileState {
  float m, l;        // this lane's row: the maximum in use (log2 domain), the sum over this lane's keys
  floatx16_t o[4];   // O^T: row l % 32, d = 32n + 8j + 4(l / 32) + r in o[n][4j + r]
};

XV_INLINE void reset(TileState& st) {
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) st.o[n][r] = 0.f;
}

// Four K A-operands (d-steps 4 half .. + 3) of key tile MT, and the wait for all but the newest N LDS reads before they
// are used.
template <int MT>
XV_INLINE void read_k4(bf16x8_t (&kf)[4], const uint32_t (&at)[8], int half) {
  __asm__ __volatile__(
      "ds_read_b128 %0, %4 offset:%8\n\t"
      "ds_read_b128 %1, %5 offset:%8\n\t"
      "ds_read_b128 %2, %6 offset:%8\n\t"
      "ds_read_b128 %3, %7 offset:%8"
      : "=&v"(kf[0]), "=&v"(kf[1]), "=&v"(kf[2]), "=&v"(kf[3])
      : "v"(at[4 * half]), "v"(at[4 * half + 1]), "v"(at[4 * half + 2]), "v"(at[4 * half + 3]), "n"(MT * 32 * 256)
      : "memory");
}
template <int N>
XV_INLINE void wait_k4(bf16x8_t (&kf)[4]) {
  __asm__ __volatile__("s_waitcnt lgkmcnt(%4)" : "+v"(kf[0]), "+v"(kf[1]), "+v"(kf[2]), "+v"(kf[3]) : "n"(N) : "memory");
}

// S^T of one tile.  Its K operands come four at a time, the next four in flight behind the products of the last ones:
// all sixteen at once would take 64 registers and spill.
XV_INLINE void s_tile(floatx16_t (&s)[2], const bf16x8_t (&qb)[8], const LdsAddr& ad) {
  bf16x8_t k0[4], k1[4], k2[4], k3[4];
#pragma unroll
  for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
  auto product = [&](floatx16_t& d, const bf16x8_t (&k)[4], int half) {
#pragma unroll
    for (int u = 0; u < 4; ++u) d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k[u], qb[4 * half + u], d, 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);  // what follows stays behind these products
  };
  read_k4<0>(k0, ad.k, 0);
  read_k4<0>(k1, ad.k, 1);
  wait_k4<4>(k0);
  product(s[0], k0, 0);
  read_k4<1>(k2, ad.k, 0);
  wait_k4<4>(k1);
  product(s[0], k1, 1);
  read_k4<1>(k3, ad.k, 1);
  wait_k4<4>(k2);
  product(s[1], k2, 0);
  wait_k4<0>(k3);
  product(s[1], k3, 1);
}

// Scores of the keys that the lane's row does not see (bit k of `seen` clear): -inf.
XV_INLINE void mask_tile(floatx16_t (&s)[2], uint64_t seen, int h) {
  // s[mt][r] is key 32 mt + 8 (r / 4) + 4 h + r % 4
  const uint32_t bits[2] = {(uint32_t)seen >> (4 * h), (uint32_t)(seen >> 32) >> (4 * h)};
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[mt][r] = (bits[mt] >> (8 * (r >> 2) + (r & 3))) & 1 ? s[mt][r] : -INFINITY;
}

// Online softmax of a tile's scores: P (bf16), O and l rescaled as needed.
XV_INLINE void softmax_tile(TileState& st, const floatx16_t (&s)[2], bf16x8_t (&pb)[2][2], float scale_log2) {
  float mx = -INFINITY;
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[mt][r]);
  mx = xor32_max(mx) * scale_log2;
  // the maximum in use moves only when the row's grew by more than kLazy
  if (mx > st.m + kLazy) {
    const float alpha = __builtin_amdgcn_exp2f(st.m - mx);  // 0 on the first tile
    st.m = mx;
    st.l *= alpha;
#pragma unroll
    for (int n = 0; n < 4; ++n) st.o[n] *= alpha;
  }
  const float nm = st.m == -INFINITY ? 0.f : -st.m;  // a row that has seen nothing yet: p = 0
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 8 * kk + 2 * e;
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][r], scale_log2, nm));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][r + 1], scale_log2, nm));
        w[e] = pack_bf16x2(p0, p1);
        // the row sum takes the bf16 weights that the product multiplies: their rounding (2^-8 of a weight at most) moves
        // the output by that share of the values' spread only
        st.l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(xv_bf16x2, w[e]), kOnes, st.l, false);
      }
      __builtin_memcpy(&pb[mt][kk], w, 16);
    }
}

// O^T += V^T P^T.
XV_INLINE void pv_tile(TileState& st, const bf16x8_t (&pb)[2][2], const LdsAddr& ad) {
#pragma unroll
  for (int k2 = 0; k2 < 2; ++k2) {  // key-steps 2 k2, 2 k2 + 1
    short4_t vt[16];
    if (k2 == 0) read_vt_ks2<0, 0>(vt, ad); else read_vt_ks2<0, 2>(vt, ad);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int n = 0; n < 2; ++n)
        st.o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt_operand(vt, n, j), pb[k2][j], st.o[n], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    vt_wait_rest(vt);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int n = 2; n < 4; ++n)
        st.o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt_operand(vt, n, j), pb[k2][j], st.o[n], 0, 0, 0);
  }
}

// The OR of x over the wave.
XV_INLINE uint64_t wave_or(uint64_t x) {
  uint32_t w[2] = {(uint32_t)x, (uint32_t)(x >> 32)};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    w[k] |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[k], 0x128, 0xf, 0xf, false);
    w[k] |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[k], 0x124, 0xf, 0xf, false);
    w[k] |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[k], 0x4E, 0xf, 0xf, false);
    w[k] |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[k], 0xB1, 0xf, 0xf, false);
    auto r = __builtin_amdgcn_permlane16_swap(w[k], w[k], false, false);
    w[k] = r[0] | r[1];
    r = __builtin_amdgcn_permlane32_swap(w[k], w[k], false, false);
    w[k] = r[0] | r[1];
  }
  return (uint64_t)w[1] << 32 | w[0];
}

// The finished segment's row of this lane: bf16 output (slot < 0), else a partial's fp32 row.
XV_INLINE void finish_row(const RowsArgs& a, const TileState& st, int tok0, int kvh, int row, int nrows, int slot, int h) {
  typedef u32x2_t __attribute__((aligned(4))) u32x2_a4;  // the caller's rows need not be 8-byte aligned
  const float lsum = xor32_sum(st.l);
  const float inv = lsum == 0.f ? 0.f : 1.0f / lsum;  // a row that sees nothing: zeros; NaN stays NaN
  if (row >= nrows) return;
  if (slot < 0) {
    const int node = row >> a.glog, head = (kvh << a.glog) + (row & ((1 << a.glog) - 1));
    bf16_t* dst = a.out + (int64_t)(tok0 + node) * a.out_st + (int64_t)head * kD + 4 * h;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<u32x2_a4*>(dst + 32 * n + 8 * j) =
            u32x2_t{pack_bf16x2(st.o[n][4 * j] * inv, st.o[n][4 * j + 1] * inv),
                    pack_bf16x2(st.o[n][4 * j + 2] * inv, st.o[n][4 * j + 3] * inv)};
  } else {
    const int64_t at = (int64_t)slot * a.rows + row;
    float* dst = a.ws_o + at * kD + 4 * h;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<floatx4_t*>(dst + 32 * n + 8 * j) =
            floatx4_t{st.o[n][4 * j], st.o[n][4 * j + 1], st.o[n][4 * j + 2], st.o[n][4 * j + 3]} * inv;
    if (h == 0) a.ws_lse[at] = lsum == 0.f ? -INFINITY : st.m + __log2f(lsum);
  }
}

// A workgroup barrier behind this wave's LDS accesses.  (A plain __syncthreads also waits for every tile in flight.)
XV_INLINE void barrier() {
  __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __asm__ __volatile__("" ::: "memory");
}

__global__ __launch_bounds__(kWaves * 64, 2) void tree_tile_kernel(RowsArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[kRing * kBuf];
  __shared__ Sequences seqs;
  __shared__ uint64_t any[kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  if (wave == 0) load_sequences<true, true>(seqs, a, lane, [](int ctx) { return (ctx + kKeys - 1) / kKeys; });
  __syncthreads();
  const Ranges rg = ranges_of<true>(seqs, a, gridDim.x, lane);
  const int id = blockIdx.x;
  const int64_t f0 = (int64_t)id * rg.len;
  const int n = (int)max((int64_t)0, min(f0 + rg.len, rg.total) - f0);
  if (n == 0) return;
  const int row0 = wave * 32, row = row0 + l32;  // this lane's row of every segment
  const LdsAddr ad = lds_addr(lds, lane);

  // ---- The tiles' feed.  This wave loads rows r0 .. r0 + kRows - 1 of a tile, all in one cache block: row `r` on of block
  // `blk`, of which `valid` (and more behind them) are in the sequence; rows past its end read as zeros, and so does every
  // row past the range, so that an iteration issues the same number of loads wherever it is.
  const int r0 = kRows * wave;
  const int block = a.nsub * kPage;
  const int step_blocks = kKeys / block, step_rows = kKeys % block;
  Cursor ic = cursor_at<true>(seqs, a, f0);
  int issued = 0, idx = 0, r = 0, valid = 0, blk = 0;
  const int32_t* table = a.bt;
  auto fetch = [&] { blk = valid > 0 ? load_index(table + idx) : 0; };
  auto enter = [&] {  // at ic, wherever that is in its segment
    const int j = ic.u * kKeys + r0;
    idx = j / block;
    r = j - idx * block;
    valid = ic.ctx - j;
    table = a.bt + (int64_t)ic.b * a.bt_stride;
  };
  auto issue = [&] {
    const int64_t off = (int64_t)((uint64_t)(uint32_t)blk * (uint32_t)a.ps) + (int64_t)((uint64_t)(uint32_t)r * (uint32_t)a.ts) +
                        (int64_t)ic.kvh * a.hs;
    const uint32_t bytes = valid > 0 ? (uint32_t)(((min(valid, kRows) - 1) * (int)a.ts + kD) * 2) : 0u;
    const __amdgpu_buffer_rsrc_t rk = page_rsrc(a.kc + off, bytes), rv = page_rsrc(a.vc + off, bytes);
    char* const buf = lds + (issued % kRing) * kBuf + r0 * 256;
#pragma unroll
    for (int s = 0; s < kRows / 4; ++s) {
      const int rr = 4 * s + (lane >> 4), R = r0 + rr;
      const int vo = (int)(rr * a.ts * 2);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(buf + 1024 * s), 16, vo + (((lane & 15) ^ swz_k(R)) << 4), 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(buf + kTile + 1024 * s), 16,
                                               vo + (((lane & 15) ^ swz_v(R)) << 4), 0, 0, 0);
    }
    if (++issued >= n) {
      valid = 0;
    } else if (++ic.u < ic.nu) {
      idx += step_blocks;
      r += step_rows;
      if (r >= block) {
        r -= block;
        ++idx;
      }
      valid -= kKeys;
    } else {
      --ic.u;
      advance<true>(ic, seqs, a);
      enter();
    }
    fetch();
  };
  enter();
  fetch();

  // ---- Segments: the first row of q, the rows (all from the pass's first on), and this lane's q
  Cursor pc = ic;  // tile x
  auto rows_in = [&](const Cursor& c, int& tok, int& rows) {
    tok = lds_int(seqs.cq + c.b) + c.pass * (kPassRows >> a.glog);
    rows = (lds_int(seqs.cq + c.b + 1) - tok) << a.glog;
  };
  Vec8 raw[8];
  auto load_q = [&](int kvh, int tok, int rows) {
    const int q = min(row, rows - 1);
    const bf16_t* src = a.q + (int64_t)(tok + (q >> a.glog)) * a.q_st +
                        (int64_t)((kvh << a.glog) + (q & ((1 << a.glog) - 1))) * a.q_sh + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) raw[s] = load_vec8(src + 16 * s);
  };
  bf16x8_t qb[8];
  auto take_q = [&] {
#pragma unroll
    for (int s = 0; s < 8; ++s) {
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[s].w[e] = (raw[s].w[e] & a.q_keep) ^ a.q_flip;
      __builtin_memcpy(&qb[s], &raw[s], 16);
    }
  };
  // ---- Masks: a tile's first key as a node of its tree; where that is above -kKeys some row may not see every key.
  // This lane's words are loaded an iteration ahead.
  auto node_of = [&](const Cursor& c, int rows) { return c.u * kKeys - c.ctx + ((rows + c.pass * kPassRows) >> a.glog); };
  uint64_t w0 = 0, w1 = 0;
  auto load_words = [&](int tok, int rows, int at) {
    const uint64_t* m = a.mask + (int64_t)(tok + (min(row, rows - 1) >> a.glog)) * a.mask_st;
    const int w = max(at, 0) >> 6;
    w0 = w < a.words ? m[w] : 0;
    w1 = at > 0 && (at & 63) && w + 1 < a.words ? m[w + 1] : 0;
  };
  int tok, nrows;
  rows_in(pc, tok, nrows);
  int at = node_of(pc, nrows);
  if (row0 < nrows) {
    load_q(pc.kvh, tok, nrows);
    if (at > -kKeys) load_words(tok, nrows, at);
  }
#pragma unroll
  for (int k = 0; k < kRing - 1; ++k) issue();
  if (row0 < nrows) take_q();
  TileState st;
  reset(st);
  for (int x = 0; x < n; ++x) {
    __asm__ __volatile__("s_waitcnt vmcnt(%0)" ::"n"((kRing - 2) * kOps) : "memory");
    barrier();  // tile x is in LDS; every wave is done with tile x - 1
    const uint64_t c0 = w0, c1 = w1;
    Cursor nc = pc;
    int tok1 = tok, nrows1 = nrows;
    const bool last = x + 1 == n, turn = pc.u + 1 == pc.nu || last;  // tile x ends its segment, or the range
    if (!last) {
      advance<true>(nc, seqs, a);
      if (turn) rows_in(nc, tok1, nrows1);
    }
    const int at1 = node_of(nc, nrows1);
    if (row0 < nrows1) {  // ahead of the tiles: waiting for these does not wait for those
      if (turn) load_q(nc.kvh, tok1, nrows1);
      if (at1 > -kKeys) load_words(tok1, nrows1, at1);
    }
    issue();
    const uint32_t slot = (uint32_t)(x % kRing) * kBuf;
    uint64_t seen = 0;  // keys of the tile that this lane's row sees
    const bool edge = at > -kKeys;
    if (edge) {
      const int sh = at & 63;
      if (row0 < nrows)
        seen = low_bits64(pc.ctx - pc.u * kKeys) & (at < 0 ? c0 << -at | low_bits64(-at) : sh ? c0 >> sh | c1 << (64 - sh) : c0);
      // V of keys that no row sees may be anything, NaN included: zeros in its place
      const uint64_t mine = wave_or(seen);
      if (lane == 0) any[wave] = mine;
      barrier();
      uint64_t all = 0;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) all |= any[k];
#pragma unroll
      for (int s = 0; s < kRows / 4; ++s) {
        const int R = r0 + 4 * s + (lane >> 4);
        if (!(all >> R & 1)) *reinterpret_cast<uint4*>(lds + slot + kTile + R * 256 + (lane & 15) * 16) = make_uint4(0, 0, 0, 0);
      }
      barrier();
    }
    if (row0 < nrows) {
      LdsAddr cur;
#pragma unroll
      for (int k = 0; k < 8; ++k) cur.k[k] = ad.k[k] + slot;
#pragma unroll
      for (int k = 0; k < 4; ++k) cur.v[k] = ad.v[k] + slot;
      floatx16_t s[2];
      bf16x8_t pb[2][2];
      s_tile(s, qb, cur);
      if (edge) mask_tile(s, seen, h);
      softmax_tile(st, s, pb, a.scale_log2);
      pv_tile(st, pb, cur);
    }
    if (turn) {
      finish_row(a, st, tok, pc.kvh, row, nrows, finish_slot(seqs, a, pc, f0, n, id, rg.len, row == 0 && h == 0), h);
      reset(st);
      tok = tok1;
      nrows = nrows1;
      if (row0 < nrows) take_q();
    }
    pc = nc;
    at = at1;
  }
  __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");  // nothing is on its way to LDS behind the wave's end
}

}  // namespace

int xv_rows::launch_tiles(const RowsArgs& a, hipStream_t stream) {
  tree_tile_kernel<<<kTileGroups, kWaves * 64, 0, stream>>>(a);
  return (int)hipGetLastError();
}
