// Varlen causal prefill attention (chunked prefill / cached prefix) for gfx950.
//
// Workgroup = 4 waves over one (sequence, query block, kv head): the waves
// serve min(G, 4) query heads of the kv group x 32 queries each, so every
// 64-key K/V tile staged in LDS is shared by all of them.  Per tile and wave
// (32 queries x 64 keys), all on v_mfma_f32_32x32x16_bf16:
//   S^T = K Q^T      2 key tiles x 8 d-steps; A = K rows from LDS
//                    (ds_read_b128), B = Q^T held in VGPRs.  Lane l holds query
//                    l%32 and keys 8j + 4(l/32) + r of each 32-key tile, so the
//                    online softmax is in-lane plus one cross-half exchange.
//   O^T += V^T P^T   4 d-tiles x 4 key-steps; A = V^T read transposed from LDS
//                    (ds_read_b64_tr_b16), B = P^T straight from the S^T
//                    registers: each key-step takes the lane's 8 consecutive
//                    accumulators, and V^T is read in the same key order.
// K and V tiles travel HBM -> LDS by LDS-DMA (buffer_load ... lds), whole
// 256-byte rows, into swizzled images (16-byte chunk c of row r at slot
// c ^ swz(r)) that keep the K and V^T reads free of bank conflicts on the
// 64-bank LDS.  The softmax runs in the exp2 domain with the scale folded
// into one FMA, masks only on tiles that cross the diagonal and rescales O
// lazily (only when a query's running max grew by more than 2^8).  Tiles
// are double buffered: the next tile's loads are in flight while the current
// one is computed; one barrier per tile.  Causal masking is bottom-right
// aligned (query i of q_len sees keys j <= k_len - q_len + i) and applied only
// on tiles that cross a wave's diagonal; tiles past it are skipped.  Rows past
// k_len read as zeros (bounded buffer resources), so unused cache slots never
// reach P.V.
//
// With a window and sinks a workgroup's tiles are four sixteens of keys each, the
// sinks', then those from its first query's window on; tiles at either edge are
// masked, and a wave passes over those that none of its queries sees.  Bound by the
// softmax beside the products, as without a window (products busy 52 % of the time,
// vector work 44 %): one document of 16001 with a window of 4096, 16 / 8 heads, 474
// GFLOP, 516 us a call (919 TFLOP/s); 16 chunks of up to 512 over up to 12000
// cached tokens, window 2000, 64 / 8 heads, 379 GFLOP, 471 us (803); 12 prompts of
// 40 to 2500, window 512, 32 / 8 heads, 97 GFLOP, 165 us (589: seven tiles a
// workgroup, a third of whose time is start and end).  Under a profiler the kernels
// alone take 580, 545 and 194 us (medians; 527, 490 and 172 at best).
#include "xv_common.h"
#include "xv_kernels.h"
#include "xv_tile.h"
#include <math.h>
#include <type_traits>

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr float kLazy = 8.0f;
const xv_bf16x2 kOnes = {(__bf16)1.0f, (__bf16)1.0f};

typedef __attribute__((address_space(3))) void lds_void;

struct PrefillArgs {
  const bf16_t* q; int64_t q_st, q_sh;
  const bf16_t* k; const bf16_t* v; int64_t kv_st, kv_sh;
  const bf16_t* kc; const bf16_t* vc; int64_t page_stride, tok_stride, head_stride;
  const int32_t* bt; int64_t bt_stride; int block_size;
  const int32_t* cu_q; const int32_t* cu_k;
  bf16_t* out; int64_t out_st;
  int hq, hkv, qblocks, batch;
  float scale_log2;
  int window, sinks;  // windowed calls only: tokens a query sees up to itself, first tokens that stay visible
};

XV_INLINE __amdgpu_buffer_rsrc_t rsrc(const bf16_t* base, uint32_t bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
  void* q = reinterpret_cast<void*>(((uint64_t)hi << 32) | lo);
  return __builtin_amdgcn_make_buffer_rsrc(q, (short)0, (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// A wave's 16 keys of a tile in the cache: block id, first row in it.
struct Page {
  int block;
  int row;
};

// Wave w moves the 16 keys from j0 on (one cache page when paged), rows 16w .. +15
// of the tile: 4 LDS-DMA instructions for K and/or 4 for V, each 4 whole rows.
// WIN: keys sinks .. lo - 1 are seen by no query of the workgroup: their V
// reads as zeros (whatever the cache holds there), and 16 keys that are all
// such are not read at all (their block-table entry may be gone).
template <bool PAGED, bool DO_K, bool DO_V, bool WIN>
XV_INLINE void load_rows(char* buf, const PrefillArgs& a, int b, int kvh, int j0, int k0, int k_len,
                         Page page, int lo, int wave, int lane) {
  const int valid = WIN && j0 >= a.sinks && j0 + 16 <= lo ? 0 : min(16, k_len - j0);
  const bf16_t *kb, *vb;
  int64_t rs;  // row stride (elements)
  if (PAGED) {
    const int64_t off = (int64_t)page.block * a.page_stride + (int64_t)page.row * a.tok_stride + (int64_t)kvh * a.head_stride;
    kb = a.kc + off; vb = a.vc + off; rs = a.tok_stride;
  } else {
    const int64_t off = (int64_t)(k0 + j0) * a.kv_st + (int64_t)kvh * a.kv_sh;
    kb = a.k + off; vb = a.v + off; rs = a.kv_st;
  }
  const uint32_t bytes = valid > 0 ? (uint32_t)(((int64_t)(valid - 1) * rs + kD) * 2) : 0u;
  const __amdgpu_buffer_rsrc_t rk = rsrc(kb, bytes), rv = rsrc(vb, bytes);
  const int slot = lane & 15;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int r = 4 * s + (lane >> 4);  // row within the wave's 16
    const int R = 16 * wave + r;        // row within the tile
    const int vo_k = (int)(r * rs * 2) + ((slot ^ swz_k(R)) << 4);
    int vo_v = (int)(r * rs * 2) + ((slot ^ swz_v(R)) << 4);
    if (WIN && j0 + r >= a.sinks && j0 + r < lo) vo_v = INT32_MIN;  // past every resource: zeros
    if (DO_K)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(buf + (16 * wave + 4 * s) * 256), 16, vo_k, 0, 0, 0);
    if (DO_V)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(buf + kTile + (16 * wave + 4 * s) * 256), 16, vo_v,
                                               0, 0, 0);
  }
}

// Sequence of dispatch slot j: sequences in descending causal work
// q_len * (k_len - q_len) + q_len * (q_len + 1) / 2 (ties: lower index
// first), so the costliest sequences' blocks are dispatched first and the
// cheapest ones finish the grid.  Each sequence's blocks stay together in the
// dispatch order (they share K/V tiles in L2).  Batches above 64 keep their
// own order.
struct Sequence {
  int b, q0, q_len, k0, k_len;
};
XV_INLINE Sequence seq_by_work(const int* cu_q, const int* cu_k, int batch, int j) {
  if (batch > 64) return Sequence{j, cu_q[j], cu_q[j + 1] - cu_q[j], cu_k[j], cu_k[j + 1] - cu_k[j]};
  const int lane = threadIdx.x & 63;
  int64_t w = -1;
  int q0 = 0, ql = 0, k0 = 0, kl = 0;
  if (lane < batch) {
    q0 = cu_q[lane];
    k0 = cu_k[lane];
    ql = cu_q[lane + 1] - q0;
    kl = cu_k[lane + 1] - k0;
    w = (int64_t)ql * (kl - ql) + (int64_t)ql * (ql + 1) / 2;
  }
  int pos = 0;
  for (int t = 0; t < batch; ++t) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)w, t);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)w >> 32), t);
    const int64_t wt = (int64_t)(((uint64_t)hi << 32) | lo);
    pos += (wt > w || (wt == w && t < lane)) ? 1 : 0;
  }
  const uint64_t m = __ballot(lane < batch && pos == j);
  const int b = __builtin_amdgcn_readfirstlane(__builtin_ctzll(m));
  // its lengths from the lane that has them: a second trip to memory costs every workgroup a microsecond
  return Sequence{b, __builtin_amdgcn_readlane(q0, b), __builtin_amdgcn_readlane(ql, b), __builtin_amdgcn_readlane(k0, b),
                  __builtin_amdgcn_readlane(kl, b)};
}

// Block `flat` of the sequences' blocks of BQ queries one after the other, in the
// order above: its sequence, and its rank in it (-1: there is none).  For a grid
// without the places of blocks that shorter sequences do not have.
struct Block {
  Sequence seq;
  int rank;
};
template <int BQ>
XV_INLINE Block block_by_work(const int* cu_q, const int* cu_k, int batch, int flat) {
  const int lane = threadIdx.x & 63;
  for (int c = 0; c < batch; c += 64) {
    const int i = c + lane;
    int q0 = 0, ql = 0, k0 = 0, kl = 0;
    if (i < batch) {
      q0 = cu_q[i];
      k0 = cu_k[i];
      ql = cu_q[i + 1] - q0;
      kl = cu_k[i + 1] - k0;
    }
    // the work to 17 bits, the lane behind it: no two are alike, and one comparison of 32 bits a sequence
    const int64_t w = (int64_t)ql * (kl - ql) + (int64_t)ql * (ql + 1) / 2;
    const uint32_t key = (__builtin_bit_cast(uint32_t, (float)max((int64_t)0, w)) & ~63u) | (63 - lane);
    const int blocks = max(0, (ql + BQ - 1) / BQ);
    int before = 0, all = 0;  // blocks of the sequences dispatched before this lane's, and of all 64
    const int n = min(64, batch - c);
#pragma unroll 4
    for (int t = 0; t < n; ++t) {
      const int bt = __builtin_amdgcn_readlane(blocks, t);
      before += (uint32_t)__builtin_amdgcn_readlane((int)key, t) > key ? bt : 0;
      all += bt;
    }
    const uint64_t m = __ballot(flat >= before && flat < before + blocks);
    if (m) {
      const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(m));
      return Block{Sequence{c + l, __builtin_amdgcn_readlane(q0, l), __builtin_amdgcn_readlane(ql, l),
                            __builtin_amdgcn_readlane(k0, l), __builtin_amdgcn_readlane(kl, l)},
                   flat - __builtin_amdgcn_readlane(before, l)};
    }
    flat -= all;
  }
  return Block{Sequence{0, 0, 0, 0, 0}, -1};
}

template <int G, bool PAGED, bool WIN>
__global__ __launch_bounds__(kThreads, 2) void prefill_kernel(PrefillArgs a) {
  constexpr int GW = G < 4 ? G : 4;   // query heads per workgroup
  constexpr int QS = 4 / GW;          // 32-query sub-blocks per workgroup
  constexpr int kBlockQ = 32 * QS;
  __shared__ __attribute__((aligned(16))) char lds[2 * kBuf];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: keeps per-wave values scalar
  const int l32 = lane & 31, h = lane >> 5;
  // XCD-aware order: workgroups go round-robin to the 8 XCDs, so with the head
  // slot fastest every XCD serves the same kv head(s) and keeps their K/V tiles
  // in its own L2; each head carries the same work, which balances the XCDs.
  const int hsel = blockIdx.x;
  const Block blk = WIN ? block_by_work<kBlockQ>(a.cu_q, a.cu_k, a.batch, (int)(blockIdx.z * gridDim.y + blockIdx.y))
                        : Block{seq_by_work(a.cu_q, a.cu_k, a.batch, blockIdx.z), (int)blockIdx.y};
  if (WIN && blk.rank < 0) return;
  const Sequence seq = blk.seq;
  const int rank = blk.rank;
  const int b = seq.b;
  // group 8: two slots per kv head (query heads 0-3 and 4-7), slot = half * Hkv
  // + kvh, so both halves of a kv head land on the same XCD
  const int kvh = G == 8 ? hsel % a.hkv : hsel;
  const int head = G == 8 ? kvh * 8 + (hsel / a.hkv) * 4 + wave : kvh * G + wave % GW;
  const int q0 = seq.q0, q_len = seq.q_len, k0 = seq.k0, k_len = seq.k_len;
  // rank from the sequence's own end: the last (longest) block of the causal
  // triangle is dispatched first, then the next-to-last, ...
  const int qb0 = ((q_len + kBlockQ - 1) / kBlockQ - 1 - rank) * kBlockQ;
  if (qb0 < 0) return;
  const int shift = k_len - q_len;  // bottom-right alignment
  const int qw0 = qb0 + (wave / GW) * 32;  // the wave's first query
  const int my_q = qw0 + l32;
  const int kv_end = min(k_len, shift + min(qb0 + kBlockQ, q_len));  // keys the block needs
  // The keys that the block needs, 16 at a time: all of them; WIN: the sinks', then those from its first query's window on.
  // Four sixteens are a tile.
  const int blk_lo = WIN ? max(0, shift + qb0 + 1 - a.window) : 0;
  const int sink_16 = WIN ? (min(a.sinks, blk_lo) + 15) / 16 : 0;
  const int skip = WIN ? max(0, blk_lo / 16 - sink_16) : 0;
  const int ntiles = WIN ? max(0, (kv_end + 15) / 16 - skip + 3) / 4 : max(0, (kv_end + kKeys - 1) / kKeys);
  auto key_of = [&](int t, int g) {  // first key of tile t's sixteen g
    const int i = 4 * t + g;
    return 16 * (WIN && i >= sink_16 ? i + skip : i);
  };
  const bool active = qw0 < q_len;
  const int wave_kend = active ? min(k_len, shift + min(qw0 + 32, q_len)) : 0;  // keys any query of the wave sees
  const int wave_kfull = shift + qw0 + 1;  // keys every query of the wave sees
  const int my_kend = shift + my_q + 1;
  const int my_lo = WIN ? my_kend - a.window : 0;            // first key of this lane's window
  const int wave_lo = WIN ? wave_kfull - a.window : 0;       // of the wave's first query's, and of its last one's
  const int wave_lo_last = WIN ? wave_lo + 31 : 0;
  auto needed = [&](int t) {  // whether any query of the wave sees a key of tile t
    const int key0 = key_of(t, 0);
    return key0 < wave_kend && (!WIN || key_of(t, 3) + 16 > wave_lo || key0 < a.sinks);
  };

  // Q^T B-operands: lane holds query my_q, d = 16s + 8(l/32) .. +7
  bf16x8_t qb[8];
  {
    const int qi = min(my_q, q_len - 1);
    const bf16_t* qp = a.q + (int64_t)(q0 + qi) * a.q_st + (int64_t)head * a.q_sh + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const Vec8 v = load_vec8(qp + 16 * s);
      __builtin_memcpy(&qb[s], &v, 16);
    }
  }
  floatx16_t o[4];
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[n][r] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  // Where the wave's 16 keys of a tile (a 16-aligned run inside one cache block of block_size tokens) are: block, row in
  // it.  Asked for tile after tile; the block id is not touched before the tile's loads, a tile later, so nothing waits
  // for it.
  const int step_blocks = PAGED ? kKeys / a.block_size : 0, step_rows = PAGED ? kKeys % a.block_size : 0;
  int at_block = 0, at_row = 0;
  auto page_of = [&](int t) {
    if (!PAGED) return Page{0, 0};
    const int j = key_of(t, wave);
    if (t == 0 || (WIN && 4 * t + wave < sink_16 + 4)) {  // not 64 keys behind the last ones, or maybe not
      at_block = j / a.block_size;
      at_row = j - at_block * a.block_size;
    } else {
      at_block += step_blocks;
      at_row += step_rows;
      if (at_row >= a.block_size) {
        at_row -= a.block_size;
        ++at_block;
      }
    }
    if (j >= k_len || (WIN && j >= a.sinks && j + 16 <= blk_lo)) return Page{0, 0};
    return Page{load_index(a.bt + (int64_t)b * a.bt_stride + at_block), at_row};
  };
  const LdsAddr ad = lds_addr(lds, lane);
  // S^T of one tile from K buffer PAR
  auto s_tile = [&](auto par_tag, floatx16_t (&s)[2]) {
    constexpr int PAR = decltype(par_tag)::value;
    bf16x8_t kf[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
    read_k16<PAR>(kf, ad);
#pragma unroll
    for (int u = 0; u < 8; ++u) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u], qb[u], s[0], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);  // the wait below stays behind these MFMAs
    k_wait_rest(kf);
#pragma unroll
    for (int u = 0; u < 8; ++u) s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[8 + u], qb[u], s[1], 0, 0, 0);
  };
  // online softmax of tile t's scores s -> P (bf16), O and l rescaled as needed
  auto softmax = [&](int t, floatx16_t (&s)[2], bf16x8_t (&pb)[2][2]) {
    const int key0 = key_of(t, 0), key3 = key_of(t, 3);
    // (on raw scores: scale > 0 keeps the order; p = exp2(s*scale - m*scale))
    // the tile crosses some query's diagonal, or the first key of some query's window
    if (key3 + 16 > wave_kfull || (WIN && key0 < wave_lo_last && key3 + 16 > a.sinks)) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = key_of(t, 2 * mt + (r >> 3)) + 8 * ((r >> 2) & 1) + 4 * h + (r & 3);
          s[mt][r] = key < my_kend && (!WIN || key >= my_lo || key < a.sinks) ? s[mt][r] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[mt][r]);
    mx = xor32_max(mx) * a.scale_log2;  // running max in the exp2 domain
    // lazy rescale: the max used for exp2 moves only when it grew by more
    // than kLazy (p <= 2^kLazy meanwhile; exact after the final 1/l)
    if (mx > m_run + kLazy) {
      const float alpha = __builtin_amdgcn_exp2f(m_run - mx);  // 0 on the first tile
      m_run = mx;
      l_run *= alpha;
#pragma unroll
      for (int n = 0; n < 4; ++n) o[n] *= alpha;
    }
    const float nm = m_run == -INFINITY ? 0.f : -m_run;  // fully masked so far: p = 0
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][8 * kk + 2 * e], a.scale_log2, nm));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][8 * kk + 2 * e + 1], a.scale_log2, nm));
          w[e] = pack_bf16x2(p0, p1);
          // the row sum takes the bf16 values P.V multiplies: their rounding (2^-8 of a weight at most, as in the other
          // kernels over bf16 pages) moves the output by that share of the values' spread only
          l_run = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(xv_bf16x2, w[e]), kOnes, l_run, false);
        }
        __builtin_memcpy(&pb[mt][kk], w, 16);
      }
  };
  // O^T += V^T P^T from V buffer PAR
  auto pv_tile = [&](auto par_tag, const bf16x8_t (&pb)[2][2]) {
    constexpr int PAR = decltype(par_tag)::value;
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {  // key-steps 2k2, 2k2+1 (= key tile mt = k2)
      short4_t vt[16];
      if (k2 == 0) read_vt_ks2<PAR, 0>(vt, ad); else read_vt_ks2<PAR, 2>(vt, ad);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt_operand(vt, n, j), pb[k2][j], o[n], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      vt_wait_rest(vt);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int n = 2; n < 4; ++n)
          o[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt_operand(vt, n, j), pb[k2][j], o[n], 0, 0, 0);
    }
  };

  // Software pipeline, one tile deep: iteration t computes S(t+1) from K
  // buffer (t+1)&1 while the softmax of tile t (scores from the previous
  // iteration) runs on the VALU, then O += P(t) V(t) from V buffer t&1.  K
  // therefore runs a tile ahead of V: iteration t loads K(t+2) into the K
  // buffer S(t) used and V(t+1) into the V buffer P(t-1) V(t-1) used, both
  // freed by the barrier at its top.
  const Page page0 = page_of(0);
  Page pv_page = ntiles > 1 ? page_of(1) : Page{0, 0}, pk_page = ntiles > 2 ? page_of(2) : Page{0, 0};
  if (ntiles > 0) load_rows<PAGED, true, true, WIN>(lds, a, b, kvh, key_of(0, wave), k0, k_len, page0, blk_lo, wave, lane);
  if (ntiles > 1)
    load_rows<PAGED, true, false, WIN>(lds + kBuf, a, b, kvh, key_of(1, wave), k0, k_len, pv_page, blk_lo, wave, lane);
  __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  // scores of even tiles in s_even, of odd tiles in s_odd (no copies)
  floatx16_t s_even[2], s_odd[2];
  if (ntiles > 0 && needed(0)) s_tile(std::integral_constant<int, 0>{}, s_even);
  auto iter = [&](auto par_tag, int t, floatx16_t (&sc)[2], floatx16_t (&sn)[2]) {
    constexpr int PAR = decltype(par_tag)::value;  // t & 1
    __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // K(t+1) and V(t) are in LDS; every wave is done with iteration t-1
    if (t + 2 < ntiles)
      load_rows<PAGED, true, false, WIN>(lds + PAR * kBuf, a, b, kvh, key_of(t + 2, wave), k0, k_len, pk_page, blk_lo, wave, lane);
    if (t + 1 < ntiles)
      load_rows<PAGED, false, true, WIN>(lds + (1 - PAR) * kBuf, a, b, kvh, key_of(t + 1, wave), k0, k_len, pv_page, blk_lo, wave, lane);
    pv_page = pk_page;
    if (t + 3 < ntiles) pk_page = page_of(t + 3);
    if (t + 1 < ntiles && needed(t + 1)) s_tile(std::integral_constant<int, 1 - PAR>{}, sn);
    if (needed(t)) {
      bf16x8_t pb[2][2];
      // the softmax is the serial link between MFMA phases: at raised issue
      // priority it runs ahead of the other wave on this SIMD, whose MFMAs
      // fill the gaps (measured +3-5 % over equal priority)
      __builtin_amdgcn_s_setprio(1);
      softmax(t, sc, pb);
      __builtin_amdgcn_s_setprio(0);
      pv_tile(par_tag, pb);
    }
  };
  for (int t = 0; t < ntiles; t += 2) {
    iter(std::integral_constant<int, 0>{}, t, s_even, s_odd);
    if (t + 1 < ntiles) iter(std::integral_constant<int, 1>{}, t + 1, s_odd, s_even);
  }
  // ---- normalise and write: lane holds O[my_q][32n + 8j + 4(l/32) + r] ----
  const float lsum = xor32_sum(l_run);
  if (!active) return;
  const float inv = lsum > 0.f ? 1.0f / lsum : 0.f;
  // By way of LDS, so that a store instruction takes four whole rows and not a piece of all 32: 8 KB of the K buffers, which
  // nobody reads from the last iteration's barrier on.  16-byte chunk c of row r is at slot c ^ r % 16.
  char* const mine = lds + (wave >> 1) * kBuf + (wave & 1) * (kTile / 2);
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint2 w = make_uint2(pack_bf16x2(o[n][4 * j] * inv, o[n][4 * j + 1] * inv),
                                 pack_bf16x2(o[n][4 * j + 2] * inv, o[n][4 * j + 3] * inv));
      *reinterpret_cast<uint2*>(mine + l32 * 256 + (((4 * n + j) ^ (l32 & 15)) << 4) + 8 * h) = w;
    }
  __asm__ __volatile__("" ::: "memory");  // a wave's LDS accesses stay in this order
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef u32x4 __attribute__((aligned(8))) u32x4_a8;  // the caller's rows are 8-byte aligned
  bf16_t* const op = a.out + (int64_t)(q0 + qw0) * a.out_st + (int64_t)head * kD + 8 * (lane & 15);
  u32x4 rows[8];
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int r = 4 * s + (lane >> 4);
    rows[s] = *reinterpret_cast<const u32x4*>(mine + r * 256 + (((lane & 15) ^ (r & 15)) << 4));
  }
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int r = 4 * s + (lane >> 4);
    if (qw0 + r < q_len) *reinterpret_cast<u32x4_a8*>(op + (int64_t)r * a.out_st) = rows[s];
  }
}

template <int G>
void launch(const PrefillArgs& a, dim3 grid, hipStream_t stream) {
  if (a.window > 0) {
    if (a.bt) prefill_kernel<G, true, true><<<grid, kThreads, 0, stream>>>(a);
    else prefill_kernel<G, false, true><<<grid, kThreads, 0, stream>>>(a);
  } else {
    if (a.bt) prefill_kernel<G, true, false><<<grid, kThreads, 0, stream>>>(a);
    else prefill_kernel<G, false, false><<<grid, kThreads, 0, stream>>>(a);
  }
}

// window 0: every query sees all keys up to itself (total_q is not looked at)
int prefill(const void* q, int64_t q_stride_tok, int64_t q_stride_head,
            const void* k, const void* v, int64_t kv_stride_tok, int64_t kv_stride_head,
            const void* k_cache, const void* v_cache,
            int64_t page_stride, int64_t tok_stride, int64_t head_stride,
            const int32_t* block_tables, int64_t bt_stride,
            const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
            void* out, int64_t out_stride_tok,
            int batch, int max_seqlen_q, int64_t total_q, int num_q_heads, int num_kv_heads,
            int head_dim, int block_size, int window, int sink_tokens, float scale,
            hipStream_t stream) {
  if (head_dim != kD || batch < 0 || total_q < 0 || total_q > INT32_MAX || num_kv_heads <= 0 || num_q_heads % num_kv_heads || max_seqlen_q < 0)
    return (int)hipErrorInvalidValue;
  const int group = num_q_heads / num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8) return (int)hipErrorInvalidValue;
  if (block_tables) {
    if (!k_cache || !v_cache || block_size <= 0 || block_size % 16) return (int)hipErrorInvalidValue;
    // K/V rows move by 16-byte LDS-DMA
    if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15 || (page_stride | tok_stride | head_stride) & 7)
      return (int)hipErrorInvalidValue;
  } else {
    if (!k || !v) return (int)hipErrorInvalidValue;
    if (((uintptr_t)k | (uintptr_t)v) & 15 || (kv_stride_tok | kv_stride_head) & 7) return (int)hipErrorInvalidValue;
  }
  // 32-bit offsets within 16 tokens
  const int64_t row = block_tables ? tok_stride : kv_stride_tok;
  if (row < 0 || row > (1 << 26)) return (int)hipErrorInvalidValue;
  // q rows are read as 16-byte vectors, out is written as 8-byte pieces
  if ((uintptr_t)q & 15 || (q_stride_tok | q_stride_head) & 7 || (uintptr_t)out & 7 || out_stride_tok & 3)
    return (int)hipErrorInvalidValue;
  if (batch == 0 || max_seqlen_q == 0) return 0;
  PrefillArgs a;
  a.q = (const bf16_t*)q; a.q_st = q_stride_tok; a.q_sh = q_stride_head;
  a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.kv_st = kv_stride_tok; a.kv_sh = kv_stride_head;
  a.kc = (const bf16_t*)k_cache; a.vc = (const bf16_t*)v_cache;
  a.page_stride = page_stride; a.tok_stride = tok_stride; a.head_stride = head_stride;
  a.bt = block_tables; a.bt_stride = bt_stride; a.block_size = block_size;
  a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k;
  a.out = (bf16_t*)out; a.out_st = out_stride_tok;
  a.hq = num_q_heads; a.hkv = num_kv_heads; a.batch = batch;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = min(window, 1 << 30); a.sinks = sink_tokens;  // positions are below 2^30
  const int gw = group < 4 ? group : 4;
  const int block_q = 32 * (4 / gw);
  a.qblocks = (max_seqlen_q + block_q - 1) / block_q;
  if (a.qblocks > 65535 || batch > 65535) return (int)hipErrorInvalidValue;  // grid y / z limits
  dim3 grid((unsigned)(num_kv_heads * (group == 8 ? 2 : 1)), (unsigned)a.qblocks, (unsigned)batch);
  if (window > 0) {
    if (total_q == 0) return 0;
    const int64_t blocks = min((int64_t)a.qblocks * batch, total_q / block_q + batch);
    grid.y = (unsigned)min(blocks, (int64_t)32768);
    grid.z = (unsigned)((blocks + 32767) / 32768);
  }
  switch (group) {
    case 1: launch<1>(a, grid, stream); break;
    case 2: launch<2>(a, grid, stream); break;
    case 4: launch<4>(a, grid, stream); break;
    default: launch<8>(a, grid, stream); break;
  }
  XV_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" int xv_prefill_attention(const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                                    const void* k, const void* v, int64_t kv_stride_tok, int64_t kv_stride_head,
                                    const void* k_cache, const void* v_cache,
                                    int64_t page_stride, int64_t tok_stride, int64_t head_stride,
                                    const int32_t* block_tables, int64_t bt_stride,
                                    const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                    void* out, int64_t out_stride_tok,
                                    int batch, int max_seqlen_q, int num_q_heads, int num_kv_heads,
                                    int head_dim, int block_size, float scale, hipStream_t stream) {
  return prefill(q, q_stride_tok, q_stride_head, k, v, kv_stride_tok, kv_stride_head, k_cache, v_cache, page_stride,
                 tok_stride, head_stride, block_tables, bt_stride, cu_seqlens_q, cu_seqlens_k, out, out_stride_tok, batch,
                 max_seqlen_q, 0, num_q_heads, num_kv_heads, head_dim, block_size, 0, 0, scale, stream);
}

extern "C" int xv_window_prefill_attention(const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                                           const void* k, const void* v, int64_t kv_stride_tok, int64_t kv_stride_head,
                                           const void* k_cache, const void* v_cache,
                                           int64_t page_stride, int64_t tok_stride, int64_t head_stride,
                                           const int32_t* block_tables, int64_t bt_stride,
                                           const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                           void* out, int64_t out_stride_tok,
                                           int batch, int max_seqlen_q, int64_t total_q, int num_q_heads, int num_kv_heads,
                                           int head_dim, int block_size, int window, int sink_tokens, float scale,
                                           hipStream_t stream) {
  if (window < 1 || sink_tokens < 0 || !(scale > 0.f)) return (int)hipErrorInvalidValue;
  return prefill(q, q_stride_tok, q_stride_head, k, v, kv_stride_tok, kv_stride_head, k_cache, v_cache, page_stride,
                 tok_stride, head_stride, block_tables, bt_stride, cu_seqlens_q, cu_seqlens_k, out, out_stride_tok, batch,
                 max_seqlen_q, total_q, num_q_heads, num_kv_heads, head_dim, block_size, window, sink_tokens, scale, stream);
}
