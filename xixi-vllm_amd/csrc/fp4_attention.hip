// Paged GQA decode attention over 4-bit (MXFP4) pages for gfx950.
//
// out[h] = sum_t softmax_t(scale * q[h] . K[t]) V[t], with K and V read as
// e2m1 codes (64 bytes a row of one kv head) and one e8m0 scale per 32 values
// (4 bytes a row).
//
// Work split, as the bf16 kernel's: the (sequence, kv head, 64-token unit)
// space is flattened in that order and cut into equal contiguous ranges, one
// per resident single-wave workgroup; segments cut by a range boundary leave
// partials (normalised bf16 rows and their log2-sum-exp) for a merge kernel.
// A range holds at most two cut segments (its first and its last), so a wave has two
// partial slots and the workspace does not grow with the table's width.
//
// A unit is 64 tokens: per lane that is one full set of operands.
//   K and V codes (4 KB each) and their scales (256 B each) go HBM -> LDS by
//   LDS-DMA.
//   S^T = K Q^T, v_mfma_f32_16x16x32_bf16, one product chain per 16-token row
//   block p: lane (g, i) reads the 16 bytes of token 16p + i's values 32g ..
//   32g + 31: exactly one scale block, so the conversion to bf16 (one
//   instruction per pair) applies the scale and is exact.
//   The scores land as acc[p][r] = head c % G, token 16p + 4g + r: the 16
//   tokens of lane group g, which are the k indices that group supplies to
//   O = P V.  V comes out of LDS by ds_read_b64_tr_b4, which gives a lane one
//   column of 16 rows: lane (g, i), tile n holds column 16n + i of those 16
//   tokens.  Its scale varies along the 16 rows and is folded into P, and P is
//   one operand for the columns of one scale block only.  The G heads fill G
//   of the 16 operand rows, so row rep * G + h takes head h scaled for block
//   rep (G = 8: two operands of two blocks): all blocks in one product, and
//   the outputs of the other blocks' rows are not used.
#include "xv_decode.h"
#include "xv_fp4.h"
#include "xv_kernels.h"
#include <math.h>

namespace {

constexpr int kD = 128;
constexpr int kRow = kD / 2;      // bytes of a head row's codes
constexpr int kUnit = 64;         // tokens of a unit
constexpr int kMaxBatch = 256;    // sequences per launch (larger batches are launched in chunks)
constexpr int kMaxWaves = 1024;   // workgroups of the main kernel at most
constexpr int kWavesPerCu = 4;    // one wave per SIMD
constexpr int kRing = 3;          // units in LDS per wave, kRing - 1 of them in flight
constexpr int kUnitOps = 10;      // LDS-DMA instructions a unit: 4 + 4 of codes, 1 + 1 of scales
// LDS of one unit: K codes, V codes, K scales, V scales, then the q rows of a segment that starts with it
constexpr int kVOff = 4096, kKsOff = 8192, kVsOff = 8448, kQOff = 8704;
template <int G> constexpr int kSlot = kQOff + (G <= 4 ? 1024 : G * 256);
constexpr int kIdWindow = 32;     // units per half of the block-id table (4 ids each)

struct Fp4DecodeArgs {
  const bf16_t* q; int64_t q_st, q_sh;
  const uint8_t* kc; const uint8_t* vc; int64_t ps, ts, hs;
  const uint8_t* ks; const uint8_t* vs; int64_t sps, sts, shs;
  const int32_t* bt; int64_t bt_stride;
  const int32_t* seqlens;
  bf16_t* out; int64_t out_st;
  int2* ws_seg;     // (first wave, partials) per (sequence, kv head)
  float* ws_lse;    // log2-sum-exp of partial slot s, head h at s * G + h
  bf16_t* ws_o;     // its rows, kD values each
  int batch, hq, hkv, group;
  int nsub;         // 16-token pages per cache block
  int max_ctx;      // tokens the block table has room for
  int nwaves;
  float scale_log2;
};

XV_INLINE int lds_int(const int* p) {
  int v;
  __asm__ __volatile__("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                       : "=&v"(v)
                       : "v"((uint32_t)reinterpret_cast<uintptr_t>(p))
                       : "memory");
  return __builtin_amdgcn_readfirstlane(v);
}

struct Fp4Cursor {
  int b, kvh, u;  // sequence, kv head, unit within the sequence
  int sub;        // 16-token page 4u modulo those of a cache block
  int nu, ctx;    // units and tokens of sequence b
};

// The next unit of the flat space (LDS reads in asm: a plain one would wait
// for every unit in flight).  Sequences without tokens are stepped over.
XV_INLINE void advance(Fp4Cursor& c, const int* pref, const int* sl, int hkv, int batch, int nsub) {
  if (++c.u < c.nu) {
    c.sub += 4;
    while (c.sub >= nsub) c.sub -= nsub;
    return;
  }
  c.u = 0;
  c.sub = 0;
  if (++c.kvh < hkv) return;
  c.kvh = 0;
  do {
    ++c.b;
    c.nu = lds_int(pref + c.b + 1) - lds_int(pref + c.b);
  } while (c.nu == 0 && c.b < batch - 1);
  c.ctx = lds_int(sl + c.b);
}

struct Fp4Lane {
  int g;           // global byte offset of this lane's piece of a 16-token page of codes
  uint32_t k;      // LDS offset of its K operand (row block 0)
  uint32_t v[4];   // LDS offsets of its transposed V reads of tiles 2m (tile 2m + 1: 8 bytes on)
  uint32_t ks, vs; // LDS offsets of its scales
};

// The 16-byte piece of a row sits in piece ^ (row / 4) of the row's 64 bytes:
// the 16 rows of a K read (one piece) then cover all banks once.
XV_INLINE Fp4Lane lane_offsets(int64_t tok_stride, int lane) {
  Fp4Lane o;
  const int i = lane & 15, g = lane >> 4;
  const int row = lane >> 2;
  o.g = (int)(row * tok_stride) + (((lane & 3) ^ (row >> 2)) << 4);
  o.k = (uint32_t)(64 * i + ((g ^ (i >> 2)) << 4));
  // input lane L of group g addresses token 16 (L / 4) + 4g + L % 4: output nibble L
#pragma unroll
  for (int m = 0; m < 4; ++m)
    o.v[m] = (uint32_t)(kVOff + 1024 * (i >> 2) + 64 * (4 * g + (i & 3)) + ((m ^ g) << 4));
  o.ks = (uint32_t)(kKsOff + 4 * i);
  o.vs = (uint32_t)(kVsOff + 16 * g);
  return o;
}

struct UnitRegs {
  u32x4_t k[4];                                          // K codes of row blocks 0..3
  uint32_t ks[4];                                        // the scale bytes of those tokens
  uint32_t v[8][2];                                      // V codes of column tiles 0..7, 16 tokens each
  u32x4_t vs[4];                                         // scale bytes of tokens 16p + 4g .. + 3
};

// A unit's operands out of its LDS image once at most VM vector-memory
// operations are outstanding, in one asm block with one wait.
template <int VM>
XV_INLINE void read_unit(UnitRegs& u, const char* buf, const Fp4Lane& lo) {
  typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
  const uint32_t b = (uint32_t)reinterpret_cast<uintptr_t>(buf);
  u32x2_t v[8];
  __asm__ __volatile__(
      "s_waitcnt vmcnt(%27)\n\t"
      "ds_read_b128 %0, %20\n\t"
      "ds_read_b128 %1, %20 offset:1024\n\t"
      "ds_read_b128 %2, %20 offset:2048\n\t"
      "ds_read_b128 %3, %20 offset:3072\n\t"
      "ds_read_b32 %4, %25\n\t"
      "ds_read_b32 %5, %25 offset:64\n\t"
      "ds_read_b32 %6, %25 offset:128\n\t"
      "ds_read_b32 %7, %25 offset:192\n\t"
      "ds_read_b64_tr_b4 %8, %21\n\t"
      "ds_read_b64_tr_b4 %9, %21 offset:8\n\t"
      "ds_read_b64_tr_b4 %10, %22\n\t"
      "ds_read_b64_tr_b4 %11, %22 offset:8\n\t"
      "ds_read_b64_tr_b4 %12, %23\n\t"
      "ds_read_b64_tr_b4 %13, %23 offset:8\n\t"
      "ds_read_b64_tr_b4 %14, %24\n\t"
      "ds_read_b64_tr_b4 %15, %24 offset:8\n\t"
      "ds_read_b128 %16, %26\n\t"
      "ds_read_b128 %17, %26 offset:64\n\t"
      "ds_read_b128 %18, %26 offset:128\n\t"
      "ds_read_b128 %19, %26 offset:192\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(u.k[0]), "=&v"(u.k[1]), "=&v"(u.k[2]), "=&v"(u.k[3]), "=&v"(u.ks[0]), "=&v"(u.ks[1]), "=&v"(u.ks[2]),
        "=&v"(u.ks[3]), "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]),
        "=&v"(v[7]), "=&v"(u.vs[0]), "=&v"(u.vs[1]), "=&v"(u.vs[2]), "=&v"(u.vs[3])
      : "v"(b + lo.k), "v"(b + lo.v[0]), "v"(b + lo.v[1]), "v"(b + lo.v[2]), "v"(b + lo.v[3]), "v"(b + lo.ks),
        "v"(b + lo.vs), "n"(VM)
      : "memory");
#pragma unroll
  for (int n = 0; n < 8; ++n) { u.v[n][0] = v[n][0]; u.v[n][1] = v[n][1]; }
}

struct Fp4State {
  float m;         // the softmax maximum in use (log2 domain) of head c % G, the same in the four lane rows
  float l;         // sum of p over this lane's tokens
  floatx4_t o[8];  // O tile n: operand rows 4g + r, column 16n + lane % 16
};

XV_INLINE void reset(Fp4State& st) {
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int n = 0; n < 8; ++n) st.o[n] = floatx4_t{0.f, 0.f, 0.f, 0.f};
}

XV_INLINE bf16x8_t widen8(uint32_t w, float scale) {
  uint32_t o[4];
  fp4x8_to_bf16(w, scale, o);
  bf16x8_t r;
  __builtin_memcpy(&r, o, 16);
  return r;
}

template <int G, int RR>
XV_INLINE void rescale_row(Fp4State& st, float alpha, int g) {
  const float ar = head_of_row<G, RR>(alpha, g);
#pragma unroll
  for (int n = 0; n < 8; ++n) st.o[n][RR] *= ar;
}

// Scores, softmax update and O += P V of one unit; tokens ntok .. 63 are masked.
template <int G>
XV_INLINE void unit_math(Fp4State& st, const UnitRegs& u, const bf16x8_t (&qb)[4], int ntok, float scale_log2, int lane) {
  const int g = lane >> 4, c = lane & 15;
  float sc[4][4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float s = fp4_scale(__builtin_amdgcn_ubfe(u.ks[p], 8 * g, 8));
    floatx4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(u.k[p][j], s), qb[j], acc, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) sc[p][r] = acc[r] * scale_log2;
  }
  if (ntok < kUnit) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * p + 4 * g + r >= ntok) sc[p][r] = -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int p = 0; p < 4; ++p) mx = fmaxf(mx, fmaxf(fmaxf(sc[p][0], sc[p][1]), fmaxf(sc[p][2], sc[p][3])));
  mx = xor32_max(xor16_max(mx));
  // the maximum in use moves only when some head's grew by more than kLazy
  const float m_new = fmaxf(st.m, mx);
  if (__any(m_new > st.m + kLazy)) {
    const float alpha = __builtin_amdgcn_exp2f(st.m - m_new);
    st.m = m_new;
    st.l *= alpha;
    rescale_row<G, 0>(st, alpha, g);
    rescale_row<G, 1>(st, alpha, g);
    rescale_row<G, 2>(st, alpha, g);
    rescale_row<G, 3>(st, alpha, g);
  }
  // p in fp32 for the sum; times the V scale and rounded to bf16 as the operand
  constexpr int NV = G == 8 ? 2 : 1;
  bf16x8_t pa[NV][2];
  const int shift = 8 * (G == 8 ? c >> 3 : G == 4 ? c >> 2 : (c / G) & 3);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t w[NV][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int p = 2 * j + e / 4, r = e % 4;
      const float p0 = __builtin_amdgcn_exp2f(sc[p][r] - st.m), p1 = __builtin_amdgcn_exp2f(sc[p][r + 1] - st.m);
      st.l += p0 + p1;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        // the low mantissa bit turns scale 255 into a NaN and moves the others by 2^-23 of themselves
        const float f0 = __uint_as_float((__builtin_amdgcn_ubfe(u.vs[p][r], shift + 16 * v, 8) << 23) | 1u);
        const float f1 = __uint_as_float((__builtin_amdgcn_ubfe(u.vs[p][r + 1], shift + 16 * v, 8) << 23) | 1u);
        w[v][e / 2] = pack_bf16x2(p0 * f0, p1 * f1);
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) __builtin_memcpy(&pa[v][j], w[v], 16);
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const int v = NV == 2 ? n / 4 : 0;
    st.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa[v][0], widen8(u.v[n][0], 1.0f), st.o[n], 0, 0, 0);
    st.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa[v][1], widen8(u.v[n][1], 1.0f), st.o[n], 0, 0, 0);
  }
}

template <int G>
XV_INLINE void issue_q(char* slot, const Fp4DecodeArgs& a, int b, int kvh, int lane) {
  const bf16_t* base = a.q + (int64_t)b * a.q_st + (int64_t)kvh * G * a.q_sh;
  const __amdgpu_buffer_rsrc_t rq = page_rsrc(base, (uint32_t)(((int64_t)(G - 1) * a.q_sh + kD) * 2));
#pragma unroll
  for (int j = 0; j < (G + 3) / 4; ++j) {
    const int row = 4 * j + (lane >> 4);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (lds_void*)(slot + 1024 * j), 16,
                                             (int)(row * a.q_sh * 2) + ((lane & 15) << 4), 0, 0, 0);
  }
}

// Q^T operand of step j: column c holds head c % G, its values 32g + 8j .. + 7.
template <int G, int VM>
XV_INLINE void read_q(bf16x8_t (&qb)[4], const char* slot, int lane) {
  const uint32_t a0 = (uint32_t)reinterpret_cast<uintptr_t>(slot) + ((lane & 15) % G) * 256 + (lane >> 4) * 64;
  __asm__ __volatile__(
      "s_waitcnt vmcnt(%5)\n\t"
      "ds_read_b128 %0, %4\n\t"
      "ds_read_b128 %1, %4 offset:16\n\t"
      "ds_read_b128 %2, %4 offset:32\n\t"
      "ds_read_b128 %3, %4 offset:48\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(qb[0]), "=&v"(qb[1]), "=&v"(qb[2]), "=&v"(qb[3])
      : "v"(a0), "n"(VM)
      : "memory");
}

// The finished segment's G rows: the bf16 output if the wave covered the whole
// segment (part < 0), else partial slot `part`.  They go through `stage` (the
// q slot in hand, its q in registers) and leave in 16-byte pieces; LDS access in asm.
template <int G>
XV_INLINE void finish_segment(const Fp4DecodeArgs& a, const Fp4State& st, int b, int kvh, int part, int lane, char* stage) {
  const int c = lane & 15, g = lane >> 4;
  const float lsum = xor32_sum(xor16_sum(st.l));
  const float inv_mine = 1.0f / lsum;
  const float inv[4] = {head_of_row<G, 0>(inv_mine, g), head_of_row<G, 1>(inv_mine, g), head_of_row<G, 2>(inv_mine, g),
                        head_of_row<G, 3>(inv_mine, g)};
  const uint32_t s0 = (uint32_t)reinterpret_cast<uintptr_t>(stage);
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const int rep = G == 8 ? (n >> 1) & 1 : n >> 1;  // which operand rows hold the scale block of tile n
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * g + r;
      if (row / G == rep) {
        const uint32_t at = s0 + (row % G) * (kD * 2) + 2 * (16 * n + c);
        __asm__ __volatile__("ds_write_b16 %0, %1" ::"v"(at), "v"(f32_to_bf16(st.o[n][r] * inv[r])) : "memory");
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's own writes precede its reads
  __builtin_amdgcn_wave_barrier();
  char* dst = part < 0 ? reinterpret_cast<char*>(a.out + (int64_t)b * a.out_st + (int64_t)kvh * G * kD)
                       : reinterpret_cast<char*>(a.ws_o + (int64_t)part * G * kD);
  constexpr int kBytes = G * kD * 2;
#pragma unroll
  for (int k = 0; k < (kBytes + 1023) / 1024; ++k) {
    const int off = 1024 * k + 16 * lane;
    if (off < kBytes) {
      u32x4_t v;
      __asm__ __volatile__("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(s0 + off) : "memory");
      typedef u32x4_t __attribute__((aligned(4))) u32x4_a4;  // the caller's rows need not be 16-byte aligned
      *reinterpret_cast<u32x4_a4*>(dst + off) = v;
    }
  }
  if (part >= 0 && lane < G) a.ws_lse[(int64_t)part * G + lane] = st.m + __log2f(lsum);
}

// Block ids of the wave's stream, 4 pages a unit, in a double-buffered LDS
// table filled by LDS-DMA from the block table.  Units past the range, and
// pages past a sequence's end, fetch an entry that exists.
XV_INLINE void load_window(char* half, const Fp4DecodeArgs& a, __amdgpu_buffer_rsrc_t rbt, const int* pref, const int* sl,
                           int64_t f0, int base, int n, int lane) {
#pragma unroll
  for (int j = 0; j < kIdWindow * 4 / 64; ++j) {
    const int y = base + 16 * j + (lane >> 2);
    int off = 0;
    if (y < n) {
      const int64_t f = f0 + y;
      const int b = seq_of(pref, a.batch, a.hkv, f);
      const int nu = pref[b + 1] - pref[b];
      const int r = (int)(f - (int64_t)a.hkv * pref[b]);
      const int page = min(4 * (r % nu) + (lane & 3), (sl[b] - 1) / 16);
      off = (int)(((int64_t)b * a.bt_stride + page / a.nsub) * 4);
    }
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rbt, (lds_void*)(half + 256 * j), 4, off, 0, 0, 0);
  }
}

template <int G>
__global__ __launch_bounds__(64) void fp4_decode_kernel(Fp4DecodeArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[kRing * kSlot<G>];
  __shared__ __attribute__((aligned(16))) char idtab[2 * kIdWindow * 16];
  __shared__ int pref[kMaxBatch + 1];  // units of sequences 0 .. b - 1
  __shared__ int sl[kMaxBatch];        // their tokens
  const int lane = threadIdx.x;
  int carry = 0, max_nu = 0;
  for (int c = 0; c < a.batch; c += 64) {
    const int b = c + lane;
    const int ctx = b < a.batch ? min(max(a.seqlens[b], 0), a.max_ctx) : 0;
    const int nu = (ctx + kUnit - 1) / kUnit;
    max_nu = max(max_nu, nu);
    int inc = nu;
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x111, 0xf, 0xf, true);  // inclusive scan: row_shr 1, 2, 4, 8,
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x112, 0xf, 0xf, true);  // then the row sums across rows
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x114, 0xf, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x118, 0xf, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x142, 0xa, 0xf, true);
    inc += __builtin_amdgcn_update_dpp(0, inc, 0x143, 0xc, 0xf, true);
    if (b < a.batch) {
      pref[b + 1] = carry + inc;
      sl[b] = ctx;
    }
    carry += __builtin_amdgcn_readlane(inc, 63);
  }
  if (lane == 0) pref[0] = 0;
  __syncthreads();
  max_nu = (int)wave_max((float)max_nu);  // exact in fp32 (below 2^24)
  const int64_t total = (int64_t)a.hkv * carry;
  // units per range: every wave the same, and no segment in more than kMergeMaxParts ranges
  const int L = (int)max((int64_t)max(1, (max_nu + kMergeMaxParts - 2) / (kMergeMaxParts - 1)),
                         (total + a.nwaves - 1) / a.nwaves);
  const int64_t f0 = (int64_t)blockIdx.x * L;
  const int n = (int)max((int64_t)0, min(f0 + L, total) - f0);
  if (n == 0) return;
  const Fp4Lane offs = lane_offsets(a.ts, lane);

  Fp4Cursor c0;
  c0.b = __builtin_amdgcn_readfirstlane(seq_of(pref, a.batch, a.hkv, f0));
  c0.nu = __builtin_amdgcn_readfirstlane(pref[c0.b + 1] - pref[c0.b]);
  c0.ctx = __builtin_amdgcn_readfirstlane(sl[c0.b]);
  {
    const int r = (int)(f0 - (int64_t)a.hkv * pref[c0.b]);
    c0.kvh = __builtin_amdgcn_readfirstlane(r / c0.nu);
    c0.u = __builtin_amdgcn_readfirstlane(r - c0.kvh * c0.nu);
    c0.sub = __builtin_amdgcn_readfirstlane((4 * c0.u) % a.nsub);
  }
  Fp4Cursor ic = c0, pc = c0;  // issue and process cursors
  const __amdgpu_buffer_rsrc_t rbt =
      page_rsrc(reinterpret_cast<const bf16_t*>(a.bt), (uint32_t)((int64_t)a.batch * a.bt_stride * 4));
  load_window(idtab, a, rbt, pref, sl, f0, 0, n, lane);
  load_window(idtab + kIdWindow * 16, a, rbt, pref, sl, f0, kIdWindow, n, lane);
  __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");
  int issued = -1;

  // Unit y (clamped to the range's last: a harmless re-read, so that every
  // call issues the same kUnitOps loads) into ring slot `slot`.
  auto issue = [&](int y, int slot) {
    char* buf = lds + slot * kSlot<G>;
    if (y > issued) {
      const bool newseg = issued < 0 || (advance(ic, pref, sl, a.hkv, a.batch, a.nsub), ic.u == 0);
      issued = y;
      if (y % kIdWindow == 0 && y > 0)  // entering window k (in place since window k - 1 began): request window k + 1
        load_window(idtab + ((y / kIdWindow + 1) & 1) * (kIdWindow * 16), a, rbt, pref, sl, f0, y + kIdWindow, n, lane);
      if (newseg) issue_q<G>(buf + kQOff, a, ic.b, ic.kvh, lane);
    }
    u32x4_t idv;
    __asm__ __volatile__("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                         : "=&v"(idv)
                         : "v"((uint32_t)reinterpret_cast<uintptr_t>(idtab) + ((y / kIdWindow) & 1) * (kIdWindow * 16) +
                               (y % kIdWindow) * 16)
                         : "memory");
    const int ntok = min(kUnit, ic.ctx - ic.u * kUnit);
    const int t = min(lane, ntok - 1);  // whose scales this lane fetches
    int64_t soff = 0;
    int sub = ic.sub;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t page = __builtin_amdgcn_readfirstlane(idv[j]);
      const int64_t base = page * a.ps + (int64_t)sub * (16 * a.ts) + (int64_t)ic.kvh * a.hs;
      const int rows = min(16, ntok - 16 * j);
      const uint32_t bytes = rows > 0 ? (uint32_t)((int64_t)(rows - 1) * a.ts + kRow) : 0u;  // rows past the end read as zeros
      const __amdgpu_buffer_rsrc_t rk = page_rsrc(reinterpret_cast<const bf16_t*>(a.kc + base), bytes);
      const __amdgpu_buffer_rsrc_t rv = page_rsrc(reinterpret_cast<const bf16_t*>(a.vc + base), bytes);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_void*)(buf + 1024 * j), 16, offs.g, 0, 0, kNontemporal);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_void*)(buf + kVOff + 1024 * j), 16, offs.g, 0, 0, kNontemporal);
      const int64_t sbase = page * a.sps + (int64_t)sub * (16 * a.sts) + (int64_t)ic.kvh * a.shs;
      if ((t >> 4) == j) soff = sbase;
      if (++sub == a.nsub) sub = 0;
    }
    soff += (int64_t)(t & 15) * a.sts;
    typedef const __attribute__((address_space(1))) void* gptr;
    __builtin_amdgcn_global_load_lds((gptr)(uintptr_t)(a.ks + soff), (lds_void*)(buf + kKsOff), 4, 0, 0);
    __builtin_amdgcn_global_load_lds((gptr)(uintptr_t)(a.vs + soff), (lds_void*)(buf + kVsOff), 4, 0, 0);
  };

  Fp4State st;
  reset(st);
  bf16x8_t qb[4];
  constexpr int kVm = kUnitOps * (kRing - 1);
  auto finish = [&](const Fp4Cursor& c, char* stage) {
    const int64_t seg0 = (int64_t)a.hkv * lds_int(pref + c.b) + (int64_t)c.kvh * c.nu;
    const bool first = seg0 >= f0, last = seg0 + c.nu <= f0 + n;
    // a segment that starts in this range and ends after it: slot 1 of the wave, one that started before: slot 0
    finish_segment<G>(a, st, c.b, c.kvh, first && last ? -1 : 2 * (int)blockIdx.x + (first ? 1 : 0), lane, stage);
    if (lane == 0 && last) {
      const int w0 = (int)(seg0 / L);
      a.ws_seg[c.b * a.hkv + c.kvh] = make_int2(w0, (int)blockIdx.x - w0 + 1);
    }
  };
  auto process = [&](int x, int slot) {
    char* buf = lds + slot * kSlot<G>;
    if (x > 0) {
      const Fp4Cursor prev = pc;
      advance(pc, pref, sl, a.hkv, a.batch, a.nsub);
      if (pc.u == 0) {
        read_q<G, kVm>(qb, buf + kQOff, lane);  // the new segment's q first: its slot then stages the finished one
        finish(prev, buf + kQOff);
        reset(st);
      }
    } else {
      read_q<G, kVm>(qb, buf + kQOff, lane);
    }
    UnitRegs u;
    read_unit<kVm>(u, buf, offs);
    unit_math<G>(st, u, qb, min(kUnit, pc.ctx - pc.u * kUnit), a.scale_log2, lane);
  };
#pragma unroll
  for (int k = 0; k < kRing - 1; ++k) issue(min(k, n - 1), k);
  for (int x0 = 0; x0 < n; x0 += kRing) {
#pragma unroll
    for (int u = 0; u < kRing; ++u) {
      issue(min(x0 + u + kRing - 1, n - 1), (u + kRing - 1) % kRing);
      if (x0 + u < n) process(x0 + u, u);
    }
  }
  __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");  // nothing still writes this wave's LDS when it ends
  finish(pc, lds + ((n - 1) % kRing) * kSlot<G> + kQOff);
}

// One wave per (sequence, query head): zeros for an empty sequence, else the
// weighted sum of its partials where the segment was cut.
__global__ __launch_bounds__(64) void fp4_merge_kernel(Fp4DecodeArgs a) {
  const int b = blockIdx.x / a.hq, h = blockIdx.x - b * a.hq, lane = threadIdx.x;
  const int kvh = h / a.group, hg = h - kvh * a.group;
  const int ctx = a.seqlens[b];
  const int2 seg = a.ws_seg[b * a.hkv + kvh];  // stale when ctx <= 0: not used then
  bf16_t* orow = a.out + (int64_t)b * a.out_st + (int64_t)h * kD;
  if (ctx <= 0) {
    *reinterpret_cast<uint32_t*>(orow + 2 * lane) = 0u;
    return;
  }
  if (seg.y <= 1) return;
  auto slot = [&](int j) { return (int64_t)(j == 0 ? 2 * seg.x + 1 : 2 * (seg.x + j)) * a.group + hg; };
  merge_general<false>(
      seg.y,
      [&](int j, int i, float4& lo, float4& hi) {
        float f[8];
        unpack8(load_vec8(a.ws_o + slot(j) * kD + 8 * i), f);
        lo = make_float4(f[0], f[1], f[2], f[3]);
        hi = make_float4(f[4], f[5], f[6], f[7]);
      },
      [&](int j) { return a.ws_lse[slot(j)]; }, 0.f, orow, lane);
}

int fp4_waves() {
  static int cached = 0;  // one GPU model per process
  if (!cached) {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      cus = 256;
    cached = min(kMaxWaves, max(1, cus) * kWavesPerCu);
  }
  return cached;
}

size_t al256(size_t x) { return (x + 255) / 256 * 256; }
size_t seg_bytes(int batch, int hkv) { return al256((size_t)min(batch, kMaxBatch) * hkv * sizeof(int2)); }
size_t lse_bytes(int group) { return al256((size_t)kMaxWaves * 2 * group * sizeof(float)); }

}  // namespace

extern "C" size_t xv_paged_decode_fp4_workspace_size(int batch, int num_q_heads, int num_kv_heads) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads) return 256;
  const int group = num_q_heads / num_kv_heads;
  return seg_bytes(batch, num_kv_heads) + lse_bytes(group) + (size_t)kMaxWaves * 2 * group * kD * sizeof(bf16_t);
}

extern "C" int xv_paged_decode_attention_fp4(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache, const void* v_cache,
    int64_t page_stride, int64_t tok_stride, int64_t head_stride, const void* k_scale, const void* v_scale,
    int64_t scale_page_stride, int64_t scale_tok_stride, int64_t scale_head_stride, const int32_t* block_tables,
    int64_t bt_stride, const int32_t* cache_seqlens, void* out, int64_t out_stride_tok, void* workspace,
    size_t workspace_bytes, int batch, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
    int max_blocks_per_seq, float scale, hipStream_t stream) {
  if (head_dim != kD || block_size <= 0 || block_size % 16 || batch < 0 || num_kv_heads <= 0 ||
      num_q_heads <= 0 || num_q_heads % num_kv_heads || max_blocks_per_seq <= 0)
    return (int)hipErrorInvalidValue;
  const int group = num_q_heads / num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8) return (int)hipErrorInvalidValue;
  const int64_t max_ctx = (int64_t)max_blocks_per_seq * block_size;
  if (max_ctx > (1 << 28)) return (int)hipErrorInvalidValue;  // 256M tokens per sequence
  // rows move by 16-byte (scales by 4-byte) LDS-DMA at 32-bit offsets within a page
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15 || (q_stride_tok | q_stride_head) & 7 ||
      (page_stride | tok_stride | head_stride) & 15 || ((uintptr_t)k_scale | (uintptr_t)v_scale) & 3 ||
      (scale_page_stride | scale_tok_stride | scale_head_stride) & 3)
    return (int)hipErrorInvalidValue;
  if (tok_stride < kRow || tok_stride > (1 << 26) || scale_tok_stride < 4 || scale_tok_stride > (1 << 26) ||
      q_stride_head < 0 || q_stride_head > (1 << 26) || bt_stride < max_blocks_per_seq ||
      (int64_t)kMaxBatch * bt_stride * 4 > INT32_MAX)
    return (int)hipErrorInvalidValue;
  if ((uintptr_t)out & 3 || out_stride_tok & 1) return (int)hipErrorInvalidValue;
  if (batch == 0) return 0;
  if (workspace == nullptr || (uintptr_t)workspace & 15 ||
      workspace_bytes < xv_paged_decode_fp4_workspace_size(batch, num_q_heads, num_kv_heads))
    return (int)hipErrorInvalidValue;
  Fp4DecodeArgs a;
  a.q_st = q_stride_tok; a.q_sh = q_stride_head;
  a.kc = (const uint8_t*)k_cache; a.vc = (const uint8_t*)v_cache; a.ps = page_stride; a.ts = tok_stride; a.hs = head_stride;
  a.ks = (const uint8_t*)k_scale; a.vs = (const uint8_t*)v_scale;
  a.sps = scale_page_stride; a.sts = scale_tok_stride; a.shs = scale_head_stride;
  a.bt_stride = bt_stride; a.out_st = out_stride_tok;
  a.ws_seg = (int2*)workspace;
  a.ws_lse = (float*)((char*)workspace + seg_bytes(batch, num_kv_heads));
  a.ws_o = (bf16_t*)((char*)a.ws_lse + lse_bytes(group));
  a.hq = num_q_heads; a.hkv = num_kv_heads; a.group = group;
  a.nsub = block_size / 16; a.max_ctx = (int)max_ctx;
  a.scale_log2 = scale * 1.4426950408889634f;
  for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {
    a.batch = min(kMaxBatch, batch - b0);
    a.q = (const bf16_t*)q + (int64_t)b0 * q_stride_tok;
    a.bt = block_tables + (int64_t)b0 * bt_stride;
    a.seqlens = cache_seqlens + b0;
    a.out = (bf16_t*)out + (int64_t)b0 * out_stride_tok;
    a.nwaves = (int)min((int64_t)fp4_waves(), (int64_t)a.batch * num_kv_heads * ((max_ctx + kUnit - 1) / kUnit));
    switch (group) {
      case 1: fp4_decode_kernel<1><<<a.nwaves, 64, 0, stream>>>(a); break;
      case 2: fp4_decode_kernel<2><<<a.nwaves, 64, 0, stream>>>(a); break;
      case 4: fp4_decode_kernel<4><<<a.nwaves, 64, 0, stream>>>(a); break;
      default: fp4_decode_kernel<8><<<a.nwaves, 64, 0, stream>>>(a); break;
    }
    XV_CHECK_LAUNCH();
    fp4_merge_kernel<<<(unsigned)(a.batch * num_q_heads), 64, 0, stream>>>(a);
    XV_CHECK_LAUNCH();
  }
  return 0;
}
