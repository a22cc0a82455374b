// Paged GQA decode attention over 4-bit (MXFP4) pages for gfx950.
//
// out[h] = sum_t softmax_t(scale * q[h] . K[t]) V[t], with K and V read as
// e2m1 codes (64 bytes a row of one kv head) and one e8m0 scale per 32 values
// (4 bytes a row).
//
// Work split: the (sequence, kv head, 64-token unit) space is flattened in
// that order and cut into equal contiguous ranges, one per wave, eight waves a
// CU; segments cut by a range boundary leave partials (normalised fp32 rows and
// their log2-sum-exp) for a merge kernel.  A range holds at most two cut
// segments (its first and its last), so a wave has two partial slots and the
// workspace does not grow with the table's width.
//
// A unit is 64 tokens: per lane that is one full set of operands.
//   K and V codes (4 KB each) and their scales (256 B each) go HBM -> LDS by
//   LDS-DMA, one unit ahead of the one in work.
//   S^T = K Q^T on v_mfma_scale_f32_16x16x128_f8f6f4, one 16-token row block p
//   per product: operand A is K as it is stored, lane (g, i) the 16 bytes of
//   token 16p + i's values 32g .. 32g + 31 with that block's own scale byte.
//   Operand B is q as the sum of two e4m3 terms (see split_q): no conversion of K.
//   The scores land as acc[p][r] = head c % G, token 16p + 4g + r: the 16
//   tokens of lane group g, which are the k indices that group supplies to
//   O = P V (bf16).  V comes out of LDS by ds_read_b64_tr_b4, which gives a lane
//   one column of 16 rows: lane (g, i), tile n holds column 16n + i of those 16
//   tokens.  Its scale varies along the 16 rows and is folded into P, and P is
//   one operand for the columns of one scale block only.  The G heads fill G
//   of the 16 operand rows, so row rep * G + h takes head h scaled for block
//   rep (G = 8: two operands of two blocks): all blocks in one product, and
//   the outputs of the other blocks' rows are not used.  P times the scale goes
//   in as two bf16 terms, two products each.
//
// 64 sequences of 512 .. 4096 tokens (32 heads over 8) take 44 us: 12 of
// launches, start (lengths, then block ids, then pages) and merge, the rest the
// page stream at 5 TB/s (its tail with the units' arithmetic); four of 40000 ..
// 130000 (16 over 8) 80 us, 4.9 TB/s over the whole call.  A segment is cut into
// kMaxParts at most, so one sequence of 130000 with one kv head has 185 of the
// 2048 waves at work: 36 us.
#include "xv_decode.h"
#include "xv_fp4.h"
#include "xv_kernels.h"
#include <math.h>

namespace {

constexpr int kD = 128;
constexpr int kRow = kD / 2;      // bytes of a head row's codes
constexpr int kUnit = 64;         // tokens of a unit
constexpr int kMaxBatch = 256;    // sequences per launch (larger batches are launched in chunks)
constexpr int kWaves = 8;         // waves of a workgroup, one workgroup per CU
constexpr int kMaxGroups = 256;   // workgroups at most
constexpr int kMaxWaves = kWaves * kMaxGroups;
constexpr int kMaxParts = 192;    // partials of a segment at most
constexpr int kUnitOps = 10;      // LDS-DMA instructions a unit: 4 + 4 of codes, 1 + 1 of scales
// LDS of one unit: K codes, V codes, K scales, V scales
constexpr int kVOff = 4096, kKsOff = 8192, kVsOff = 8448, kUnitLds = 8704;
constexpr int kIdWindow = 16;     // units per half of the block-id table (4 ids each)
// LDS of one wave: two units, the q rows of a segment, the block-id table
template <int G> constexpr int kQBytes = G <= 4 ? 1024 : G * 256;
template <int G> constexpr int kWaveLds = 2 * kUnitLds + kQBytes<G> + 2 * kIdWindow * 16;

struct Fp4DecodeArgs {
  const bf16_t* q; int64_t q_st, q_sh;
  const uint8_t* kc; const uint8_t* vc; uint32_t ps, ts, hs;
  const uint8_t* ks; const uint8_t* vs; uint32_t sps, sts, shs;
  const int32_t* bt; int64_t bt_stride;
  const int32_t* seqlens;
  bf16_t* out; int64_t out_st;
  int2* ws_seg;     // (first wave, partials) per (sequence, kv head)
  float* ws_lse;    // log2-sum-exp of partial slot s, head h at s * G + h
  float* ws_o;      // its rows, kD values each
  int batch, hq, hkv, group;
  int nsub;         // 16-token pages per cache block
  int max_ctx;      // tokens the block table has room for
  float scale_log2; // not negative: q_sign carries the sign of the scale
  float q_sign;
};

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(1))) void* global_cptr;

XV_INLINE int lds_int(const int* p) {
  int v;
  __asm__ __volatile__("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                       : "=&v"(v)
                       : "v"((uint32_t)reinterpret_cast<uintptr_t>(p))
                       : "memory");
  return __builtin_amdgcn_readfirstlane(v);
}
XV_INLINE u32x4_t lds_ids(const char* p) {
  u32x4_t v;
  __asm__ __volatile__("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                       : "=&v"(v)
                       : "v"((uint32_t)reinterpret_cast<uintptr_t>(p))
                       : "memory");
  return v;
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

// LDS offsets of a lane within a unit, and of its 16-byte piece within a page
// of codes.  Piece j of a row sits in slot j ^ swz4(row) of the row's 64 bytes.
struct Fp4Lane {
  uint32_t g;      // global byte offset of this lane's piece of a 16-token page
  uint32_t k;      // K operand, row block 0 (block p: + 1024 p)
  uint32_t v[4];   // transposed V reads of tiles 2m (tile 2m + 1: 8 bytes on)
  uint32_t ks, vs; // scales
  uint32_t own;    // V scales of token `lane`
};

XV_INLINE Fp4Lane lane_offsets(uint32_t tok_stride, int lane) {
  Fp4Lane o;
  const int i = lane & 15, g = lane >> 4;
  const int row = lane >> 2;
  o.g = row * tok_stride + (((lane & 3) ^ swz4(row)) << 4);
  o.k = (uint32_t)(64 * i + ((g ^ swz4(i)) << 4));
  // input lane L of group g addresses token 16 (L / 4) + 4g + L % 4: output nibble L
#pragma unroll
  for (int m = 0; m < 4; ++m)
    o.v[m] = (uint32_t)(kVOff + 1024 * (i >> 2) + 64 * (4 * g + (i & 3)) + ((m ^ swz4(4 * g)) << 4));
  o.ks = (uint32_t)(kKsOff + 4 * i);
  o.vs = (uint32_t)(kVsOff + 16 * g);
  o.own = (uint32_t)(kVsOff + 4 * lane);
  return o;
}

struct UnitRegs {
  u32x4_t k[4];      // K codes of row blocks 0..3
  uint32_t ks[4];    // the scale bytes of those tokens
  uint32_t v[8][2];  // V codes of column tiles 0..7, 16 tokens each
  u32x4_t vs[4];     // scale bytes of tokens 16p + 4g .. + 3
  uint32_t own;      // those of token `lane`
  u32x4_t ids;       // block ids of a later unit
};

// A unit's operands out of its LDS image (its loads have arrived) in one asm block with one wait.
XV_INLINE void read_unit(UnitRegs& u, const char* buf, const Fp4Lane& lo, const char* ids) {
  typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
  const uint32_t b = (uint32_t)reinterpret_cast<uintptr_t>(buf);
  u32x2_t v[8];
  __asm__ __volatile__(
      "ds_read_b128 %0, %22\n\t"
      "ds_read_b128 %1, %22 offset:1024\n\t"
      "ds_read_b128 %2, %22 offset:2048\n\t"
      "ds_read_b128 %3, %22 offset:0xc00\n\t"
      "ds_read_b32 %4, %27\n\t"
      "ds_read_b32 %5, %27 offset:64\n\t"
      "ds_read_b32 %6, %27 offset:128\n\t"
      "ds_read_b32 %7, %27 offset:192\n\t"
      "ds_read_b64_tr_b4 %8, %23\n\t"
      "ds_read_b64_tr_b4 %9, %23 offset:8\n\t"
      "ds_read_b64_tr_b4 %10, %24\n\t"
      "ds_read_b64_tr_b4 %11, %24 offset:8\n\t"
      "ds_read_b64_tr_b4 %12, %25\n\t"
      "ds_read_b64_tr_b4 %13, %25 offset:8\n\t"
      "ds_read_b64_tr_b4 %14, %26\n\t"
      "ds_read_b64_tr_b4 %15, %26 offset:8\n\t"
      "ds_read_b128 %16, %28\n\t"
      "ds_read_b128 %17, %28 offset:64\n\t"
      "ds_read_b128 %18, %28 offset:128\n\t"
      "ds_read_b128 %19, %28 offset:192\n\t"
      "ds_read_b128 %20, %29\n\t"
      "ds_read_b32 %21, %30\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(u.k[0]), "=&v"(u.k[1]), "=&v"(u.k[2]), "=&v"(u.k[3]), "=&v"(u.ks[0]), "=&v"(u.ks[1]), "=&v"(u.ks[2]),
        "=&v"(u.ks[3]), "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]),
        "=&v"(v[7]), "=&v"(u.vs[0]), "=&v"(u.vs[1]), "=&v"(u.vs[2]), "=&v"(u.vs[3]), "=&v"(u.ids),
        "=&v"(u.own)
      : "v"(b + lo.k), "v"(b + lo.v[0]), "v"(b + lo.v[1]), "v"(b + lo.v[2]), "v"(b + lo.v[3]), "v"(b + lo.ks),
        "v"(b + lo.vs), "v"((uint32_t)reinterpret_cast<uintptr_t>(ids)), "v"(b + lo.own)
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

// q as two e4m3 terms with power-of-two scales per 32 values.  The first is
// scaled to a largest magnitude of 128 .. 256 and rounds to 4 significant
// bits; the rest (at most 8, and at most 2^-4 of the value) is exact in 4 more
// bits for values within 2^-10 of the block's largest, and within 2^-21 of the
// largest otherwise: far below the fp32 rounding of a 128-term product of
// values of that size.  An infinity or NaN converts to NaN.
struct QSplit {
  v8i_t hi, lo;       // operand B of 128 values: lane (g, c) holds values 16g .. + 15 and 64 + 16g .. + 15 of head c % G
  int s_hi, s_lo;     // the scale bytes of block g (values 32g .. 32g + 31)
};

XV_INLINE void split_q(QSplit& o, const u32x4_t (&raw)[4], float sign, int lane) {
  typedef short v2s_t __attribute__((ext_vector_type(2)));
  int byte[2];
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float f[16];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t w = raw[2 * half + e / 4][e % 4];
      top = max(top, max((w >> 16) & 0x7fffu, w & 0x7fffu));
      f[2 * e] = bf16lo(w) * sign;
      f[2 * e + 1] = bf16hi(w) * sign;
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));  // the block's other 16 values: lane group g ^ 1
    byte[half] = max((int)(top >> 7) - 7, 5);
    const float inv = __uint_as_float((uint32_t)(254 - byte[half]) << 23), s4 = 0.0625f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v2s_t h = {0, 0}, l = {0, 0};
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = f[4 * e + j] * inv;
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, x[0], x[1], 1.0f, false);
      h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, x[2], x[3], 1.0f, true);
      uint32_t hb, lb;
      __builtin_memcpy(&hb, &h, 4);
      const auto b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hb, 1.0f, false);
      const auto b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hb, 1.0f, true);
      l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, x[0] - b0[0], x[1] - b0[1], s4, false);
      l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, x[2] - b1[0], x[3] - b1[1], s4, true);
      __builtin_memcpy(&lb, &l, 4);
      hi[4 * half + e] = hb;
      lo[4 * half + e] = lb;
    }
  }
  __builtin_memcpy(&o.hi, hi, 32);
  __builtin_memcpy(&o.lo, lo, 32);
  // lane group g holds blocks g / 2 and 2 + g / 2; block b's scale comes from group 2 (b % 2)
  const int g = lane >> 4, c = lane & 15;
  const int b0 = __shfl(byte[0], 32 * (g & 1) + c), b1 = __shfl(byte[1], 32 * (g & 1) + c);
  o.s_hi = g < 2 ? b0 : b1;
  o.s_lo = o.s_hi - 4;
}

XV_INLINE bf16x8_t widen8(uint32_t w) {
  uint32_t o[4];
  fp4x8_to_bf16(w, 1.0f, o);
  bf16x8_t r;
  __builtin_memcpy(&r, o, 16);
  return r;
}

// The scales 2^(byte - 127) of one byte each of t0 and t1 (sel: a v_perm_b32 selector that brings them to bytes 0 and
// 2), as the two bf16 of a dword.  Byte 0 is the subnormal 2^-127; 255 is an infinity here, which the second
// operand of P turns into a NaN (infinity less infinity).
XV_INLINE uint32_t v_scales(uint32_t t0, uint32_t t1, uint32_t sel) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const uint32_t w = __builtin_amdgcn_perm(t1, t0, sel);
  u16x2 b;
  __builtin_memcpy(&b, &w, 4);
  b = __builtin_elementwise_max((u16x2)(b << (uint16_t)7), (u16x2){0x0040, 0x0040});
  uint32_t r;
  __builtin_memcpy(&r, &b, 4);
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
XV_INLINE void unit_math(Fp4State& st, const UnitRegs& u, const QSplit& q, int ntok, float scale_log2, int lane) {
  const int g = lane >> 4, c = lane & 15;
  floatx4_t acc[4];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const v8i_t k = {(int)u.k[p][0], (int)u.k[p][1], (int)u.k[p][2], (int)u.k[p][3], 0, 0, 0, 0};
    const int s = (int)(u.ks[p] >> (8 * g));  // byte 0: the scale of this lane's block
    acc[p] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    acc[p] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q.lo, acc[p], 4, 0, 0, s, 0, q.s_lo);
    acc[p] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q.hi, acc[p], 4, 0, 0, s, 0, q.s_hi);
  }
  const bool tail = ntok < kUnit;
  if (tail) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * p + 4 * g + r >= ntok) acc[p][r] = -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int p = 0; p < 4; ++p) mx = fmaxf(mx, fmaxf(fmaxf(acc[p][0], acc[p][1]), fmaxf(acc[p][2], acc[p][3])));
  // Weights reach 2^kLazy, times V's scale they are bf16 operands, times up to 6 and summed over up to 2^28 tokens
  // fp32 outputs: where a scale of the unit is 2^65 or more (two top bits set; 2^125 is the largest that the store
  // writes) its weights stay 2^40 lower, and where all are below 2^-63 they go 2^64 higher, out of the subnormals.
  // The maximum in use moves by as much, and the sum of the weights with it.
  const bool huge = __any(u.own & (u.own << 1) & 0x80808080u), tiny = !__any(u.own & 0xc0c0c0c0u);
  mx = xor32_max(xor16_max(mx)) * scale_log2 + (huge ? 40.f : tiny ? -64.f : 0.f);
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
  float pr[4][4];
#pragma unroll
  for (int p = 0; p < 4; ++p)
#pragma unroll
    for (int r = 0; r < 4; ++r) pr[p][r] = __builtin_amdgcn_exp2f(fmaf(acc[p][r], scale_log2, -st.m));
  if (tail) {  // also where a scale of 0 makes -inf * scale a NaN
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * p + 4 * g + r >= ntok) pr[p][r] = 0.f;
  }
  // p in fp32 for the sum; times the V scale as the sum of two bf16 operands, its nearest bf16 and the nearest one
  // of the rest, together within 2^-16 of it.  (The first alone, within 2^-8: 64 rows 40.8 us against 43.5, 48 with 8
  // heads a group 43.0 against 46.2, but where few tokens share the weight its error is as large as the output's own
  // rounding.)
  constexpr int NV = G == 8 ? 2 : 1;
  bf16x8_t pa[NV][2], pb[NV][2];
  const uint32_t sel = 0x0c040c00u + 0x10001u * (uint32_t)(G == 8 ? c >> 3 : G == 4 ? c >> 2 : (c / G) & 3);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t w[NV][4], rest[NV][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int p = 2 * j + e / 4, r = e % 4;
      st.l += pr[p][r] + pr[p][r + 1];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const uint32_t f = v_scales(u.vs[p][r], u.vs[p][r + 1], sel + 0x20002u * v);
        const float p0 = pr[p][r] * bf16lo(f), p1 = pr[p][r + 1] * bf16hi(f);
        w[v][e / 2] = pack_bf16x2(p0, p1);
        rest[v][e / 2] = pack_bf16x2(p0 - bf16lo(w[v][e / 2]), p1 - bf16hi(w[v][e / 2]));
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      __builtin_memcpy(&pa[v][j], w[v], 16);
      __builtin_memcpy(&pb[v][j], rest[v], 16);
    }
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const int v = NV == 2 ? n / 4 : 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bf16x8_t t = widen8(u.v[n][j]);
      st.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pb[v][j], t, st.o[n], 0, 0, 0);
      st.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pa[v][j], t, st.o[n], 0, 0, 0);
    }
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

// This lane's 32 values of head c % G out of the q slot: 16g .. + 15 and 64 + 16g .. + 15.
template <int G>
XV_INLINE void read_q(u32x4_t (&raw)[4], const char* slot, int lane) {
  const uint32_t a0 = (uint32_t)reinterpret_cast<uintptr_t>(slot) + ((lane & 15) % G) * 256 + (lane >> 4) * 32;
  __asm__ __volatile__(
      "ds_read_b128 %0, %4\n\t"
      "ds_read_b128 %1, %4 offset:16\n\t"
      "ds_read_b128 %2, %4 offset:128\n\t"
      "ds_read_b128 %3, %4 offset:144\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(raw[0]), "=&v"(raw[1]), "=&v"(raw[2]), "=&v"(raw[3])
      : "v"(a0)
      : "memory");
}

// 1 KB or less from the stage to row pieces of ROW bytes, BYTES apart in memory.
template <int SIZE, int ROW, typename Dst>
XV_INLINE void unstage(uint32_t s0, char* dst, int64_t stride, int lane) {
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the wave's own writes precede its reads
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int k = 0; k < (SIZE + 1023) / 1024; ++k) {
    const int off = 1024 * k + 16 * lane;
    if (off < SIZE) {
      u32x4_t v;
      __asm__ __volatile__("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(s0 + off) : "memory");
      *reinterpret_cast<Dst*>(dst + off / ROW * stride + off % ROW) = v;
    }
  }
}

// The finished segment's G rows: the bf16 output if the wave covered the whole
// segment (part < 0), else partial slot `part`, in fp32.  They go through
// `stage` (the q slot, its q in registers), a partial by halves of its rows, and
// leave in 16-byte pieces; LDS access in asm.
template <int G>
XV_INLINE void finish_segment(const Fp4DecodeArgs& a, const Fp4State& st, int b, int kvh, int part, int lane, char* stage) {
  const int c = lane & 15, g = lane >> 4;
  const float lsum = xor32_sum(xor16_sum(st.l));
  const float inv_mine = 1.0f / lsum;
  const float inv[4] = {head_of_row<G, 0>(inv_mine, g), head_of_row<G, 1>(inv_mine, g), head_of_row<G, 2>(inv_mine, g),
                        head_of_row<G, 3>(inv_mine, g)};
  const uint32_t s0 = (uint32_t)reinterpret_cast<uintptr_t>(stage);
  constexpr int kStage = G * kD * 2;
  auto put = [&](int n, auto store) {  // column tile n: store(head, column within the tile, value)
    const int rep = G == 8 ? (n >> 1) & 1 : n >> 1;  // which operand rows hold the scale block of tile n
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 4 * g + r;
      if (row / G == rep) store(row % G, c, st.o[n][r] * inv[r]);
    }
  };
  if (part < 0) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
      put(n, [&](int h, int col, float v) {
        __asm__ __volatile__("ds_write_b16 %0, %1" ::"v"(s0 + h * (kD * 2) + 2 * (16 * n + col)), "v"(f32_to_bf16(v)) : "memory");
      });
    typedef u32x4_t __attribute__((aligned(4))) u32x4_a4;  // the caller's rows need not be 16-byte aligned
    unstage<kStage, kStage, u32x4_a4>(s0, reinterpret_cast<char*>(a.out + (int64_t)b * a.out_st + (int64_t)kvh * G * kD), 0, lane);
    return;
  }
  char* const dst = reinterpret_cast<char*>(a.ws_o + (int64_t)part * G * kD);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int n = 4 * half; n < 4 * half + 4; ++n)
      put(n, [&](int h, int col, float v) {
        __asm__ __volatile__("ds_write_b32 %0, %1" ::"v"(s0 + h * (kD * 2) + 4 * (16 * (n & 3) + col)), "v"(v) : "memory");
      });
    unstage<kStage, kD * 2, u32x4_t>(s0, dst + half * (kD * 2), kD * 4, lane);
  }
  if (lane < G) a.ws_lse[(int64_t)part * G + lane] = st.m + __log2f(lsum);
}

// Block ids of the wave's stream, 4 pages a unit, in a double-buffered LDS
// table filled by LDS-DMA from the block table.  Units past the range, and
// pages past a sequence's end, fetch an entry that exists.
XV_INLINE void load_window(char* half, const Fp4DecodeArgs& a, __amdgpu_buffer_rsrc_t rbt, const int* pref, const int* sl,
                           int64_t f0, int base, int n, int lane) {
  static_assert(kIdWindow * 4 == 64, "one id per lane");
  const int y = base + (lane >> 2);
  int off = 0;
  if (y < n) {
    const int64_t f = f0 + y;
    const int b = seq_of(pref, a.batch, a.hkv, f);
    const int nu = pref[b + 1] - pref[b];
    const int r = (int)(f - (int64_t)a.hkv * pref[b]);
    const int page = min(4 * (r % nu) + (lane & 3), (sl[b] - 1) / 16);
    off = (int)(((int64_t)b * a.bt_stride + page / a.nsub) * 4);
  }
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rbt, (lds_void*)half, 4, off, 0, 0, 0);
}

template <int G>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp4_decode_kernel(Fp4DecodeArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kWaveLds<G>];
  __shared__ int pref[kMaxBatch + 1];  // units of sequences 0 .. b - 1
  __shared__ int sl[kMaxBatch];        // their tokens
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave == 0) {
    int carry = 0;
    for (int c = 0; c < a.batch; c += 64) {
      const int b = c + lane;
      const int ctx = b < a.batch ? min(max(a.seqlens[b], 0), a.max_ctx) : 0;
      int inc = (ctx + kUnit - 1) / kUnit;
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
  }
  __syncthreads();
  int longest = 0;
  for (int b = lane; b < a.batch; b += 64) longest = max(longest, sl[b]);
  const int max_nu = ((int)wave_max((float)((longest + kUnit - 1) / kUnit)));  // exact in fp32 (below 2^24)
  const int64_t total = (int64_t)a.hkv * __builtin_amdgcn_readfirstlane(pref[a.batch]);
  // units per range: every wave the same, and no segment in more than kMaxParts ranges
  const int nwaves = gridDim.x * kWaves;
  const int L = (int)max((int64_t)max(1, (max_nu + kMaxParts - 2) / (kMaxParts - 1)), (total + nwaves - 1) / nwaves);
  const int id = wave * gridDim.x + blockIdx.x;  // short launches spread over the CUs first
  const int64_t f0 = (int64_t)id * L;
  const int n = (int)max((int64_t)0, min(f0 + L, total) - f0);
  if (n == 0) return;
  char* const mine = lds + wave * kWaveLds<G>;
  char* const qslot = mine + 2 * kUnitLds;
  char* const idtab = qslot + kQBytes<G>;
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
  if (n > kIdWindow) load_window(idtab + kIdWindow * 16, a, rbt, pref, sl, f0, kIdWindow, n, lane);
  __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");

  // Unit y, whose cursor is ic and whose block ids are idv, into its ring
  // slot, non-temporally (64 rows 44.3 us, 45.8 through the caches; four long ones 81 and 89).  A page's rows past the
  // sequence's end are read as they are (they are masked, and every code is finite); their scales are those of the last
  // token.
  auto issue = [&](int y, const u32x4_t& idv) {
    char* buf = mine + (y & 1) * kUnitLds;
    if (y % kIdWindow == 0 && y > 0)  // entering window k (in place since window k - 1 began): request window k + 1
      load_window(idtab + ((y / kIdWindow + 1) & 1) * (kIdWindow * 16), a, rbt, pref, sl, f0, y + kIdWindow, n, lane);
    const int t = min(lane, ic.ctx - ic.u * kUnit - 1);  // whose scales this lane fetches
    const uint64_t hoff = (uint64_t)(uint32_t)ic.kvh * a.hs;
    uint32_t id_t = 0, row_t = 0;
    int sub = ic.sub;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t page = (uint32_t)__builtin_amdgcn_readfirstlane((int)idv[j]);
      const uint64_t base = (uint64_t)page * a.ps + hoff + (uint64_t)(uint32_t)(16 * sub) * a.ts;
      __builtin_amdgcn_global_load_lds((global_cptr)(a.kc + base + offs.g), (lds_void*)(buf + 1024 * j), 16, 0, kNontemporal);
      __builtin_amdgcn_global_load_lds((global_cptr)(a.vc + base + offs.g), (lds_void*)(buf + kVOff + 1024 * j), 16, 0,
                                       kNontemporal);
      if ((t >> 4) == j) {
        id_t = page;
        row_t = 16 * sub;
      }
      if (++sub == a.nsub) sub = 0;
    }
    const uint64_t soff = (uint64_t)id_t * a.sps + (uint64_t)(row_t + (t & 15)) * a.sts + (uint64_t)(uint32_t)ic.kvh * a.shs;
    __builtin_amdgcn_global_load_lds((global_cptr)(a.ks + soff), (lds_void*)(buf + kKsOff), 4, 0, 0);
    __builtin_amdgcn_global_load_lds((global_cptr)(a.vs + soff), (lds_void*)(buf + kVsOff), 4, 0, 0);
  };
  auto ids_at = [&](int y) { return idtab + ((y / kIdWindow) & 1) * (kIdWindow * 16) + (y % kIdWindow) * 16; };

  Fp4State st;
  QSplit q;
  auto finish = [&](const Fp4Cursor& c) {
    const int64_t seg0 = (int64_t)a.hkv * lds_int(pref + c.b) + (int64_t)c.kvh * c.nu;
    const bool first = seg0 >= f0, last = seg0 + c.nu <= f0 + n;
    // a segment that starts in this range and ends after it: slot 1 of the wave, one that started before: slot 0
    finish_segment<G>(a, st, c.b, c.kvh, first && last ? -1 : 2 * id + (first ? 1 : 0), lane, qslot);
    if (lane == 0 && last) {
      const int w0 = (int)(seg0 / L);
      a.ws_seg[c.b * a.hkv + c.kvh] = make_int2(w0, id - w0 + 1);
    }
  };
  // Unit x begins a segment (or the range): take its q, then write out the segment before through the q slot.
  auto begin_segment = [&](int x, const Fp4Cursor& prev) {
    u32x4_t raw[4];
    read_q<G>(raw, qslot, lane);
    if (x > 0) finish(prev);
    reset(st);
    split_q(q, raw, a.q_sign, lane);
  };
  issue_q<G>(qslot, a, ic.b, ic.kvh, lane);
  issue(0, lds_ids(ids_at(0)));
  UnitRegs u;
  u.ids = lds_ids(ids_at(1));
  for (int x = 0; x < n; ++x) {
    const Fp4Cursor prev = pc;
    if (x > 0) pc = ic;
    const bool seg = x == 0 || pc.u == 0;
    const bool next = x + 1 < n;
    // where the next unit begins a segment too, its q would overwrite this one's before it is read
    const bool early = seg && next && pc.u + 1 == pc.nu;
    if (early) {
      __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");
      begin_segment(x, prev);
    }
    if (next) {
      advance(ic, pref, sl, a.hkv, a.batch, a.nsub);
      if (ic.u == 0) issue_q<G>(qslot, a, ic.b, ic.kvh, lane);
      issue(x + 1, u.ids);
      static_assert(kUnitOps == 10, "the wait below");
      __asm__ __volatile__("s_waitcnt vmcnt(10)" ::: "memory");
    } else {
      __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if (seg && !early) begin_segment(x, prev);
    read_unit(u, mine + (x & 1) * kUnitLds, offs, ids_at(x + 2));
    unit_math<G>(st, u, q, min(kUnit, pc.ctx - pc.u * kUnit), a.scale_log2, lane);
  }
  finish(pc);
}

// One wave per (sequence, query head), four a workgroup: zeros for an empty
// sequence, else the sum of its partials, each by its share of the segment's
// mass, where the segment was cut.  16 lanes hold a row (8 values each), the
// four lane rows take every fourth partial, four in flight each: up to sixteen
// partials cost one memory round trip after the segment's record.
__global__ __launch_bounds__(256) void fp4_merge_kernel(Fp4DecodeArgs a) {
  const int task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
  if (task >= a.batch * a.hq) return;
  const int b = task / a.hq, h = task - b * a.hq;
  const int kvh = h / a.group, hg = h - kvh * a.group;
  const int ctx = a.seqlens[b];
  const int2 seg = a.ws_seg[b * a.hkv + kvh];  // stale when ctx <= 0: not used then
  bf16_t* orow = a.out + (int64_t)b * a.out_st + (int64_t)h * kD;
  if (ctx <= 0) {
    *reinterpret_cast<uint32_t*>(orow + 2 * lane) = 0u;
    return;
  }
  const int n = seg.y;
  if (n <= 1) return;
  auto slot = [&](int j) { return (j == 0 ? 2 * seg.x + 1 : 2 * (seg.x + j)) * a.group + hg; };  // < 2^15
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
  const float mx = wave_max(fmaxf(la, fmaxf(lb, lc)));
  float wa = __builtin_amdgcn_exp2f(la - mx), wb = __builtin_amdgcn_exp2f(lb - mx), wc = __builtin_amdgcn_exp2f(lc - mx);
  const float inv = 1.0f / wave_sum(wa + wb + wc);  // before the rows: their sum stays within their own range
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

int fp4_groups() {
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

size_t al256(size_t x) { return (x + 255) / 256 * 256; }
size_t seg_bytes(int batch, int hkv) { return al256((size_t)min(batch, kMaxBatch) * hkv * sizeof(int2)); }
size_t lse_bytes(int group) { return al256((size_t)kMaxWaves * 2 * group * sizeof(float)); }

}  // namespace

extern "C" size_t xv_paged_decode_fp4_workspace_size(int batch, int num_q_heads, int num_kv_heads) {
  if (batch <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads) return 256;
  const int group = num_q_heads / num_kv_heads;
  return seg_bytes(batch, num_kv_heads) + lse_bytes(group) + (size_t)kMaxWaves * 2 * group * kD * sizeof(float);
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
      page_stride < 0 || page_stride > INT32_MAX || head_stride < 0 || head_stride > INT32_MAX || scale_page_stride < 0 ||
      scale_page_stride > INT32_MAX || scale_head_stride < 0 || scale_head_stride > INT32_MAX || q_stride_head < 0 ||
      q_stride_head > (1 << 26) || bt_stride < max_blocks_per_seq || bt_stride > INT32_MAX ||
      min(batch, kMaxBatch) * bt_stride * 4 > INT32_MAX)  // the rows of a launch's table: one buffer
    return (int)hipErrorInvalidValue;
  if ((uintptr_t)out & 3 || out_stride_tok & 1) return (int)hipErrorInvalidValue;
  if (batch == 0) return 0;
  if (workspace == nullptr || (uintptr_t)workspace & 15 ||
      workspace_bytes < xv_paged_decode_fp4_workspace_size(batch, num_q_heads, num_kv_heads))
    return (int)hipErrorInvalidValue;
  Fp4DecodeArgs a;
  a.q_st = q_stride_tok; a.q_sh = q_stride_head;
  a.kc = (const uint8_t*)k_cache; a.vc = (const uint8_t*)v_cache;
  a.ps = (uint32_t)page_stride; a.ts = (uint32_t)tok_stride; a.hs = (uint32_t)head_stride;
  a.ks = (const uint8_t*)k_scale; a.vs = (const uint8_t*)v_scale;
  a.sps = (uint32_t)scale_page_stride; a.sts = (uint32_t)scale_tok_stride; a.shs = (uint32_t)scale_head_stride;
  a.bt_stride = bt_stride; a.out_st = out_stride_tok;
  a.ws_seg = (int2*)workspace;
  a.ws_lse = (float*)((char*)workspace + seg_bytes(batch, num_kv_heads));
  a.ws_o = (float*)((char*)a.ws_lse + lse_bytes(group));
  a.hq = num_q_heads; a.hkv = num_kv_heads; a.group = group;
  a.nsub = block_size / 16; a.max_ctx = (int)max_ctx;
  a.scale_log2 = fabsf(scale) * 1.4426950408889634f;
  a.q_sign = scale < 0.f ? -1.f : 1.f;
  for (int b0 = 0; b0 < batch; b0 += kMaxBatch) {
    a.batch = min(kMaxBatch, batch - b0);
    a.q = (const bf16_t*)q + (int64_t)b0 * q_stride_tok;
    a.bt = block_tables + (int64_t)b0 * bt_stride;
    a.seqlens = cache_seqlens + b0;
    a.out = (bf16_t*)out + (int64_t)b0 * out_stride_tok;
    const int64_t units = (int64_t)a.batch * num_kv_heads * ((max_ctx + kUnit - 1) / kUnit);
    const unsigned groups = (unsigned)min((int64_t)fp4_groups(), units);
    switch (group) {
      case 1: fp4_decode_kernel<1><<<groups, kWaves * 64, 0, stream>>>(a); break;
      case 2: fp4_decode_kernel<2><<<groups, kWaves * 64, 0, stream>>>(a); break;
      case 4: fp4_decode_kernel<4><<<groups, kWaves * 64, 0, stream>>>(a); break;
      default: fp4_decode_kernel<8><<<groups, kWaves * 64, 0, stream>>>(a); break;
    }
    XV_CHECK_LAUNCH();
    fp4_merge_kernel<<<(unsigned)((a.batch * num_q_heads + 3) / 4), 256, 0, stream>>>(a);
    XV_CHECK_LAUNCH();
  }
  return 0;
}
