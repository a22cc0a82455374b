// Products of a decode batch with 4-bit (MXFP4) weights on gfx950:
//   out[m, n] = sum_k x[m, k] * code[n, k] * 2^(scale[n, k / 32] - 127)
// and, of a gate / up weight, silu(gate) * up.
//
// A short batch is bound by the weight's bytes (N K / 2 of codes, N K / 32 of
// scales).  v_mfma_f32_16x16x32_bf16 with the weight as operand A: lane (g, i)
// of 128 values takes weight row i's values 32g .. 32g + 31, 16 bytes and
// exactly one scale block, widened to bf16 with the scale applied by the
// conversion (one instruction per pair, exact); operand B is x, column = row
// of x, the same values.
//
// Up to kShort rows: a workgroup owns T tiles of 16 weight rows, its eight
// waves take turns of KS values along K (their fp32 sums meet in LDS at the
// end), and a wave runs its T tiles over one slice before the next: x is read
// once per workgroup and its slice waits in registers, while the weight streams
// through a private LDS ring.  Both travel by LDS-DMA, whole row segments per
// instruction.  One row through a gate / up weight of 24576 x 4096 takes 12.5 us
// (4.3 TB/s), 8 rows through 4096 x 12288 9.5 us.  Direct loads into the operand
// registers, where neighbouring lanes are neighbouring rows, were bound by the
// address unit (weights so: 22 us for the first; x alone so: 12.7 us for the
// second).  Every workgroup reads all of its part of x through its LDS-DMA, which
// is what bounds more than 16 rows (37 rows of an odd 5003 x 4704 weight 12.0 us).
#include "xv_decode.h"
#include "xv_fp4.h"
#include "xv_fp4_plan.h"
#include "xv_kernels.h"
#include <type_traits>

namespace {

struct Fp4GemmArgs {
  const bf16_t* x; int64_t x_st;
  const uint8_t* w; int64_t w_st;   // codes, bytes between rows
  const uint8_t* s; int64_t s_st;   // scales, bytes between rows
  bf16_t* out; int64_t out_st;
  int m, n, k;                      // n: outputs (of SILU: half the weight's rows)
};

// A product whose K may be cut into parts, which a second kernel adds.
struct Fp4PartArgs {
  Fp4GemmArgs g;
  float* parts;       // null: out is written
  int64_t part_size;  // floats of a part: m x (rows of the weight)
  int per;            // slices or steps of a part
};

// 16 bytes a lane, `off` behind `base` (both of these wave uniform), into LDS in lane order, with the bytes from base to
// end as the buffer's size: past it nothing is read.
template <int POLICY>
XV_INLINE void load_lds(const void* base, const void* end, char* to, uint32_t off) {
  const uint64_t n = reinterpret_cast<uint64_t>(end) - reinterpret_cast<uint64_t>(base);
  const __amdgpu_buffer_rsrc_t r = page_rsrc(static_cast<const bf16_t*>(base), n < 0xffffffffu ? (uint32_t)n : 0xffffffffu);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)to, 16, off, 0, 0, POLICY);
}

XV_INLINE float silu_mul(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

XV_INLINE bf16x8_t widen8(uint32_t w, float scale) {
  uint32_t o[4];
  fp4x8_to_bf16(w, scale, o);
  bf16x8_t r;
  __builtin_memcpy(&r, o, 16);
  return r;
}

typedef const __attribute__((address_space(1))) void* global_cptr;

constexpr int kWaves = kFp4Waves;

// One stage: the codes of 16 weight rows x KS values, rows of KS / 2 bytes,
// swizzled.  Scales come with a slice of x, a window of SW dwords of each of the
// workgroup's rows: a load of few lanes costs what a full one does (with every
// stage its own scales: 32 rows through a 24576 x 4096 gate / up weight 21.6 us).
// A scale row need not start at a multiple of 4 bytes (WIDE): the window then
// starts at the dword that holds the first byte.
template <int KS, bool WIDE>
struct Stage {
  static constexpr int kPieces = KS / 32;               // 16-byte pieces (scale blocks) of a row
  static constexpr int kBytes = 16 * KS / 2;
  static constexpr int kLoads = kBytes / 1024;          // LDS-DMA instructions
  static constexpr int kRowsPer = 64 / kPieces;         // rows one of them covers
  static constexpr int SW = !WIDE ? KS / 128 : KS / 64;
  static constexpr int kSteps = KS / 128;               // operand loads of 128 values
  static XV_INLINE int swz(int row) {
    static_assert(KS == 128 || KS == 256, "rows of 64 or 128 bytes");
    return KS == 128 ? swz4(row) : swz8p(row);
  }
};

// Where piece j of x row r sits in LDS: slot j ^ swz_x(r).  Eight rows serve
// all sixteen lanes of a group; bit 2, where neighbouring groups' pieces
// differ, stays free.
template <int XR>
XV_INLINE int swz_x(int r) {
  return XR == 8 ? (r & 3) | ((r & 4) << 1) : swz16(r);
}

// A stage's operands of the lane in one asm block with one wait: one piece of
// codes (at wa) and one scale byte (sa, 4 bytes on) for each 128 values.
template <int N>
XV_INLINE void read_stage(u32x4_t (&w)[N], uint32_t (&s)[N], const uint32_t (&wa)[N], uint32_t sa) {
  static_assert(N == 1 || N == 2, "slices of 128 or 256 values");
  if constexpr (N == 2) {
    __asm__ __volatile__(
        "ds_read_b128 %0, %4\n\t"
        "ds_read_b128 %1, %5\n\t"
        "ds_read_u8 %2, %6\n\t"
        "ds_read_u8 %3, %6 offset:4\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(s[0]), "=&v"(s[1])
        : "v"(wa[0]), "v"(wa[1]), "v"(sa)
        : "memory");
  } else {
    __asm__ __volatile__(
        "ds_read_b128 %0, %2\n\t"
        "ds_read_u8 %1, %3\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(s[0])
        : "v"(wa[0]), "v"(sa)
        : "memory");
  }
}

// Eight operand reads of x in one asm block with one wait.
XV_INLINE void read_x8(u32x4_t (&v)[8], const uint32_t (&at)[8]) {
  __asm__ __volatile__(
      "ds_read_b128 %0, %8\n\t"
      "ds_read_b128 %1, %9\n\t"
      "ds_read_b128 %2, %10\n\t"
      "ds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %12\n\t"
      "ds_read_b128 %5, %13\n\t"
      "ds_read_b128 %6, %14\n\t"
      "ds_read_b128 %7, %15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7])
      : "memory");
}

template <int N>
XV_INLINE void wait_vm() {
  static_assert(N >= 0 && N <= 63, "the counter's range");
  __asm__ __volatile__("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Wait until at most A + min(n, MAX) * B are outstanding; n known where it is unrolled.
template <int A, int B, int MAX>
XV_INLINE void wait_vm_of(int n) {
  if constexpr (MAX > 0) {
    if (n < MAX) return wait_vm_of<A, B, MAX - 1>(n);
  }
  wait_vm<A + B * MAX>();
}

// m <= XR rows of x as MT column tiles of 16 (XR = 8: the tile's upper half
// repeats the lower, its outputs are not stored); XD slices of x in LDS.
template <int MT, int XR, int KS, int XD, int T, bool SILU, bool WIDE>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp4_gemm_kernel(Fp4PartArgs pa) {
  const Fp4GemmArgs& a = pa.g;
  using S = Stage<KS, WIDE>;
  constexpr int kXBytes = XR * KS * 2, kXLoads = kXBytes / 1024, kXPieces = KS / 8;
  constexpr int kSLoads = (T * 16 * S::SW + 63) / 64, kSBytes = kSLoads * 256;  // the scales of a slice
  constexpr int kSlice = kXLoads + kSLoads;                                      // instructions that come with a slice
  // Stages in a wave's ring, one less of them in flight.  (Four to eight: no faster.)
  constexpr int kRest = XD * kXBytes + (XD + 1) * kSBytes, kDepth = kRest + 3 * S::kBytes <= 163840 / kWaves ? 3 : 2;
  constexpr int kWave = kDepth * S::kBytes + kRest;         // LDS of one wave
  // Weight loads are non-temporal where a wave runs through whole 128-byte lines of several tiles (one row of a 24576 x
  // 4096 weight 12.1 us against 13.0), not where two waves share a line (64 rows through 4096 x 12288 22.9 against 29.2)
  // or the workgroup has one tile (8 rows through it 9.5 against 11.1).
  constexpr int kPolicy = KS == 256 && T > 2 ? kNontemporal : 0;
  constexpr int P = SILU ? 2 : 1;
  // tiles summed over the waves at a time: all that LDS holds
  constexpr int kTR = 163840 / (kWaves * MT * 1024) / P * P, TR = T < kTR ? T : kTR;
  constexpr int kRed = kWaves * TR * MT * 1024;
  static_assert(kXLoads >= 1 && kWaves * kWave <= 163840 && kRed <= 163840, "LDS of a CU");
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kWave > kRed ? kWaves * kWave : kRed];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (SILU ? T / 2 : T) * 16;
  char* const ring = lds + wave * kWave;
  char* const xring = ring + kDepth * S::kBytes;
  char* const sring = xring + XD * kXBytes;
  const int blocks = a.k / kFp4Block;
  const int first = blockIdx.y * pa.per + wave, last = min((a.k + KS - 1) / KS, (int)(blockIdx.y + 1) * pa.per);
  const int mine = last > first ? (last - first + kWaves - 1) / kWaves : 0;  // slices first, first + 8, ... below last
  const int total = mine * T;                                                // stages of this wave

  // weight row of operand row r of tile t: SILU has the gate and the up rows of the same outputs in tiles 2p, 2p + 1
  auto wrow = [&](int t, int r) {
    const int o = min(n0 + (SILU ? t >> 1 : t) * 16 + r, a.n - 1);
    return (int64_t)o + (SILU && (t & 1) ? a.n : 0);
  };
  const uintptr_t s_last =  // the dword that holds the last scale
      (reinterpret_cast<uintptr_t>(a.s) + (uint64_t)((SILU ? 2 * (int64_t)a.n : a.n) - 1) * a.s_st + blocks - 1) & ~(uintptr_t)3;
  // This lane's offsets within a stage and within a slice of x.  The code of a stage is short on purpose: a wave
  // runs it few times, mostly for the first time.  Rows and blocks past the end are left to the buffers' bounds (their
  // outputs are not stored, or x is zero there).  (With clamped rows by address, twice the instructions: 64 rows
  // of the 24576 x 4096 gate / up weight 26.7 us against 25.9.)
  uint32_t coff[S::kLoads], xoff[kXLoads];
#pragma unroll
  for (int q = 0; q < S::kLoads; ++q) {
    const int row = S::kRowsPer * q + lane / S::kPieces;
    coff[q] = row * (uint32_t)a.w_st + 16 * ((lane % S::kPieces) ^ S::swz(row));
  }
#pragma unroll
  for (int q = 0; q < kXLoads; ++q) {
    const int row = (64 * q + lane) / kXPieces;
    xoff[q] = row * 2 * (uint32_t)a.x_st + 16 * ((lane % kXPieces) ^ swz_x<XR>(row));
  }
  const uint8_t* const w_end = a.w + ((SILU ? 2 * (int64_t)a.n : a.n) - 1) * a.w_st + 16 * (int64_t)blocks;
  const uint8_t* const wg = a.w + n0 * a.w_st;
  const uint8_t* const wu = wg + (SILU ? (int64_t)a.n * a.w_st : 0);
  const bf16_t* const x_end = a.x + (a.m - 1) * a.x_st + a.k;
  // the scale rows this lane fetches from, and the dword of the window
  uintptr_t srow[kSLoads];
  uint32_t sdw[kSLoads];
#pragma unroll
  for (int q = 0; q < kSLoads; ++q) {
    const int at = min(64 * q + lane, T * 16 * S::SW - 1);
    srow[q] = reinterpret_cast<uintptr_t>(a.s) + (uint64_t)(wrow(at / (16 * S::SW), at / S::SW % 16) * a.s_st);
    sdw[q] = 4 * (at % S::SW);
  }
  // LDS-DMA instructions issued so far, and the count when each slice of x's last one left: what was issued
  // since may still be in flight when it is waited for
  int ops = 0, xmark[XD];
#pragma unroll
  for (int d = 0; d < XD; ++d) xmark[d] = 0;
  int issued = 0, is = first;  // stages issued, the next one's slice
  auto issue = [&](int slot, int it) {  // it: the next one's tile
    char* buf = ring + slot * S::kBytes;
    const uint32_t at = (uint32_t)(SILU ? it >> 1 : it) * 16 * (uint32_t)a.w_st + 16 * S::kPieces * (uint32_t)is;
#pragma unroll
    for (int q = 0; q < S::kLoads; ++q) load_lds<kPolicy>(SILU && (it & 1) ? wu : wg, w_end, buf + 1024 * q, coff[q] + at);
    ++issued;
    ops += S::kLoads;
    if (it == T - 1) is += kWaves;
  };
  // Slice `slice` of x: row r's KS values (2 KS bytes, swizzled) at r * 2 KS; and its scales.
  auto issue_x = [&](int slice, int slot, int sslot) {
#pragma unroll
    for (int q = 0; q < kXLoads; ++q)
      load_lds<0>(a.x, x_end, xring + slot * kXBytes + 1024 * q, xoff[q] + 2 * KS * (uint32_t)slice);
#pragma unroll
    for (int q = 0; q < kSLoads; ++q) {
      const uintptr_t src = min(((srow[q] + (uint32_t)(slice * S::kPieces)) & ~(uintptr_t)3) + sdw[q], s_last);
      __builtin_amdgcn_global_load_lds((global_cptr)src, (lds_void*)(sring + sslot * kSBytes + 256 * q), 4, 0, 0);
    }
    ops += kSlice;
    xmark[slot] = ops;
  };

  // operand B: lane (g, i) of step h, substep j holds row i's values 128 h + 32 g + 8 j .. + 7
  u32x4_t x[S::kSteps * MT * 4];
  auto take_x = [&](int slice, int slot) {
    const uint32_t b = (uint32_t)reinterpret_cast<uintptr_t>(xring + slot * kXBytes);
#pragma unroll
    for (int p = 0; p < S::kSteps * MT; p += 2) {
      uint32_t at[8];
      u32x4_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int pe = min(p + (e >> 2), S::kSteps * MT - 1), h = pe / MT, u = pe % MT;
        const int row = (16 * u + i) % XR;
        at[e] = b + row * (KS * 2) + (((16 * h + 4 * g + (e & 3)) ^ swz_x<XR>(row)) << 4);
      }
      read_x8(v, at);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (p + (e >> 2) < S::kSteps * MT) x[(p + (e >> 2)) * 4 + (e & 3)] = v[e];
    }
    if (slice * KS + KS > a.k) {
#pragma unroll
      for (int h = 0; h < S::kSteps; ++h)
        if (slice * KS + 128 * h + 32 * g >= a.k) {  // whole blocks: a lane's 32 values lie inside or outside
#pragma unroll
          for (int e = 0; e < MT * 4; ++e) x[h * MT * 4 + e] = u32x4_t{0, 0, 0, 0};
        }
    }
  };

  floatx4_t acc[T][MT];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = floatx4_t{0.f, 0.f, 0.f, 0.f};

  // this lane's pieces within a stage
  uint32_t wat[S::kSteps];
#pragma unroll
  for (int h = 0; h < S::kSteps; ++h)
    wat[h] = (uint32_t)(i * (KS / 2) + (((4 * h + g) ^ S::swz(i)) << 4));
  int wslot = 0, xslot = 0, sslot = 0;  // ring slots of the next stage, slice and its scales to use
  if (mine > 0) {
#pragma unroll
    for (int d = 0; d < XD; ++d)
      if (d < mine) issue_x(first + d * kWaves, d, d);
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d)
      if (issued < total) issue(d, d % T);
  }
  for (int s = 0; s < mine; ++s) {
    const int slice = first + s * kWaves;
    {
      int since = ops;
#pragma unroll
      for (int d = 0; d < XD; ++d)
        if (d == xslot) since = ops - xmark[d];
      constexpr int kFull = XD > 1 ? XD * S::kLoads + (XD - 1) * kSlice : (T < kDepth ? T : kDepth - 1) * S::kLoads;
      constexpr int kFirst = (kDepth - 1) * S::kLoads + (XD - 1) * kSlice;  // the first slice: the first loads of all
      if (since >= kFull) wait_vm<kFull>();
      else if (kFirst < kFull && since >= kFirst) wait_vm<kFirst>();
      else wait_vm<0>();
      take_x(slice, xslot);
      if (s + XD < mine) issue_x(slice + XD * kWaves, xslot, sslot == 0 ? XD : sslot - 1);  // past the last slice's scales
      if (++xslot == XD) xslot = 0;
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      // This stage left kDepth - 1 stages ago.  Slices that began since, each with a slice of x (of which at most XD
      // are still in flight):
      constexpr int kSince = kDepth - 1;
      const int kSlices = t < kSince ? (kSince - t + T - 1) / T : 0;
      const bool steady = issued < total;
      if (steady) issue(wslot == 0 ? kDepth - 1 : wslot - 1, (t + kSince) % T);
      const uint32_t b = (uint32_t)reinterpret_cast<uintptr_t>(ring + wslot * S::kBytes);
      uint32_t wa[S::kSteps];
#pragma unroll
      for (int h = 0; h < S::kSteps; ++h) wa[h] = b + wat[h];
      uint32_t m4 = 0;  // where in its first dword the row's scale bytes start
      if constexpr (WIDE) m4 = (uint32_t)((reinterpret_cast<uintptr_t>(a.s) + (uint64_t)(wrow(t, i) * a.s_st + slice * S::kPieces)) & 3);
      const uint32_t sa = (uint32_t)reinterpret_cast<uintptr_t>(sring + sslot * kSBytes) + (t * 16 + i) * (4 * S::SW) + m4 + g;
      if (++wslot == kDepth) wslot = 0;
      if (steady) {
        if (s + XD < mine && s * T + t >= kSince - 1) wait_vm_of<kSince * S::kLoads, kSlice, XD>(kSlices);
        else wait_vm<kSince * S::kLoads>();
      } else {
        // the stages behind it were all issued: of the last slice, those of its further tiles
        if (s + 1 == mine) wait_vm_of<0, S::kLoads, kSince - 1>(T - 1 - t);
        else wait_vm<0>();
      }
      u32x4_t w[S::kSteps];
      uint32_t sc[S::kSteps];
      read_stage<S::kSteps>(w, sc, wa, sa);
#pragma unroll
      for (int h = 0; h < S::kSteps; ++h) {
        // blocks past the end: scale 0 keeps their products with x = 0 finite
        const float f = fp4_scale(slice * KS + 128 * h + 32 * g < a.k ? sc[h] : 0u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bf16x8_t av = widen8(w[h][j], f);
#pragma unroll
          for (int u = 0; u < MT; ++u) {
            bf16x8_t bv;
            __builtin_memcpy(&bv, &x[(h * MT + u) * 4 + j], 16);
            acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv, acc[t][u], 0, 0, 0);
          }
        }
      }
    }
    if (++sslot == XD + 1) sslot = 0;
  }
  // The waves' sums: lane (g, i) of tile (t, u) holds weight rows 4g .. 4g + 3 of x row i.  A thread adds whole
  // lanes of eight waves and writes four outputs.  (Two tiles at a time by single floats: 64 rows of the 24576 x 4096
  // gate / up weight 5 us in this end, 27.5 in all.)
  floatx4_t* const red = reinterpret_cast<floatx4_t*>(lds);
  const bool quads = (a.out_st & 3) == 0 && ((uintptr_t)a.out & 7) == 0 && (a.n & 3) == 0;
#pragma unroll
  for (int t0 = 0; t0 < T; t0 += TR) {
    const int tiles = T - t0 < TR ? T - t0 : TR;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TR; ++t)
      if (t < tiles) {
#pragma unroll
        for (int u = 0; u < MT; ++u) red[((wave * TR + t) * MT + u) * 64 + lane] = acc[t0 + t < T ? t0 + t : 0][u];
      }
    __syncthreads();
    for (int e = threadIdx.x; e < tiles / P * MT * 64; e += kWaves * 64) {
      const int at = e & 63, u = (e >> 6) % MT, p = (e >> 6) / MT;
      const int n = n0 + (t0 / P + p) * 16 + 4 * (at >> 4), m = u * 16 + (at & 15);
      if (n >= a.n || m >= a.m) continue;
      floatx4_t v = {0.f, 0.f, 0.f, 0.f}, up = v;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        v += red[((w * TR + p * P) * MT + u) * 64 + at];
        if constexpr (SILU) up += red[((w * TR + p * P + 1) * MT + u) * 64 + at];
      }
      if (pa.parts != nullptr) {
        float* to = pa.parts + blockIdx.y * pa.part_size + (int64_t)m * (P * a.n) + n;
        if (quads) {
          *reinterpret_cast<floatx4_t*>(to) = v;
          if constexpr (SILU) *reinterpret_cast<floatx4_t*>(to + a.n) = up;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < a.n) {
              to[r] = v[r];
              if constexpr (SILU) to[a.n + r] = up[r];
            }
        }
        continue;
      }
      if constexpr (SILU) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = silu_mul(v[r], up[r]);
      }
      bf16_t* o = a.out + (int64_t)m * a.out_st + n;
      if (quads) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < a.n) o[r] = (bf16_t)f32_to_bf16(v[r]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// More rows than that are bound by the matrix units (200 rows of a 51200 x 5120
// weight: 105 GFLOP against 139 MB), and x is worth sharing: a workgroup takes
// 64 NT weight rows and up to 224 rows of x, eight waves as 2 halves of x by 4
// of the weight.  Along K the weight comes in steps of 128 values (whole
// 64-byte pieces of its rows), several of them ahead since they come from HBM;
// x, from L2, in half steps, so that the LDS it leaves holds those.  The two
// halves of the waves, one of each on every SIMD, take turns: between two
// barriers one reads its operands and then runs its products, the other runs
// the products of what it read before and then reads, so that the matrix units
// and LDS work at once: 200 rows of a 51200 x 5120 weight in 119 us, 880
// TFLOP/s.  (All waves in step, reading and multiplying together, 129 us.  The
// products alone take 79, the loads and reads alone 84.  Weight loads are not
// non-temporal: a step takes half a line, and 133 us then.)  Where the tiles give too few workgroups, K is split
// and a second kernel adds the fp32 parts.

// The operands of a half step in one asm block with one wait: of N column
// tiles (16 rows of 128 bytes apart) both substeps, of NT row tiles (16 rows of
// 64 bytes apart) two words of codes and the scale byte.  The scales of even and
// odd tiles have their own address: gate and up rows need not start alike
// within a dword.
#define XV_XR(j, u) "ds_read_b128 %[x" #j #u "], %[a" #j "] offset:2048*" #u "\n\t"
#define XV_XO(j, u) [x##j##u] "=&v"(x[j][u])
#define XV_XR2 XV_XR(0, 0) XV_XR(0, 1) XV_XR(1, 0) XV_XR(1, 1)
#define XV_XO2 XV_XO(0, 0), XV_XO(0, 1), XV_XO(1, 0), XV_XO(1, 1)
#define XV_XR3 XV_XR2 XV_XR(0, 2) XV_XR(1, 2)
#define XV_XO3 XV_XO2, XV_XO(0, 2), XV_XO(1, 2)
#define XV_XR4 XV_XR3 XV_XR(0, 3) XV_XR(1, 3)
#define XV_XO4 XV_XO3, XV_XO(0, 3), XV_XO(1, 3)
#define XV_XR5 XV_XR4 XV_XR(0, 4) XV_XR(1, 4)
#define XV_XO5 XV_XO4, XV_XO(0, 4), XV_XO(1, 4)
#define XV_XR6 XV_XR5 XV_XR(0, 5) XV_XR(1, 5)
#define XV_XO6 XV_XO5, XV_XO(0, 5), XV_XO(1, 5)
#define XV_XR7 XV_XR6 XV_XR(0, 6) XV_XR(1, 6)
#define XV_XO7 XV_XO6, XV_XO(0, 6), XV_XO(1, 6)
#define XV_WR(t, e) "ds_read_b64 %[w" #t "], %[wa] offset:1024*" #t "\n\t" "ds_read_u8 %[s" #t "], %[s" #e "a] offset:128*" #t "\n\t"
#define XV_WO(t) [w##t] "=&v"(w[t]), [s##t] "=&v"(s[t])
#define XV_WR1 XV_WR(0, 0)
#define XV_WO1 XV_WO(0)
#define XV_WR2 XV_WR1 XV_WR(1, 1)
#define XV_WO2 XV_WO1, XV_WO(1)
#define XV_WR4 XV_WR2 XV_WR(2, 0) XV_WR(3, 1)
#define XV_WO4 XV_WO2, XV_WO(2), XV_WO(3)
#define XV_HALF(N, T)                                                                                               \
  if constexpr (MU == N && NT == T) {                                                                               \
    __asm__ __volatile__(XV_WR##T XV_XR##N "s_waitcnt lgkmcnt(0)"                                                   \
                         : XV_WO##T, XV_XO##N                                                                       \
                         : [wa] "v"(wa), [s0a] "v"(sa0), [s1a] "v"(sa1), [a0] "v"(xa[0]), [a1] "v"(xa[1])           \
                         : "memory");                                                                               \
  }
#define XV_HALVES(N) XV_HALF(N, 1) XV_HALF(N, 2) XV_HALF(N, 4)
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <int MU, int NT>
XV_INLINE void read_half(u32x4_t (&x)[2][MU], u32x2_t (&w)[NT], uint32_t (&s)[NT], const uint32_t (&xa)[2], uint32_t wa,
                         uint32_t sa0, uint32_t sa1) {
  static_assert(MU >= 2 && MU <= kMaxM && (NT == 1 || NT == 2 || NT == 4), "tiles of a wave");
  XV_HALVES(2) XV_HALVES(3) XV_HALVES(4) XV_HALVES(5) XV_HALVES(6) XV_HALVES(7)
}

template <int NT, int MTW, bool SILU>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp4_tile_kernel(Fp4PartArgs ta) {
  const Fp4GemmArgs& a = ta.g;
  constexpr int BM = 32 * MTW, BN = 64 * NT;
  constexpr int kXB = BM * 128;                // bytes of a half step of x
  constexpr int kWB = BN * 64 + BN * 8;        // of a step of the weight; scale rows have windows of two dwords
  constexpr int kLds = 163840;
  constexpr int DX = MTW <= 5 ? 4 : 3;         // half steps of x in LDS, and steps of the weight
  constexpr int DW = (kLds - DX * kXB) / kWB < 8 ? (kLds - DX * kXB) / kWB : 8;
  static_assert(DW >= 3, "two steps of the weight in flight");
  // Waves 0 .. 3 fetch the weight, 4 .. 7 x: loads return in order within a
  // wave, so that one that fetched both would wait with every half step of x for
  // weight steps it does not need yet.
  constexpr int kXQ = MTW, kWQ = NT, kSQ = (NT + 1) / 2;  // LDS-DMA instructions of a wave and half step, or step
  __shared__ __attribute__((aligned(16))) char lds[DX * kXB + DW * kWB];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int nw = wave & 3, mw = wave >> 2;
  const int n0 = blockIdx.x * (SILU ? BN / 2 : BN), m0 = blockIdx.y * BM;
  const int blocks = a.k / kFp4Block, steps = (a.k + 127) / 128;
  const int s0 = blockIdx.z * ta.per, s1 = min(steps, s0 + ta.per);
  // weight row of the workgroup's row R (SILU: 16 gate and 16 up rows of the same outputs in turn), clamped
  auto wrow = [&](int R) {
    const int t = R >> 4, o = min(n0 + (SILU ? t >> 1 : t) * 16 + (R & 15), a.n - 1);
    return (int64_t)o + (SILU && (t & 1) ? a.n : 0);
  };
  const uintptr_t s_base = reinterpret_cast<uintptr_t>(a.s);
  const uintptr_t s_last = (s_base + (uint64_t)((SILU ? 2 * (int64_t)a.n : a.n) - 1) * a.s_st + blocks - 1) & ~(uintptr_t)3;
  const uint32_t base = (uint32_t)reinterpret_cast<uintptr_t>(lds), wbase = base + DX * kXB;
  floatx4_t acc[NT][MTW];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MTW; ++u) acc[t][u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  // this lane's operands within the buffers; a row's scale bytes start where in its window: the same 16 rows
  // on, but not for gate and up rows
  const uint32_t xoff[2] = {(uint32_t)((mw * MTW * 16 + i) * 128 + (((2 * g) ^ swz8p(i)) << 4)),
                            (uint32_t)((mw * MTW * 16 + i) * 128 + (((2 * g + 1) ^ swz8p(i)) << 4))};
  uint32_t soff[2], woff[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    soff[t] = (uint32_t)(BN * 64 + (nw * NT * 16 + i) * 8 + (g >> 1)) +
              (uint32_t)((s_base + (uint64_t)(wrow((nw * NT + t) * 16 + i) * a.s_st)) & 3);
    woff[t] = (uint32_t)((nw * NT * 16 + i) * 64 + (((2 * t + (g >> 1)) ^ swz4(i)) << 4) + 8 * (g & 1));  // half step t
  }

  // Half step 2s + H: lane (g, i) takes values 16g .. + 15 of its row, half of scale block 2 H + g / 2.
  auto read = [&](auto count, auto parity, u32x4_t (&x)[2][decltype(count)::value], u32x2_t (&w)[NT], uint32_t (&sc)[NT], int s,
                  int xslot, int wslot) {
    constexpr int MU = decltype(count)::value, H = decltype(parity)::value;
    const uint32_t xb = base + xslot * kXB, wb = wbase + wslot * kWB;
    const uint32_t xa[2] = {xb + xoff[0], xb + xoff[1]};
    read_half<MU, NT>(x, w, sc, xa, wb + woff[H], wb + soff[0] + 2 * H, wb + soff[1] + 2 * H);
    if (128 * s + 64 * (H + 1) > a.k) {  // the last half steps: blocks past the end
      if (128 * s + 64 * H + 16 * g >= a.k) {  // whole blocks: a lane's 16 values lie inside or outside
#pragma unroll
        for (int u = 0; u < MU; ++u) { x[0][u] = u32x4_t{0, 0, 0, 0}; x[1][u] = u32x4_t{0, 0, 0, 0}; }
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t] = 0u;  // keeps the products with x = 0 finite
      }
    }
  };
  auto multiply = [&](auto count, const u32x4_t (&x)[2][decltype(count)::value], const u32x2_t (&w)[NT], const uint32_t (&sc)[NT]) {
    constexpr int MU = decltype(count)::value;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const bf16x8_t av = widen8(w[t][j], fp4_scale(sc[t]));
#pragma unroll
        for (int u = 0; u < MU; ++u) {
          bf16x8_t bv;
          __builtin_memcpy(&bv, &x[j][u], 16);
          acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv, acc[t][u], 0, 0, 0);
        }
      }
  };
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> odd{};
  // Every step has two barriers: past one, what its half step reads has arrived and nobody reads the half step
  // before any more.  Loads of steps past the end of the range repeat its last: every step issues the same.

  // Waves 0 .. 3: fetch the weight; read, then multiply.
  auto run_w = [&](auto count) {
    constexpr int MU = decltype(count)::value;
    const int wr = lane >> 2, wpiece = (lane & 3) ^ swz4(wr);
    const uint8_t* from[kWQ];  // instruction q: the 16-row tile 4q + nw
    uint32_t row[kWQ];
#pragma unroll
    for (int q = 0; q < kWQ; ++q) {
      from[q] = a.w + wrow(16 * (4 * q + nw)) * a.w_st;
      row[q] = (uint32_t)(wrow(16 * (4 * q + nw) + wr) - wrow(16 * (4 * q + nw))) * (uint32_t)a.w_st;
    }
    uintptr_t ssrc[kSQ];
#pragma unroll
    for (int q = 0; q < kSQ; ++q)  // (64 rows: two waves repeat the others)
      ssrc[q] = s_base + (uint64_t)(wrow((32 * (4 * q + nw) + (lane >> 1)) % BN) * a.s_st);
    auto issue = [&](int s_at, int slot) {
      const int s = min(s_at, s1 - 1);
      char* buf = lds + DX * kXB + slot * kWB;
      const uint32_t piece = 16 * (uint32_t)min(4 * s + wpiece, blocks - 1);  // past the end: any valid one
#pragma unroll
      for (int q = 0; q < kWQ; ++q)
        __builtin_amdgcn_global_load_lds((global_cptr)(from[q] + (size_t)(row[q] + piece)), (lds_void*)(buf + 1024 * (4 * q + nw)),
                                         16, 0, 0);
#pragma unroll
      for (int q = 0; q < kSQ; ++q) {
        const uintptr_t src = min(((ssrc[q] + 4 * s) & ~(uintptr_t)3) + 4 * (lane & 1), s_last);
        __builtin_amdgcn_global_load_lds((global_cptr)src, (lds_void*)(buf + BN * 64 + (256 * (4 * q + nw)) % (BN * 8)), 4, 0, 0);
      }
    };
#pragma unroll
    for (int d = 0; d < DW - 1; ++d) issue(s0 + d, d);
    u32x4_t x[2][MU];
    u32x2_t w[NT];
    uint32_t sc[NT];
    int xslot = 0, wslot = 0;
    for (int s = s0; s < s1; ++s) {
      wait_vm<(DW - 2) * (kWQ + kSQ)>();
      __builtin_amdgcn_s_barrier();
      issue(s + DW - 1, wslot == 0 ? DW - 1 : wslot - 1);
      read(count, even, x, w, sc, s, xslot, wslot);
      multiply(count, x, w, sc);
      xslot = xslot + 1 == DX ? 0 : xslot + 1;
      __builtin_amdgcn_s_barrier();
      read(count, odd, x, w, sc, s, xslot, wslot);
      multiply(count, x, w, sc);
      xslot = xslot + 1 == DX ? 0 : xslot + 1;
      wslot = wslot + 1 == DW ? 0 : wslot + 1;
    }
  };
  // Waves 4 .. 7: fetch x; multiply what the last half step read, then read.
  auto run_x = [&](auto count) {
    constexpr int MU = decltype(count)::value;
    // instruction q: 8 rows of 128 bytes
    const char* const from = reinterpret_cast<const char*>(a.x + (int64_t)m0 * a.x_st);
    uint32_t row[kXQ];
    int piece[kXQ];
#pragma unroll
    for (int q = 0; q < kXQ; ++q) {
      const int r = 8 * (4 * q + nw) + (lane >> 3);
      row[q] = 2 * (uint32_t)min(r, a.m - 1 - m0) * (uint32_t)a.x_st;
      piece[q] = 8 * ((lane & 7) ^ swz8p(r & 15));
    }
    auto issue = [&](int h_at, int slot) {
      const int h = min(h_at, 2 * s1 - 1);
#pragma unroll
      for (int q = 0; q < kXQ; ++q) {
        const uint32_t at = row[q] + 2 * (uint32_t)min(64 * h + piece[q], a.k - 8);  // past the end: any valid piece
        __builtin_amdgcn_global_load_lds((global_cptr)(from + (size_t)at), (lds_void*)(lds + slot * kXB + 1024 * (4 * q + nw)), 16,
                                         0, 0);
      }
    };
#pragma unroll
    for (int d = 0; d < DX - 1; ++d) issue(2 * s0 + d, d);
    u32x4_t x[2][MU];
    u32x2_t w[NT];
    uint32_t sc[NT];
#pragma unroll
    for (int u = 0; u < MU; ++u) { x[0][u] = u32x4_t{0, 0, 0, 0}; x[1][u] = u32x4_t{0, 0, 0, 0}; }
#pragma unroll
    for (int t = 0; t < NT; ++t) { w[t] = u32x2_t{0, 0}; sc[t] = 0u; }
    int xslot = 0, wslot = 0;
    for (int s = s0; s < s1; ++s) {
      wait_vm<(DX - 2) * kXQ>();
      __builtin_amdgcn_s_barrier();
      issue(2 * s + DX - 1, xslot == 0 ? DX - 1 : xslot - 1);
      multiply(count, x, w, sc);
      read(count, even, x, w, sc, s, xslot, wslot);
      xslot = xslot + 1 == DX ? 0 : xslot + 1;
      wait_vm<(DX - 2) * kXQ>();
      __builtin_amdgcn_s_barrier();
      issue(2 * s + DX, xslot == 0 ? DX - 1 : xslot - 1);
      multiply(count, x, w, sc);
      read(count, odd, x, w, sc, s, xslot, wslot);
      xslot = xslot + 1 == DX ? 0 : xslot + 1;
      wslot = wslot + 1 == DW ? 0 : wslot + 1;
    }
    multiply(count, x, w, sc);
  };
  if (s0 < s1) {
    if (mw == 0) run_w(std::integral_constant<int, MTW>{});
    else if (m0 + (2 * MTW - 1) * 16 < a.m) run_x(std::integral_constant<int, MTW>{});
    else run_x(std::integral_constant<int, MTW - 1>{});  // the second half may have one column tile fewer
    wait_vm<0>();  // nothing still writes LDS when the workgroup ends
  }
  // lane (g, i) of tile (t, u): weight rows 4g .. 4g + 3 of x row i
  const bool quads = (a.out_st & 3) == 0 && ((uintptr_t)a.out & 7) == 0 && (a.n & 3) == 0;
#pragma unroll
  for (int u = 0; u < MTW; ++u) {
    const int m = m0 + (mw * MTW + u) * 16 + i;
    if (m >= a.m) continue;
#pragma unroll
    for (int t = 0; t < NT; t += SILU ? 2 : 1) {
      const int n = n0 + (SILU ? (nw * NT + t) >> 1 : nw * NT + t) * 16 + 4 * g;
      if (ta.parts != nullptr) {
        float* p = ta.parts + blockIdx.z * ta.part_size + (int64_t)m * (SILU ? 2 * a.n : a.n) + n;
#pragma unroll
        for (int e = 0; e < (SILU ? 2 : 1); ++e) {
          const floatx4_t v = acc[t + e][u];
          if (quads) {
            if (n < a.n) *reinterpret_cast<floatx4_t*>(p + (e ? a.n : 0)) = v;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n + r < a.n) p[(e ? a.n : 0) + r] = v[r];
          }
        }
      } else {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = acc[t][u][r];
          if constexpr (SILU) v[r] = silu_mul(v[r], acc[t + 1][u][r]);
        }
        bf16_t* o = a.out + (int64_t)m * a.out_st + n;
        if (quads) {
          if (n < a.n) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < a.n) o[r] = (bf16_t)f32_to_bf16(v[r]);
        }
      }
    }
  }
}

// The sum of the parts of a split product, four outputs per thread where rows
// are whole fours (QUAD), else one.
template <bool SILU, bool QUAD>
__global__ __launch_bounds__(256) void fp4_sum_kernel(Fp4PartArgs ta, int parts) {
  const Fp4GemmArgs& a = ta.g;
  constexpr int V = QUAD ? 4 : 1;
  const int per = a.n / V;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int m = (int)(idx / per), n = (int)(idx - (int64_t)m * per) * V;
  if (m >= a.m) return;
  const float* p = ta.parts + (int64_t)m * (SILU ? 2 * a.n : a.n) + n;
  float v[V], up[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = up[e] = 0.f;
  auto add = [&](float (&to)[V], const float* from) {
    if constexpr (QUAD) {
      const floatx4_t f = *reinterpret_cast<const floatx4_t*>(from);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] += f[e];
    } else {
      to[0] += *from;
    }
  };
#pragma unroll 8
  for (int z = 0; z < parts; ++z) {
    add(v, p + z * ta.part_size);
    if constexpr (SILU) add(up, p + z * ta.part_size + a.n);
  }
  if constexpr (SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = silu_mul(v[e], up[e]);
  }
  bf16_t* o = a.out + (int64_t)m * a.out_st + n;
  if constexpr (QUAD) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  else *o = (bf16_t)f32_to_bf16(v[0]);
}

template <bool SILU>
void launch_sum(const Fp4PartArgs& pa, int parts, hipStream_t stream) {
  const Fp4GemmArgs& a = pa.g;
  if ((a.out_st & 3) == 0 && ((uintptr_t)a.out & 7) == 0 && (a.n & 3) == 0)
    fp4_sum_kernel<SILU, true><<<(unsigned)(((int64_t)a.m * a.n / 4 + 255) / 256), 256, 0, stream>>>(pa, parts);
  else
    fp4_sum_kernel<SILU, false><<<(unsigned)(((int64_t)a.m * a.n + 255) / 256), 256, 0, stream>>>(pa, parts);
}

template <int MT, int XR, int KS, int XD, int T, bool SILU>
void launch(const Fp4PartArgs& pa, dim3 grid, hipStream_t stream) {
  // scale rows that start at multiples of 4 bytes have narrower windows
  if (((uintptr_t)pa.g.s | (uint64_t)pa.g.s_st) & 3)
    fp4_gemm_kernel<MT, XR, KS, XD, T, SILU, true><<<grid, kWaves * 64, 0, stream>>>(pa);
  else fp4_gemm_kernel<MT, XR, KS, XD, T, SILU, false><<<grid, kWaves * 64, 0, stream>>>(pa);
}

// One tile a workgroup takes a new slice of x with every stage: as many in
// flight (XD) as stages, in shorter slices where 16 rows of x would not fit.
template <int MT, int XR, int KS1, int XD1, int KS, bool SILU>
void launch_tiles(const Fp4GemmArgs& a, float* ws, hipStream_t stream) {
  const int rows = SILU ? 2 * a.n : a.n;
  const ShortPlan p = short_plan(a.m, rows, a.k, SILU);
  const int slices = p.tiles == 1 ? (a.k + KS1 - 1) / KS1 : (a.k + KS - 1) / KS, outs = p.tiles / (SILU ? 2 : 1) * 16;
  const Fp4PartArgs pa = {a, p.parts > 1 ? ws : nullptr, (int64_t)a.m * rows, (slices + p.parts - 1) / p.parts};
  const dim3 grid((unsigned)((a.n + outs - 1) / outs), (unsigned)p.parts);
  switch (p.tiles) {
    case 1: if constexpr (!SILU) launch<MT, XR, KS1, XD1, 1, SILU>(pa, grid, stream); break;
    case 2: launch<MT, XR, KS, 1, 2, SILU>(pa, grid, stream); break;
    case 4: launch<MT, XR, KS, 1, 4, SILU>(pa, grid, stream); break;
    default: launch<MT, XR, KS, 1, 6, SILU>(pa, grid, stream); break;
  }
  if (p.parts > 1) launch_sum<SILU>(pa, p.parts, stream);
}

template <int NT, bool SILU>
void launch_tile(const Fp4PartArgs& ta, int mtw, dim3 grid, hipStream_t stream) {
  constexpr int threads = kWaves * 64;
  switch (mtw) {
    case 3: fp4_tile_kernel<NT, 3, SILU><<<grid, threads, 0, stream>>>(ta); break;
    case 4: fp4_tile_kernel<NT, 4, SILU><<<grid, threads, 0, stream>>>(ta); break;
    case 5: fp4_tile_kernel<NT, 5, SILU><<<grid, threads, 0, stream>>>(ta); break;
    case 6: fp4_tile_kernel<NT, 6, SILU><<<grid, threads, 0, stream>>>(ta); break;
    default: fp4_tile_kernel<NT, 7, SILU><<<grid, threads, 0, stream>>>(ta); break;
  }
}

template <bool SILU>
void dispatch_tile(const Fp4GemmArgs& a, float* ws, hipStream_t stream) {
  const int rows = SILU ? 2 * a.n : a.n, steps = (a.k + 127) / 128;
  const TilePlan p = tile_plan(a.m, rows, a.k, SILU);
  const Fp4PartArgs ta = {a, p.parts > 1 ? ws : nullptr, (int64_t)a.m * rows, (steps + p.parts - 1) / p.parts};
  const dim3 grid((unsigned)((rows + 64 * p.nt - 1) / (64 * p.nt)), (unsigned)((a.m + 32 * p.mtw - 1) / (32 * p.mtw)),
                  (unsigned)p.parts);
  if (p.nt == 4) launch_tile<4, SILU>(ta, p.mtw, grid, stream);
  else if (p.nt == 2) launch_tile<2, SILU>(ta, p.mtw, grid, stream);
  else if constexpr (!SILU) launch_tile<1, SILU>(ta, p.mtw, grid, stream);
  if (p.parts > 1) launch_sum<SILU>(ta, p.parts, stream);
}

template <bool SILU>
void dispatch(const Fp4GemmArgs& a, float* ws, hipStream_t stream) {
  if (a.m <= 8) launch_tiles<1, 8, 256, 3, 256, SILU>(a, ws, stream);
  else if (a.m <= 16) launch_tiles<1, 16, 128, 3, 256, SILU>(a, ws, stream);
  else if (a.m <= 32) launch_tiles<2, 32, 128, 1, 128, SILU>(a, ws, stream);
  else if (a.m <= 48) launch_tiles<3, 48, 128, 1, 128, SILU>(a, ws, stream);
  else if (a.m <= kShort) launch_tiles<4, 64, 128, 1, 128, SILU>(a, ws, stream);
  else dispatch_tile<SILU>(a, ws, stream);
}

}  // namespace

extern "C" size_t xv_mxfp4_gemm_workspace_size(int m, int n, int k, int silu_mul) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const int parts = m <= kShort ? short_plan(m, n, k, silu_mul != 0).parts : tile_plan(m, n, k, silu_mul != 0).parts;
  return parts > 1 ? (size_t)parts * m * n * sizeof(float) : 0;
}

extern "C" int xv_mxfp4_gemm(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* w_scale,
                             int64_t scale_stride, void* out, int64_t out_stride, int m, int n, int k, int silu_mul,
                             void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (m < 0 || n <= 0 || k <= 0 || k % kFp4Block || (silu_mul && n % 2)) return (int)hipErrorInvalidValue;
  if (!x || !w || !w_scale || !out || !xv_al16(x) || !xv_al16(w) || !xv_st8(x_stride) || w_stride & 15 ||
      (m > 1 && x_stride < k) || w_stride < k / 2 || scale_stride < k / kFp4Block || (uintptr_t)out & 1 ||
      (m > 1 && out_stride < (silu_mul ? n / 2 : n)))
    return (int)hipErrorInvalidValue;
  // 32-bit offsets within a tile, rows that round up; a grid of fewer than 2^32 threads (such weights have 96 or 256
  // rows to a workgroup of 512)
  if (m > 65535 * 64 || n > (1 << 29) || w_stride > (1 << 25) || scale_stride > (1 << 27) || (m > 1 && x_stride > (1 << 22)))
    return (int)hipErrorInvalidValue;
  if (m == 0) return 0;
  if (workspace_bytes < xv_mxfp4_gemm_workspace_size(m, n, k, silu_mul) || (uintptr_t)workspace & 15)
    return (int)hipErrorInvalidValue;
  const Fp4GemmArgs a = {(const bf16_t*)x, m > 1 ? x_stride : k, (const uint8_t*)w, w_stride, (const uint8_t*)w_scale, scale_stride,
                         (bf16_t*)out, out_stride, m, silu_mul ? n / 2 : n, k};
  silu_mul ? dispatch<true>(a, (float*)workspace, stream) : dispatch<false>(a, (float*)workspace, stream);
  XV_CHECK_LAUNCH();
  return 0;
}
