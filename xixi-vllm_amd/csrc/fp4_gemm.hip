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
// A workgroup owns T tiles of 16 weight rows, its eight waves take turns of KS
// values along K (their fp32 sums meet in LDS at the end), and a wave runs its T tiles
// over one slice before the next: x is read once per workgroup and its slice
// waits in registers, while the weight streams through a private LDS ring.
// Both travel by LDS-DMA, whole row segments per instruction.  Direct loads into the
// operand registers, where neighbouring lanes are neighbouring rows, were
// bound by the address unit instead (weights so: a gate / up weight of 24576 x
// 4096 at one row 22 us; x alone so: 8 rows through 4096 x 12288 12.7 us).
#include "xv_decode.h"
#include "xv_fp4.h"
#include "xv_kernels.h"

namespace {

struct Fp4GemmArgs {
  const bf16_t* x; int64_t x_st;
  const uint8_t* w; int64_t w_st;   // codes, bytes between rows
  const uint8_t* s; int64_t s_st;   // scales, bytes between rows
  bf16_t* out; int64_t out_st;
  int m, n, k;                      // n: outputs (of SILU: half the weight's rows)
};

XV_INLINE float silu_mul(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

XV_INLINE bf16x8_t widen8(uint32_t w, float scale) {
  uint32_t o[4];
  fp4x8_to_bf16(w, scale, o);
  bf16x8_t r;
  __builtin_memcpy(&r, o, 16);
  return r;
}

typedef const __attribute__((address_space(1))) void* global_cptr;

constexpr int kWaves = 8;
constexpr int kDepth = 3;  // stages in a wave's ring, kDepth - 1 of them in flight

// One stage: 16 weight rows x KS values.  LDS image: the rows' codes (KS / 2
// bytes each, 16-byte piece j in slot j ^ (row * pieces / 16): the 16 rows of
// an operand read cover all banks once), then a window of SW dwords of each row's
// scale bytes.  A scale row need not start at a multiple of 4 bytes
// (WIDE): the window then starts at the dword that holds the first byte.
template <int KS, bool WIDE>
struct Stage {
  static constexpr int kPieces = KS / 32;               // 16-byte pieces (scale blocks) of a row
  static constexpr int kCodes = 16 * KS / 2;
  static constexpr int kLoads = kCodes / 1024;          // LDS-DMA instructions of the codes
  static constexpr int kRowsPer = 64 / kPieces;         // rows one of them covers
  static constexpr int SW = !WIDE ? KS / 128 : KS == 512 ? 8 : KS / 64;
  static constexpr int kScaleLoads = (16 * SW + 63) / 64;
  static constexpr int kBytes = kCodes + kScaleLoads * 256;
  static constexpr int kOps = kLoads + kScaleLoads;
  static constexpr int kSteps = KS / 128;               // operand loads of 128 values
};

// Pieces of 128 values each from the stage's image (address `a`, the lane's
// pieces at a ^ (64 * step), see below) and their scale bytes, once at most VM
// vector-memory operations are outstanding: one asm block with one wait.
template <int N, int VM>
XV_INLINE void read_stage(u32x4_t (&w)[N], uint32_t (&s)[N], const uint32_t (&wa)[N], uint32_t sa) {
  if constexpr (N == 4) {
    __asm__ __volatile__(
        "s_waitcnt vmcnt(%13)\n\t"
        "ds_read_b128 %0, %8\n\t"
        "ds_read_b128 %1, %9\n\t"
        "ds_read_b128 %2, %10\n\t"
        "ds_read_b128 %3, %11\n\t"
        "ds_read_u8 %4, %12\n\t"
        "ds_read_u8 %5, %12 offset:4\n\t"
        "ds_read_u8 %6, %12 offset:8\n\t"
        "ds_read_u8 %7, %12 offset:12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(s[0]), "=&v"(s[1]), "=&v"(s[2]), "=&v"(s[3])
        : "v"(wa[0]), "v"(wa[1]), "v"(wa[2]), "v"(wa[3]), "v"(sa), "n"(VM)
        : "memory");
  } else if constexpr (N == 2) {
    __asm__ __volatile__(
        "s_waitcnt vmcnt(%7)\n\t"
        "ds_read_b128 %0, %4\n\t"
        "ds_read_b128 %1, %5\n\t"
        "ds_read_u8 %2, %6\n\t"
        "ds_read_u8 %3, %6 offset:4\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(s[0]), "=&v"(s[1])
        : "v"(wa[0]), "v"(wa[1]), "v"(sa), "n"(VM)
        : "memory");
  } else {
    __asm__ __volatile__(
        "s_waitcnt vmcnt(%4)\n\t"
        "ds_read_b128 %0, %2\n\t"
        "ds_read_u8 %1, %3\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(w[0]), "=&v"(s[0])
        : "v"(wa[0]), "v"(sa), "n"(VM)
        : "memory");
  }
}

// Eight operand reads of x (pairs of 4, `b` apart) in one asm block with one wait.
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
  __asm__ __volatile__("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// MT column tiles of 16 rows of x, XR of them fetched (8: the tile's upper
// half repeats the lower, its outputs are not stored); XD slices of x in LDS.
template <int MT, int XR, int KS, int XD, int T, bool SILU, bool WIDE>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp4_gemm_kernel(Fp4GemmArgs a) {
  using S = Stage<KS, WIDE>;
  constexpr int kXBytes = XR * KS * 2, kXLoads = kXBytes / 1024, kXPieces = KS / 8;
  constexpr int kWave = kDepth * S::kBytes + XD * kXBytes;  // LDS of one wave
  constexpr int TR = SILU ? 2 : 1;                          // tiles summed over the waves at a time
  constexpr int kRed = kWaves * TR * MT * 1024;
  static_assert(kXLoads >= 1 && kWaves * kWave <= 163840 && kRed <= 163840, "LDS of a CU");
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kWave > kRed ? kWaves * kWave : kRed];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (SILU ? T / 2 : T) * 16, m0 = blockIdx.y * (MT * 16);
  char* const ring = lds + wave * kWave;
  char* const xring = ring + kDepth * S::kBytes;
  const int blocks = a.k / kFp4Block;
  const int slices = (a.k + KS - 1) / KS;
  const int mine = slices > wave ? (slices - wave + kWaves - 1) / kWaves : 0;  // slices wave, wave + 8, ...
  const int total = mine * T;                                                   // stages of this wave

  // weight row of operand row r of tile t: SILU has the gate and the up rows of the same outputs in tiles 2p, 2p + 1
  auto wrow = [&](int t, int r) {
    const int o = min(n0 + (SILU ? t >> 1 : t) * 16 + r, a.n - 1);
    return (int64_t)o + (SILU && (t & 1) ? a.n : 0);
  };
  const uint8_t* const s_last = reinterpret_cast<const uint8_t*>(
      (reinterpret_cast<uintptr_t>(a.s) + (uint64_t)((SILU ? 2 * (int64_t)a.n : a.n) - 1) * a.s_st + blocks - 1) & ~(uintptr_t)3);
  // this lane's offsets within a stage of whole rows and blocks
  uint32_t coff[S::kLoads], soff[S::kScaleLoads];
#pragma unroll
  for (int q = 0; q < S::kLoads; ++q) {
    const int row = S::kRowsPer * q + lane / S::kPieces;
    coff[q] = row * (uint32_t)a.w_st + 16 * ((lane % S::kPieces) ^ ((row * S::kPieces) >> 4));
  }
#pragma unroll
  for (int q = 0; q < S::kScaleLoads; ++q) {
    const int at = min(64 * q + lane, 16 * S::SW - 1);
    soff[q] = (at / S::SW) * (uint32_t)a.s_st + 4 * (at % S::SW);
  }
  // LDS-DMA instructions issued so far, and the count when each stage's and slice's last one left: what
  // was issued since may still be in flight when it is waited for
  int ops = 0, wmark[kDepth], xmark[XD];
#pragma unroll
  for (int d = 0; d < kDepth; ++d) wmark[d] = 0;
#pragma unroll
  for (int d = 0; d < XD; ++d) xmark[d] = 0;
  int issued = 0, it = 0, is = wave;  // stages issued; the next one's tile and slice
  auto issue = [&](int slot) {
    char* buf = ring + slot * S::kBytes;
    const int b0 = is * S::kPieces;  // the slice's first block
    const int o0 = n0 + (SILU ? it >> 1 : it) * 16;
    const bool whole = o0 + 16 <= a.n && b0 + S::kPieces <= blocks;
    const int64_t row0 = (int64_t)o0 + (SILU && (it & 1) ? a.n : 0);
    if (whole) {
      const uint8_t* src = a.w + row0 * a.w_st + 16 * (int64_t)b0;
#pragma unroll
      for (int q = 0; q < S::kLoads; ++q)
        __builtin_amdgcn_global_load_lds((global_cptr)(src + coff[q]), (lds_void*)(buf + 1024 * q), 16, 0, kNontemporal);
    } else {
#pragma unroll
      for (int q = 0; q < S::kLoads; ++q) {
        const int row = S::kRowsPer * q + lane / S::kPieces;
        const int piece = (lane % S::kPieces) ^ ((row * S::kPieces) >> 4);
        // rows and blocks past the end: valid ones (not stored, and their x is zero)
        const uint8_t* src = a.w + wrow(it, row) * a.w_st + 16 * (int64_t)min(b0 + piece, blocks - 1);
        __builtin_amdgcn_global_load_lds((global_cptr)src, (lds_void*)(buf + 1024 * q), 16, 0, kNontemporal);
      }
    }
    if (whole && !WIDE) {
      const uint8_t* src = a.s + row0 * a.s_st + b0;
#pragma unroll
      for (int q = 0; q < S::kScaleLoads; ++q)
        __builtin_amdgcn_global_load_lds((global_cptr)(src + soff[q]), (lds_void*)(buf + S::kCodes + 256 * q), 4, 0, 0);
    } else {
#pragma unroll
      for (int q = 0; q < S::kScaleLoads; ++q) {
        const int at = min(64 * q + lane, 16 * S::SW - 1);
        uintptr_t src = (reinterpret_cast<uintptr_t>(a.s) + (uint64_t)(wrow(it, at / S::SW) * a.s_st + b0)) & ~(uintptr_t)3;
        src = min(src + 4 * (at % S::SW), reinterpret_cast<uintptr_t>(s_last));  // dwords that hold a byte of the tensor
        __builtin_amdgcn_global_load_lds((global_cptr)src, (lds_void*)(buf + S::kCodes + 256 * q), 4, 0, 0);
      }
    }
    ++issued;
    ops += S::kOps;
    wmark[slot] = ops;
    if (++it == T) {
      it = 0;
      is += kWaves;
    }
  };
  // Slice `slice` of x: row r's KS values (2 KS bytes, 16-byte piece j in slot j ^ (r % 16)) at r * 2 KS.
  auto issue_x = [&](int slice, int slot) {
#pragma unroll
    for (int q = 0; q < kXLoads; ++q) {
      const int at = 64 * q + lane, row = at / kXPieces, piece = (at % kXPieces) ^ (row & 15);
      const int k = min(slice * KS + 8 * piece, a.k - 8);  // past the end: any valid piece (zeroed below)
      const bf16_t* src = a.x + (int64_t)min(m0 + row, a.m - 1) * a.x_st + k;
      __builtin_amdgcn_global_load_lds((global_cptr)src, (lds_void*)(xring + slot * kXBytes + 1024 * q), 16, 0, 0);
    }
    ops += kXLoads;
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
        at[e] = b + row * (KS * 2) + (((16 * h + 4 * g + (e & 3)) ^ (row & 15)) << 4);
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
    wat[h] = (uint32_t)(i * (KS / 2) + (((4 * h + g) ^ ((i * S::kPieces) >> 4)) << 4));
  int wslot = 0, xslot = 0;  // ring slots of the next stage and slice to use
  if (mine > 0) {
#pragma unroll
    for (int d = 0; d < XD; ++d)
      if (d < mine) issue_x(wave + d * kWaves, d);
#pragma unroll
    for (int d = 0; d < kDepth - 1; ++d)
      if (issued < total) issue(d);
  }
  for (int s = 0; s < mine; ++s) {
    const int slice = wave + s * kWaves;
    {
      int since = ops;
#pragma unroll
      for (int d = 0; d < XD; ++d)
        if (d == xslot) since = ops - xmark[d];
      constexpr int kFull = XD > 1 ? XD * S::kOps + (XD - 1) * kXLoads : (T < kDepth ? T : kDepth - 1) * S::kOps;
      constexpr int kFirst = (kDepth - 1) * S::kOps + (XD - 1) * kXLoads;  // the first slice: the first loads of all
      if (since >= kFull) wait_vm<kFull>();
      else if (kFirst < kFull && since >= kFirst) wait_vm<kFirst>();
      else wait_vm<0>();
      take_x(slice, xslot);
      if (s + XD < mine) issue_x(slice + XD * kWaves, xslot);
      if (++xslot == XD) xslot = 0;
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if (issued < total) issue(wslot == 0 ? kDepth - 1 : wslot - 1);
      const uint32_t b = (uint32_t)reinterpret_cast<uintptr_t>(ring + wslot * S::kBytes);
      uint32_t wa[S::kSteps];
#pragma unroll
      for (int h = 0; h < S::kSteps; ++h) wa[h] = b + wat[h];
      uint32_t m4 = 0;  // where in its first dword the row's scale bytes start
      if constexpr (WIDE) m4 = (uint32_t)((reinterpret_cast<uintptr_t>(a.s) + (uint64_t)(wrow(t, i) * a.s_st + slice * S::kPieces)) & 3);
      const uint32_t sa = b + S::kCodes + i * (4 * S::SW) + m4 + g;
      int since = ops;
#pragma unroll
      for (int d = 0; d < kDepth; ++d)
        if (d == wslot) since = ops - wmark[d];
      if (++wslot == kDepth) wslot = 0;
      u32x4_t w[S::kSteps];
      uint32_t sc[S::kSteps];
      constexpr int kTwo = (kDepth - 1) * S::kOps;
      constexpr int kOne = kTwo + kXLoads, kBoth = kTwo + 2 * kXLoads;  // with the x slices issued since
      if (T == 1 && since >= kBoth) read_stage<S::kSteps, kBoth>(w, sc, wa, sa);
      else if (since >= kOne) read_stage<S::kSteps, kOne>(w, sc, wa, sa);
      else if (since >= kTwo) read_stage<S::kSteps, kTwo>(w, sc, wa, sa);
      else read_stage<S::kSteps, 0>(w, sc, wa, sa);
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
  }
  // the waves' sums: lane (g, i) of tile (t, u) holds weight rows 4g + r of x row i
  float* red = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int t0 = 0; t0 < T; t0 += TR) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TR; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u)
        *reinterpret_cast<floatx4_t*>(&red[((wave * TR + t) * MT + u) * 256 + lane * 4]) = acc[t0 + t][u];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * 256; e += kWaves * 64) {
      const int o = e & 15, m = e >> 4;  // output within the tile, x row
      const int at = (m >> 4) * 256 + (o >> 2) * 64 + (m & 15) * 4 + (o & 3);
      const int n = n0 + (t0 / TR) * 16 + o;
      if (n >= a.n || m0 + m >= a.m) continue;
      float v = 0.f, up = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        v += red[(w * TR * MT) * 256 + at];
        if constexpr (SILU) up += red[((w * TR + 1) * MT) * 256 + at];
      }
      a.out[(int64_t)(m0 + m) * a.out_st + n] = (bf16_t)f32_to_bf16(SILU ? silu_mul(v, up) : v);
    }
  }
}

template <int MT, int XR, int KS, int XD, int T, bool SILU>
void launch(const Fp4GemmArgs& a, hipStream_t stream) {
  constexpr int outs = (SILU ? T / 2 : T) * 16;
  const dim3 grid((unsigned)((a.n + outs - 1) / outs), (unsigned)((a.m + MT * 16 - 1) / (MT * 16)));
  // scale rows that start at multiples of 4 bytes have narrower windows
  if (((uintptr_t)a.s | (uint64_t)a.s_st) & 3) fp4_gemm_kernel<MT, XR, KS, XD, T, SILU, true><<<grid, kWaves * 64, 0, stream>>>(a);
  else fp4_gemm_kernel<MT, XR, KS, XD, T, SILU, false><<<grid, kWaves * 64, 0, stream>>>(a);
}

// Tiles per workgroup: the fewest turns of the chip (one workgroup per CU),
// each as long as its tiles plus its start and end, about one and a half tiles.
template <bool SILU>
int tiles_per_group(int n) {
  const int tiles = (n + 15) / 16 * (SILU ? 2 : 1);
  int best = SILU ? 2 : 1;
  double cost = 1e30;
  for (int t : {1, 2, 4, 6}) {
    if (SILU && t % 2) continue;
    const int groups = (tiles + t - 1) / t;
    const double c = ((groups + 255) / 256) * (t + 1.5);
    if (c <= cost) { cost = c; best = t; }
  }
  return best;
}

// One tile a workgroup takes a new slice of x with every stage: as many in
// flight (XD) as stages, in shorter slices where 16 rows of x would not fit.
template <int MT, int XR, int KS1, int XD1, int KS, bool SILU>
void launch_tiles(const Fp4GemmArgs& a, hipStream_t stream) {
  switch (tiles_per_group<SILU>(a.n)) {
    case 1: if constexpr (!SILU) launch<MT, XR, KS1, XD1, 1, SILU>(a, stream); break;
    case 2: launch<MT, XR, KS, 1, 2, SILU>(a, stream); break;
    case 4: launch<MT, XR, KS, 1, 4, SILU>(a, stream); break;
    default: launch<MT, XR, KS, 1, 6, SILU>(a, stream); break;
  }
}

template <bool SILU>
void dispatch(const Fp4GemmArgs& a, hipStream_t stream) {
  if (a.m <= 8) launch_tiles<1, 8, 256, 3, 256, SILU>(a, stream);
  else if (a.m <= 16) launch_tiles<1, 16, 128, 3, 256, SILU>(a, stream);
  else if (a.m <= 32) launch_tiles<2, 32, 128, 1, 128, SILU>(a, stream);
  else launch_tiles<4, 64, 128, 1, 128, SILU>(a, stream);
}

}  // namespace

extern "C" int xv_mxfp4_gemm(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* w_scale,
                             int64_t scale_stride, void* out, int64_t out_stride, int m, int n, int k, int silu_mul,
                             hipStream_t stream) {
  if (m < 0 || n <= 0 || k <= 0 || k % kFp4Block || (silu_mul && n % 2)) return (int)hipErrorInvalidValue;
  if (!x || !w || !w_scale || !out || !xv_al16(x) || !xv_al16(w) || !xv_st8(x_stride) || w_stride & 15 ||
      (m > 1 && x_stride < k) || w_stride < k / 2 || scale_stride < k / kFp4Block || (uintptr_t)out & 1 ||
      (m > 1 && out_stride < (silu_mul ? n / 2 : n)))
    return (int)hipErrorInvalidValue;
  if (m > 65535 * 16 || w_stride > (1 << 27) || scale_stride > (1 << 27)) return (int)hipErrorInvalidValue;  // 32-bit offsets
  if (m == 0) return 0;
  const Fp4GemmArgs a = {(const bf16_t*)x, x_stride, (const uint8_t*)w, w_stride, (const uint8_t*)w_scale, scale_stride,
                         (bf16_t*)out, out_stride, m, silu_mul ? n / 2 : n, k};
  silu_mul ? dispatch<true>(a, stream) : dispatch<false>(a, stream);
  XV_CHECK_LAUNCH();
  return 0;
}
