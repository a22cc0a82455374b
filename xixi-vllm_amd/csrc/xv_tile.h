// 64-key K and V tiles in LDS as the prefill and tree attention kernels read
// them: their layout, and a wave's operands for 32 rows on
// v_mfma_f32_32x32x16_bf16.
#pragma once
#include "xv_common.h"

namespace {

constexpr int kD = 128;
constexpr int kKeys = 64;                  // keys per tile
constexpr int kTile = kKeys * kD * 2;      // bytes of one K (or V) tile
constexpr int kBuf = 2 * kTile;            // K then V

typedef float floatx16_t __attribute__((ext_vector_type(16)));

// 16-byte chunk c of row r sits at slot c ^ swz(r) of the row's 256 bytes.
XV_INLINE int swz_k(int r) { return r & 15; }
// V^T reads: a 32-lane group reads 4 rows x 4 chunks (one 64-byte d-tile):
// chunk 4n + j of row r sits at slot 4(n ^ (r & 3)) + j, 16 distinct slots.
XV_INLINE int swz_v(int r) { return (r & 3) << 2; }

// Per-lane LDS addresses, fixed for the whole kernel; tile, buffer and row
// offsets go into the instructions' immediate offsets.
//   K A-operand of d-step s (any key tile mt): row l%32 (+32mt), d-chunk 2s + l/32.
//   V^T A-operand of d-tile n: rows 4(l/32) + (l%16)/4 (+16ks + 8half),
//   chunk 4n + 2((l/16)%2) + (l%4)/2, 8-byte half l%2 -- swizzled slot
//   4(n ^ row%4) + chunk%4.
struct LdsAddr {
  uint32_t k[8];
  uint32_t v[4];
};
XV_INLINE LdsAddr lds_addr(const char* lds, int lane) {
  LdsAddr a;
  const uint32_t base = (uint32_t)reinterpret_cast<uintptr_t>(lds);
  const int l32 = lane & 31, h = lane >> 5, q = lane >> 4, i = lane & 15;
#pragma unroll
  for (int s = 0; s < 8; ++s) a.k[s] = base + l32 * 256 + (((2 * s + h) ^ swz_k(l32)) << 4);
  const int row = 4 * h + (i >> 2);
  const int cl = 2 * (q & 1) + ((i & 3) >> 1);
#pragma unroll
  for (int n = 0; n < 4; ++n) a.v[n] = base + kTile + row * 256 + (((4 * n + cl) ^ swz_v(row)) << 4) + 8 * (i & 1);
  return a;
}

// All 16 K A-operands of a tile (kf[8mt + s]) in two asm blocks: the reads
// are issued together and only the first eight are waited for; k_wait_rest
// completes the other eight (passed through it, so nothing reads them
// earlier).
template <int PAR>
XV_INLINE void read_k16(bf16x8_t (&kf)[16], const LdsAddr& ad) {
  __asm__ __volatile__(
      "ds_read_b128 %0, %16 offset:%24\n\t"
      "ds_read_b128 %1, %17 offset:%24\n\t"
      "ds_read_b128 %2, %18 offset:%24\n\t"
      "ds_read_b128 %3, %19 offset:%24\n\t"
      "ds_read_b128 %4, %20 offset:%24\n\t"
      "ds_read_b128 %5, %21 offset:%24\n\t"
      "ds_read_b128 %6, %22 offset:%24\n\t"
      "ds_read_b128 %7, %23 offset:%24\n\t"
      "ds_read_b128 %8, %16 offset:%25\n\t"
      "ds_read_b128 %9, %17 offset:%25\n\t"
      "ds_read_b128 %10, %18 offset:%25\n\t"
      "ds_read_b128 %11, %19 offset:%25\n\t"
      "ds_read_b128 %12, %20 offset:%25\n\t"
      "ds_read_b128 %13, %21 offset:%25\n\t"
      "ds_read_b128 %14, %22 offset:%25\n\t"
      "ds_read_b128 %15, %23 offset:%25\n\t"
      "s_waitcnt lgkmcnt(8)"
      : "=&v"(kf[0]), "=&v"(kf[1]), "=&v"(kf[2]), "=&v"(kf[3]), "=&v"(kf[4]), "=&v"(kf[5]), "=&v"(kf[6]),
        "=&v"(kf[7]), "=&v"(kf[8]), "=&v"(kf[9]), "=&v"(kf[10]), "=&v"(kf[11]), "=&v"(kf[12]), "=&v"(kf[13]),
        "=&v"(kf[14]), "=&v"(kf[15])
      : "v"(ad.k[0]), "v"(ad.k[1]), "v"(ad.k[2]), "v"(ad.k[3]), "v"(ad.k[4]), "v"(ad.k[5]), "v"(ad.k[6]),
        "v"(ad.k[7]), "n"(PAR * kBuf), "n"(PAR * kBuf + 32 * 256)
      : "memory");
}
XV_INLINE void k_wait_rest(bf16x8_t (&kf)[16]) {
  __asm__ __volatile__("s_waitcnt lgkmcnt(0)"
                       : "+v"(kf[8]), "+v"(kf[9]), "+v"(kf[10]), "+v"(kf[11]), "+v"(kf[12]), "+v"(kf[13]),
                         "+v"(kf[14]), "+v"(kf[15])
                       :
                       : "memory");
}

// V^T A-operands of key-steps KS0, KS0+1 for all four d-tiles: lane l holds
// d = 32n + l%32 and keys 16ks + 4(l/32) + {0..3} and +8 (ks = 2mt + kk), two
// transposed reads of 4 rows each; t[4n + 2(ks-KS0) + half].  The 16 reads are
// issued together and the first eight (d-tiles 0, 1) waited for;
// vt_wait_rest completes the others.
typedef short short4_t __attribute__((ext_vector_type(4)));
template <int PAR, int KS0>
XV_INLINE void read_vt_ks2(short4_t (&t)[16], const LdsAddr& ad) {
  constexpr int o0 = PAR * kBuf + (16 * KS0) * 256;
  __asm__ __volatile__(
      "ds_read_b64_tr_b16 %0, %16 offset:%20\n\t"
      "ds_read_b64_tr_b16 %1, %16 offset:%21\n\t"
      "ds_read_b64_tr_b16 %2, %16 offset:%22\n\t"
      "ds_read_b64_tr_b16 %3, %16 offset:%23\n\t"
      "ds_read_b64_tr_b16 %4, %17 offset:%20\n\t"
      "ds_read_b64_tr_b16 %5, %17 offset:%21\n\t"
      "ds_read_b64_tr_b16 %6, %17 offset:%22\n\t"
      "ds_read_b64_tr_b16 %7, %17 offset:%23\n\t"
      "ds_read_b64_tr_b16 %8, %18 offset:%20\n\t"
      "ds_read_b64_tr_b16 %9, %18 offset:%21\n\t"
      "ds_read_b64_tr_b16 %10, %18 offset:%22\n\t"
      "ds_read_b64_tr_b16 %11, %18 offset:%23\n\t"
      "ds_read_b64_tr_b16 %12, %19 offset:%20\n\t"
      "ds_read_b64_tr_b16 %13, %19 offset:%21\n\t"
      "ds_read_b64_tr_b16 %14, %19 offset:%22\n\t"
      "ds_read_b64_tr_b16 %15, %19 offset:%23\n\t"
      "s_waitcnt lgkmcnt(8)"
      : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3]), "=&v"(t[4]), "=&v"(t[5]), "=&v"(t[6]), "=&v"(t[7]),
        "=&v"(t[8]), "=&v"(t[9]), "=&v"(t[10]), "=&v"(t[11]), "=&v"(t[12]), "=&v"(t[13]), "=&v"(t[14]),
        "=&v"(t[15])
      : "v"(ad.v[0]), "v"(ad.v[1]), "v"(ad.v[2]), "v"(ad.v[3]), "n"(o0), "n"(o0 + 8 * 256), "n"(o0 + 16 * 256),
        "n"(o0 + 24 * 256)
      : "memory");
}
XV_INLINE void vt_wait_rest(short4_t (&t)[16]) {
  __asm__ __volatile__("s_waitcnt lgkmcnt(0)"
                       : "+v"(t[8]), "+v"(t[9]), "+v"(t[10]), "+v"(t[11]), "+v"(t[12]), "+v"(t[13]), "+v"(t[14]),
                         "+v"(t[15])
                       :
                       : "memory");
}
// A-operand of d-tile n, key-step KS0 + j from read_vt_ks2's registers
// (a whole-vector shuffle of the two 64-bit halves: composing it from 16-bit
// elements leaves a no-op bit-field insert per register in front of the MFMA)
typedef short short8_t __attribute__((ext_vector_type(8)));
XV_INLINE bf16x8_t vt_operand(const short4_t (&t)[16], int n, int j) {
  const short8_t r = __builtin_shufflevector(t[4 * n + 2 * j], t[4 * n + 2 * j + 1], 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8_t, r);
}

// Scalar load of a table entry at a wave-uniform index: it does not wait for the tiles in flight.
XV_INLINE int load_index(const int32_t* p) {
  return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}

}  // namespace
