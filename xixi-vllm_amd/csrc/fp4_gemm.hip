// Products of a decode batch with 4-bit (MXFP4) weights on gfx950:
//   out[m, n] = sum_k x[m, k] * code[n, k] * 2^(scale[n, k / 32] - 127)
// and, of a gate / up weight, silu(gate) * up.
//
// A short batch is bound by the weight's bytes (N K / 2 of codes, N K / 32 of
// scales).  v_mfma_f32_16x16x32_bf16 with the weight as operand A: lane (g, i)
// of a step of 128 values takes weight row i's values 32g .. 32g + 31, 16 bytes
// and exactly one scale block, widened to bf16 with the scale applied by the
// conversion (one instruction per pair, exact); operand B is x, column = row
// of x, the same values.  A workgroup owns 16 NT weight rows; its waves take
// turns of 256 values (whole 128-byte lines of the weight) along K and their
// fp32 sums meet in LDS.
#include "xv_fp4.h"
#include "xv_kernels.h"

namespace {

constexpr int kWaves = 8;
constexpr int kStep = 256;  // values along K of one turn of one wave

struct Fp4GemmArgs {
  const bf16_t* x; int64_t x_st;
  const uint8_t* w; int64_t w_st;   // codes, bytes between rows
  const uint8_t* s; int64_t s_st;   // scales, bytes between rows
  bf16_t* out; int64_t out_st;
  int m, n, k;                      // n: outputs (of SILU: half the weight's rows)
};

XV_INLINE float silu_mul(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

template <int MT, int NT, bool SILU>
__global__ __launch_bounds__(kWaves * 64) void fp4_gemm_kernel(Fp4GemmArgs a) {
  __shared__ float red[kWaves][NT * MT * 256];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  // SILU: tiles 2p and 2p + 1 are the gate and the up rows of the same outputs
  constexpr int kOut = (SILU ? NT / 2 : NT) * 16;  // outputs of the workgroup
  const int n0 = blockIdx.x * kOut, m0 = blockIdx.y * (MT * 16);
  const uint8_t* wrow[NT];
  const uint8_t* srow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int o = n0 + (SILU ? (t >> 1) : t) * 16 + i;
    const int64_t row = (int64_t)min(o, a.n - 1) + (SILU && (t & 1) ? a.n : 0);
    wrow[t] = a.w + row * a.w_st + 16 * g;
    srow[t] = a.s + row * a.s_st + g;
  }
  const bf16_t* xrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xrow[t] = a.x + (int64_t)min(m0 + 16 * t + i, a.m - 1) * a.x_st + 32 * g;
  floatx4_t acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave * kStep; k0 < a.k; k0 += kWaves * kStep) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kt = k0 + 128 * h;
      const bool in = kt + 32 * g < a.k;  // whole blocks: a lane's 32 values lie inside or outside
      uint4 w[NT];
      float sc[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[t] = in ? *reinterpret_cast<const uint4*>(wrow[t] + kt / 2) : make_uint4(0, 0, 0, 0);
        sc[t] = in ? fp4_scale(srow[t][kt / kFp4Block]) : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8_t b[MT];
#pragma unroll
        for (int u = 0; u < MT; ++u) {
          const uint4 v = in ? *reinterpret_cast<const uint4*>(xrow[u] + kt + 8 * j) : make_uint4(0, 0, 0, 0);
          __builtin_memcpy(&b[u], &v, 16);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint32_t word = j == 0 ? w[t].x : j == 1 ? w[t].y : j == 2 ? w[t].z : w[t].w;
          uint32_t o[4];
          fp4x8_to_bf16(word, sc[t], o);
          bf16x8_t av;
          __builtin_memcpy(&av, o, 16);
#pragma unroll
          for (int u = 0; u < MT; ++u) acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, b[u], acc[t][u], 0, 0, 0);
        }
      }
    }
  }
  // lane (g, i) of tile (t, u) holds weight rows 4g + r of x row i: float r of lane's four
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u)
      *reinterpret_cast<floatx4_t*>(&red[wave][(t * MT + u) * 256 + lane * 4]) = acc[t][u];
  __syncthreads();
  for (int e = threadIdx.x; e < kOut * MT * 16; e += kWaves * 64) {
    const int o = e % kOut, m = e / kOut;                       // output within the workgroup, x row
    const int at = ((m >> 4) * 256) + ((o & 15) >> 2) * 64 + (m & 15) * 4 + (o & 3);
    const int t = o >> 4;
    float v = 0.f, up = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      v += red[w][(SILU ? 2 * t : t) * MT * 256 + at];
      if (SILU) up += red[w][(2 * t + 1) * MT * 256 + at];
    }
    if (n0 + o < a.n && m0 + m < a.m)
      a.out[(int64_t)(m0 + m) * a.out_st + n0 + o] = (bf16_t)f32_to_bf16(SILU ? silu_mul(v, up) : v);
  }
}

template <int MT, bool SILU>
void launch(const Fp4GemmArgs& a, hipStream_t stream) {
  constexpr int NT = 2;
  const int outs = (SILU ? NT / 2 : NT) * 16;
  fp4_gemm_kernel<MT, NT, SILU><<<dim3((unsigned)((a.n + outs - 1) / outs), (unsigned)((a.m + MT * 16 - 1) / (MT * 16))),
                                  kWaves * 64, 0, stream>>>(a);
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
  if (m > 65535 * 16) return (int)hipErrorInvalidValue;
  if (m == 0) return 0;
  const Fp4GemmArgs a = {(const bf16_t*)x, x_stride, (const uint8_t*)w, w_stride, (const uint8_t*)w_scale, scale_stride,
                         (bf16_t*)out, out_stride, m, silu_mul ? n / 2 : n, k};
  if (m <= 16) silu_mul ? launch<1, true>(a, stream) : launch<1, false>(a, stream);
  else if (m <= 32) silu_mul ? launch<2, true>(a, stream) : launch<2, false>(a, stream);
  else silu_mul ? launch<4, true>(a, stream) : launch<4, false>(a, stream);
  XV_CHECK_LAUNCH();
  return 0;
}
