// 4-bit (MXFP4) KV pages: the store that quantises new tokens as it writes
// them, and the read back into bf16 rows.
#include "xv_fp4.h"
#include "xv_kernels.h"

namespace {

// Cache codes and scales of K and V, strides in bytes.
struct Fp4Cache {
  uint8_t* kc; uint8_t* vc;
  int64_t ps, ts, hs;
  uint8_t* ks; uint8_t* vs;
  int64_t sps, sts, shs;
  int block_size;
};

bool cache_ok(const Fp4Cache& c) {
  return c.block_size > 0 && c.kc && c.vc && c.ks && c.vs && !(((uintptr_t)c.kc | (uintptr_t)c.vc) & 3) &&
         !((c.ps | c.ts | c.hs) & 3);
}

}  // namespace

// One thread quantises 8 values of K and the matching 8 of V; the four lanes
// of a 32-value block agree on its scale over DPP.
__global__ __launch_bounds__(256) void store_kvcache_fp4_kernel(
    const bf16_t* __restrict__ key, int64_t ks_tok, int64_t ks_head, const bf16_t* __restrict__ value, int64_t vs_tok,
    int64_t vs_head, Fp4Cache cd, const int32_t* __restrict__ slots, int total_chunks, int chunks_per_tok,
    int chunks_per_head) {
  const int idx = blockIdx.x * 256 + threadIdx.x;
  if (idx >= total_chunks) return;  // whole blocks of 4 lanes: total_chunks is a multiple of 4
  const int tok = idx / chunks_per_tok, c = idx - tok * chunks_per_tok;
  const int h = c / chunks_per_head, d8 = c - h * chunks_per_head;
  const Vec8 kv = load_vec8_nt(key + tok * ks_tok + h * ks_head + d8 * 8);
  const Vec8 vv = load_vec8_nt(value + tok * vs_tok + h * vs_head + d8 * 8);
  const int32_t slot = slots[tok];
  uint32_t kb, vb;
  const uint32_t kq = quantise_fp4(kv, kb), vq = quantise_fp4(vv, vb);
  if (slot < 0) return;  // padding token (slot -1) writes nothing
  const int page = slot / cd.block_size, t = slot - page * cd.block_size;
  const int64_t dst = (int64_t)page * cd.ps + (int64_t)t * cd.ts + h * cd.hs + d8 * 4;
  *reinterpret_cast<uint32_t*>(cd.kc + dst) = kq;
  *reinterpret_cast<uint32_t*>(cd.vc + dst) = vq;
  if ((d8 & 3) == 0) {
    const int64_t sdst = (int64_t)page * cd.sps + (int64_t)t * cd.sts + h * cd.shs + (d8 >> 2);
    cd.ks[sdst] = (uint8_t)kb;
    cd.vs[sdst] = (uint8_t)vb;
  }
}

extern "C" int xv_store_kvcache_fp4(const void* key, int64_t key_stride_tok, int64_t key_stride_head,
                                    const void* value, int64_t value_stride_tok, int64_t value_stride_head,
                                    void* k_cache, void* v_cache, int64_t cache_page_stride, int64_t cache_tok_stride,
                                    int64_t cache_head_stride, void* k_scale, void* v_scale, int64_t scale_page_stride,
                                    int64_t scale_tok_stride, int64_t scale_head_stride, int block_size,
                                    const int32_t* slot_mapping, int64_t num_tokens, int num_kv_heads, int head_dim,
                                    hipStream_t stream) {
  const Fp4Cache cd = {(uint8_t*)k_cache, (uint8_t*)v_cache, cache_page_stride, cache_tok_stride, cache_head_stride,
                       (uint8_t*)k_scale, (uint8_t*)v_scale, scale_page_stride, scale_tok_stride, scale_head_stride,
                       block_size};
  if (num_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || head_dim % kFp4Block || !cache_ok(cd))
    return (int)hipErrorInvalidValue;
  if (!xv_al16(key) || !xv_al16(value) || !xv_st8(key_stride_tok) || !xv_st8(key_stride_head) ||
      !xv_st8(value_stride_tok) || !xv_st8(value_stride_head))
    return (int)hipErrorInvalidValue;  // rows move as 16-byte vectors
  if (num_tokens == 0) return 0;
  const int64_t cpt = (int64_t)num_kv_heads * (head_dim / 8);
  if (num_tokens * cpt >= ((int64_t)1 << 31) - 256) return (int)hipErrorInvalidValue;  // 32-bit chunk indices
  const int total = (int)(num_tokens * cpt);
  store_kvcache_fp4_kernel<<<(unsigned)((total + 255) / 256), 256, 0, stream>>>(
      (const bf16_t*)key, key_stride_tok, key_stride_head, (const bf16_t*)value, value_stride_tok, value_stride_head,
      cd, slot_mapping, total, (int)cpt, head_dim / 8);
  XV_CHECK_LAUNCH();
  return 0;
}

// Read back: row r of the outputs is token r - cu[b] of the sequence b whose
// range of cu holds r.  One thread widens 8 values of K and of V.  Rows past
// the last sequence (or of blocks past the table's width) are left as they are.
__global__ __launch_bounds__(256) void gather_kv_fp4_kernel(
    Fp4Cache cd, const int32_t* __restrict__ bt, int64_t bt_stride, int max_blocks, const int32_t* __restrict__ cu,
    int batch, int64_t total_chunks, int chunks_per_tok, int chunks_per_head, bf16_t* __restrict__ ko,
    bf16_t* __restrict__ vo, int64_t o_st) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= total_chunks) return;
  const int row = (int)(idx / chunks_per_tok), c = (int)(idx - (int64_t)row * chunks_per_tok);
  if (row >= cu[batch]) return;
  int lo = 0, hi = batch - 1;  // the last sequence that starts at or before the row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid - 1;
  }
  const int t = row - cu[lo];
  const int blk = t / cd.block_size;
  if (t < 0 || blk >= max_blocks) return;
  const int64_t page = bt[(int64_t)lo * bt_stride + blk];
  const int r = t - blk * cd.block_size;
  const int h = c / chunks_per_head, d8 = c - h * chunks_per_head;
  const int64_t src = page * cd.ps + (int64_t)r * cd.ts + h * cd.hs + d8 * 4;
  const int64_t ssrc = page * cd.sps + (int64_t)r * cd.sts + h * cd.shs + (d8 >> 2);
  const uint32_t kw = *reinterpret_cast<const uint32_t*>(cd.kc + src);
  const uint32_t vw = *reinterpret_cast<const uint32_t*>(cd.vc + src);
  const float kf = fp4_scale(cd.ks[ssrc]), vf = fp4_scale(cd.vs[ssrc]);
  Vec8 k, v;
  fp4x8_to_bf16(kw, kf, k.w);
  fp4x8_to_bf16(vw, vf, v.w);
  const int64_t dst = (int64_t)row * o_st + c * 8;
  store_vec8(ko + dst, k);
  store_vec8(vo + dst, v);
}

extern "C" int xv_gather_kv_fp4(const void* k_cache, const void* v_cache, int64_t cache_page_stride,
                                int64_t cache_tok_stride, int64_t cache_head_stride, const void* k_scale,
                                const void* v_scale, int64_t scale_page_stride, int64_t scale_tok_stride,
                                int64_t scale_head_stride, int block_size, const int32_t* block_tables,
                                int64_t bt_stride, int max_blocks_per_seq, const int32_t* cu_seqlens_k, int batch,
                                int64_t total_tokens, int num_kv_heads, int head_dim, void* k_out, void* v_out,
                                int64_t out_stride_tok, hipStream_t stream) {
  const Fp4Cache cd = {(uint8_t*)k_cache, (uint8_t*)v_cache, cache_page_stride, cache_tok_stride, cache_head_stride,
                       (uint8_t*)k_scale, (uint8_t*)v_scale, scale_page_stride, scale_tok_stride, scale_head_stride,
                       block_size};
  if (batch < 0 || total_tokens < 0 || total_tokens > INT32_MAX || num_kv_heads <= 0 || head_dim <= 0 ||
      head_dim % kFp4Block || max_blocks_per_seq < 0 || !cache_ok(cd))
    return (int)hipErrorInvalidValue;
  if (!xv_al16(k_out) || !xv_al16(v_out) || !xv_st8(out_stride_tok) ||
      out_stride_tok < (int64_t)num_kv_heads * head_dim)
    return (int)hipErrorInvalidValue;
  if (batch == 0 || total_tokens == 0) return 0;
  const int64_t cpt = (int64_t)num_kv_heads * (head_dim / 8), total = total_tokens * cpt;
  const int64_t blocks = (total + 255) / 256;
  if (cpt > INT32_MAX || blocks > INT32_MAX) return (int)hipErrorInvalidValue;
  gather_kv_fp4_kernel<<<(unsigned)blocks, 256, 0, stream>>>(cd, block_tables, bt_stride, max_blocks_per_seq,
                                                             cu_seqlens_k, batch, total, (int)cpt, head_dim / 8,
                                                             (bf16_t*)k_out, (bf16_t*)v_out, out_stride_tok);
  XV_CHECK_LAUNCH();
  return 0;
}
