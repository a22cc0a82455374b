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

// 16 lanes (a DPP row) hold 128 values of one head row, 8 each; the four lanes
// of a 32-value block agree on its scale over DPP.  A workgroup takes 16 tokens
// and kHeads heads, a lane the same place of each, so that its token's slot is
// looked up once and the heads' loads travel together.  (One flat index per 8
// values, with its three divisions, took 10.0 us for 8192 tokens of 8 heads; this
// 9.6 us, 4.4 TB/s.)
constexpr int kTokens = 16, kHeads = 4;
__global__ __launch_bounds__(256) void store_kvcache_fp4_kernel(
    const bf16_t* __restrict__ key, int64_t ks_tok, int64_t ks_head, const bf16_t* __restrict__ value, int64_t vs_tok,
    int64_t vs_head, Fp4Cache cd, const int32_t* __restrict__ slots, int64_t tokens, int heads, int chunks_per_head) {
  const int64_t tok = (int64_t)blockIdx.x * kTokens + (threadIdx.x >> 4);
  const int h0 = blockIdx.y * kHeads;
  if (tok >= tokens) return;
  const int32_t slot = slots[tok];
  if (slot < 0) return;  // padding token (slot -1) writes nothing
  const int page = slot / cd.block_size, t = slot - page * cd.block_size;
  const int64_t dst = (int64_t)page * cd.ps + (int64_t)t * cd.ts, sdst = (int64_t)page * cd.sps + (int64_t)t * cd.sts;
  for (int d8 = threadIdx.x & 15; d8 < chunks_per_head; d8 += 16) {  // whole blocks of 4 lanes: chunks_per_head is a multiple of 4
    Vec8 kv[kHeads], vv[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (h0 + j >= heads) break;
      kv[j] = load_vec8_nt(key + tok * ks_tok + (h0 + j) * ks_head + d8 * 8);
      vv[j] = load_vec8_nt(value + tok * vs_tok + (h0 + j) * vs_head + d8 * 8);
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (h0 + j >= heads) break;
      uint32_t kb, vb;
      const uint32_t kq = quantise_fp4(kv[j], kb), vq = quantise_fp4(vv[j], vb);
      const int64_t at = dst + (h0 + j) * cd.hs + d8 * 4;
      *reinterpret_cast<uint32_t*>(cd.kc + at) = kq;
      *reinterpret_cast<uint32_t*>(cd.vc + at) = vq;
      if ((d8 & 3) == 0) {
        const int64_t sat = sdst + (h0 + j) * cd.shs + (d8 >> 2);
        cd.ks[sat] = (uint8_t)kb;
        cd.vs[sat] = (uint8_t)vb;
      }
    }
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
  const int64_t groups = (num_tokens + kTokens - 1) / kTokens;
  if (groups > INT32_MAX || num_kv_heads > 65535 * kHeads) return (int)hipErrorInvalidValue;
  store_kvcache_fp4_kernel<<<dim3((unsigned)groups, (unsigned)((num_kv_heads + kHeads - 1) / kHeads)), 256, 0, stream>>>(
      (const bf16_t*)key, key_stride_tok, key_stride_head, (const bf16_t*)value, value_stride_tok, value_stride_head,
      cd, slot_mapping, num_tokens, num_kv_heads, head_dim / 8);
  XV_CHECK_LAUNCH();
  return 0;
}

// Read back: row r of the outputs is token r - cu[b] of the sequence b whose
// range of cu holds r.  A workgroup takes kTokens consecutive rows and
// kGatherHeads heads: one lane each finds a row's place in the cache (the
// sequence by bisection, the block id), then 16 lanes widen a head row of 128
// values, 8 of K and of V each (4 bytes in, 16 out), the heads' loads in
// flight together.  Rows past the last sequence (or of blocks past the table's
// width) are left as they are; WIN: those of keys that no query sees (of a prefill
// with a window and sinks, and cu_q its queries) too, their block ids not read.
// Bound by the rows it writes: 16 sequences of 1229 tokens on average, 8 heads
// (81 MB out), with the store of their last 512 before it 28.8 us, of which this
// about 19; three of 20000 to 35000 (306 MB out) 79 us, 6.1 TB/s, in a replayed
// graph of such calls, 88 us between other work.  The codes are
// loaded as usual, a chunk's store has just written some of them (non-temporal:
// 31.2 us for the first); four heads in place of two: two sequences of 64000 124 us
// against 120, eight: 77 tokens 7.1 us against 6.5.
// Outputs that the last-level cache (256 MB) can hold are written as usual, for
// the prefill that reads them next (189 MB of them and that prefill 721 us against
// 737 non-temporal); larger ones non-temporally (NT: the second case 78 us against
// 104, though with its prefill 2594 against 2575).
constexpr int kGatherHeads = 2;
constexpr int64_t kCached = 256ll << 20;
template <bool NT, bool WIN>
__global__ __launch_bounds__(256) void gather_kv_fp4_kernel(
    Fp4Cache cd, const int32_t* __restrict__ bt, int64_t bt_stride, int max_blocks, const int32_t* __restrict__ cu,
    int batch, int total_rows, int heads, int chunks_per_head, bf16_t* __restrict__ ko, bf16_t* __restrict__ vo,
    int64_t o_st, const int32_t* __restrict__ cu_q, int window, int sinks) {
  __shared__ int64_t src[kTokens], ssrc[kTokens];  // a row's codes and scales in the cache, -1: not written
  const int row0 = blockIdx.x * kTokens, h0 = blockIdx.y * kGatherHeads;
  if (threadIdx.x < kTokens) {
    const int row = row0 + threadIdx.x;
    int64_t at = -1, sat = -1;
    if (row < total_rows && row < cu[batch]) {
      int lo = 0, hi = batch - 1;  // the last sequence that starts at or before the row
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= row) lo = mid; else hi = mid - 1;
      }
      const int t = row - cu[lo];
      const int blk = t / cd.block_size;
      const bool hidden = WIN && window_hides(t, cu[lo + 1] - cu[lo], cu_q[lo + 1] - cu_q[lo], window, sinks);
      if (t >= 0 && blk < max_blocks && !hidden) {
        const int64_t page = bt[(int64_t)lo * bt_stride + blk];
        const int r = t - blk * cd.block_size;
        at = page * cd.ps + (int64_t)r * cd.ts;
        sat = page * cd.sps + (int64_t)r * cd.sts;
      }
    }
    src[threadIdx.x] = at;
    ssrc[threadIdx.x] = sat;
  }
  __syncthreads();
  const int r = threadIdx.x >> 4;
  const int64_t at0 = src[r], sat0 = ssrc[r];
  if (at0 < 0) return;
  for (int d8 = threadIdx.x & 15; d8 < chunks_per_head; d8 += 16) {
    uint32_t kw[kGatherHeads], vw[kGatherHeads], kb[kGatherHeads], vb[kGatherHeads];
#pragma unroll
    for (int j = 0; j < kGatherHeads; ++j) {
      if (h0 + j >= heads) break;
      const int64_t at = at0 + (h0 + j) * cd.hs + d8 * 4, sat = sat0 + (h0 + j) * cd.shs + (d8 >> 2);
      kw[j] = *reinterpret_cast<const uint32_t*>(cd.kc + at);
      vw[j] = *reinterpret_cast<const uint32_t*>(cd.vc + at);
      kb[j] = cd.ks[sat];
      vb[j] = cd.vs[sat];
    }
#pragma unroll
    for (int j = 0; j < kGatherHeads; ++j) {
      if (h0 + j >= heads) break;
      Vec8 k, v;
      fp4x8_to_bf16(kw[j], fp4_scale(kb[j]), k.w);
      fp4x8_to_bf16(vw[j], fp4_scale(vb[j]), v.w);
      const int64_t dst = (int64_t)(row0 + r) * o_st + ((h0 + j) * chunks_per_head + d8) * 8;
      if constexpr (NT) {
        store_vec8_nt(ko + dst, k);
        store_vec8_nt(vo + dst, v);
      } else {
        store_vec8(ko + dst, k);
        store_vec8(vo + dst, v);
      }
    }
  }
}

namespace {

// window 0: all keys (cu_seqlens_q is not looked at)
int gather_kv_fp4(const Fp4Cache& cd, const int32_t* block_tables, int64_t bt_stride, int max_blocks_per_seq,
                  const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int64_t total_tokens,
                  int num_kv_heads, int head_dim, int window, int sink_tokens, void* k_out, void* v_out,
                  int64_t out_stride_tok, hipStream_t stream) {
  if (batch < 0 || total_tokens < 0 || total_tokens > INT32_MAX || num_kv_heads <= 0 || head_dim <= 0 ||
      head_dim % kFp4Block || max_blocks_per_seq < 0 || !cache_ok(cd))
    return (int)hipErrorInvalidValue;
  if (!xv_al16(k_out) || !xv_al16(v_out) || !xv_st8(out_stride_tok) ||
      out_stride_tok < (int64_t)num_kv_heads * head_dim)
    return (int)hipErrorInvalidValue;
  if (batch == 0 || total_tokens == 0) return 0;
  if (num_kv_heads > 65535 * kGatherHeads || (int64_t)num_kv_heads * head_dim > INT32_MAX) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)((total_tokens + kTokens - 1) / kTokens), (unsigned)((num_kv_heads + kGatherHeads - 1) / kGatherHeads));
  const bool large = total_tokens * num_kv_heads * head_dim * 4 > kCached;
  const auto kernel = window > 0 ? (large ? gather_kv_fp4_kernel<true, true> : gather_kv_fp4_kernel<false, true>)
                                 : (large ? gather_kv_fp4_kernel<true, false> : gather_kv_fp4_kernel<false, false>);
  kernel<<<grid, 256, 0, stream>>>(cd, block_tables, bt_stride, max_blocks_per_seq, cu_seqlens_k, batch, (int)total_tokens,
                                   num_kv_heads, head_dim / 8, (bf16_t*)k_out, (bf16_t*)v_out, out_stride_tok, cu_seqlens_q,
                                   window, sink_tokens);
  XV_CHECK_LAUNCH();
  return 0;
}

}  // namespace

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
  return gather_kv_fp4(cd, block_tables, bt_stride, max_blocks_per_seq, nullptr, cu_seqlens_k, batch, total_tokens,
                       num_kv_heads, head_dim, 0, 0, k_out, v_out, out_stride_tok, stream);
}

extern "C" int xv_window_gather_kv_fp4(const void* k_cache, const void* v_cache, int64_t cache_page_stride,
                                       int64_t cache_tok_stride, int64_t cache_head_stride, const void* k_scale,
                                       const void* v_scale, int64_t scale_page_stride, int64_t scale_tok_stride,
                                       int64_t scale_head_stride, int block_size, const int32_t* block_tables,
                                       int64_t bt_stride, int max_blocks_per_seq, const int32_t* cu_seqlens_q,
                                       const int32_t* cu_seqlens_k, int batch, int64_t total_tokens, int num_kv_heads,
                                       int head_dim, int window, int sink_tokens, void* k_out, void* v_out,
                                       int64_t out_stride_tok, hipStream_t stream) {
  if (window < 1 || sink_tokens < 0 || (!cu_seqlens_q && batch > 0)) return (int)hipErrorInvalidValue;
  const Fp4Cache cd = {(uint8_t*)k_cache, (uint8_t*)v_cache, cache_page_stride, cache_tok_stride, cache_head_stride,
                       (uint8_t*)k_scale, (uint8_t*)v_scale, scale_page_stride, scale_tok_stride, scale_head_stride,
                       block_size};
  return gather_kv_fp4(cd, block_tables, bt_stride, max_blocks_per_seq, cu_seqlens_q, cu_seqlens_k, batch, total_tokens,
                       num_kv_heads, head_dim, window, sink_tokens, k_out, v_out, out_stride_tok, stream);
}
