// A step's maps from its requests' lengths, for gfx950: request b has old[b]
// tokens in the paged cache and adds add[b] of them.
//
//   cu_q, cu_k   running sums of add and of old + add;  ends = old + add
//   block table  row b grows from the blocks it has, max(ceil(old / BS), owned),
//                to ceil((old + add) / BS): page f of the step, counted over
//                the rows in order, is free[head + f]
//   token t      the i-th new one of row b: position old + i (old + depth[t]
//                for a drafted tree), slot page * BS + (old + i) % BS
//
// Bound by latency.  So it is one launch: every workgroup runs the prefix
// sums over the rows itself (into LDS: they cost it less than a second launch
// would), then takes its share of the tokens or of the new pages, each found
// by a binary search there.  A token in a new page takes the page from the free
// list, not from the table, so nothing written here is read here and
// workgroups need no order.
//
// 2.5 us for one request, 6.7 for 180 that decode and 20 chunks of up to 400
// tokens, 7.5 for 256 drafted trees of up to 64 nodes.  The lengths, then the pages
// are two trips to memory in all of them; what the larger ones add are the sums (200
// requests of which one has a token 3.2) and above all the searches, chains of
// dependent LDS reads: a thread makes one for each row that its four tokens lie in,
// one after the other (200 requests of four new tokens each, one search a thread,
// 3.9; of one token each, four searches, 5.3; 16 of them 3.3 and 4.2).
#include "xv_common.h"
#include "xv_kernels.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRows = 4096;   // requests a call: their sums and lengths take 48 KB of a workgroup's LDS
constexpr int kPerThread = 4;    // tokens of a thread: one 16-byte store of slots
constexpr int kMaxGroups = 512;

struct MapsArgs {
  const int32_t* old; const int32_t* add; const int32_t* owned;
  int32_t* bt; int64_t bt_stride; int max_blocks;
  const int32_t* free; int num_free; const int32_t* head;
  const int32_t* depth;
  int32_t* cu_q; int32_t* cu_k; int32_t* ends; int32_t* own;
  int64_t* pos; int32_t* slots; int32_t* next_head;
  int rows, total, block;
  int token_groups;  // workgroups that take tokens; the others take pages
  int shift;  // log2 of block where it is a power of two (a division takes some hundred cycles of this short kernel), else -1
};

XV_INLINE int scan_add(int x) {  // inclusive sum over the wave
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true);
  return x;
}

// The row that holds element i: the largest b with cu[b] <= i (rows without elements are passed over).
XV_INLINE int row_of(const int* cu, int rows, int i) {
  int lo = 0, hi = rows - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(kThreads) void step_maps_kernel(MapsArgs a) {
  extern __shared__ int lds[];
  int* const cq = lds;                     // [rows + 1] new tokens before row b
  int* const cp = lds + a.rows + 1;        // [rows + 1] new pages before row b
  int* const olds = lds + 2 * a.rows + 2;  // [rows] tokens of row b before the step
  __shared__ int part[3][kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool writer = blockIdx.x == 0;
  const int head = a.head ? *a.head : 0;
  auto whole = [&](unsigned tokens) { return (int)(a.shift >= 0 ? tokens >> a.shift : tokens / (unsigned)a.block); };
  auto blocks = [&](int tokens) { return whole((unsigned)tokens + a.block - 1); };
  int carry[3] = {0, 0, 0};  // new tokens, new pages, all tokens
  for (int r0 = 0; r0 < a.rows; r0 += kThreads) {
    const int b = r0 + tid;
    int old = 0, add = 0, owned = 0;
    if (b < a.rows) {
      old = max(a.old[b], 0);
      add = max(a.add[b], 0);
      if (a.owned) owned = a.owned[b];
    }
    const int end = old + add, have = max(blocks(old), owned), own = max(blocks(end), have);
    int s[3] = {scan_add(add), scan_add(own - have), scan_add(end)};
    if (lane == 63)
#pragma unroll
      for (int k = 0; k < 3; ++k) part[k][wave] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int all = 0, before = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) before += part[k][w];
        all += part[k][w];
      }
      s[k] += before + carry[k];
      carry[k] += all;
    }
    __syncthreads();
    if (b < a.rows) {
      cq[b + 1] = s[0];
      cp[b + 1] = s[1];
      olds[b] = old;
      if (writer) {
        a.cu_q[b + 1] = s[0];
        a.cu_k[b + 1] = s[2];
        a.ends[b] = end;
        a.own[b] = own;
      }
    }
  }
  if (tid == 0) {
    cq[0] = cp[0] = 0;
    if (writer) {
      a.cu_q[0] = a.cu_k[0] = 0;
      *a.next_head = head + carry[1];
    }
  }
  __syncthreads();
  // blocks that row b had, where it gets new ones; else all that it needs
  auto blocks_before = [&](int b) { return blocks(olds[b] + cq[b + 1] - cq[b]) - (cp[b + 1] - cp[b]); };
  // where page f of the step is in the free list, nullptr past it
  auto fresh = [&](int f) {
    const int64_t i = (int64_t)head + f;
    return i >= 0 && i < a.num_free ? a.free + i : nullptr;
  };
  if ((int)blockIdx.x >= a.token_groups) {
    const int first = ((int)blockIdx.x - a.token_groups) * kThreads + tid, all = ((int)gridDim.x - a.token_groups) * kThreads;
    for (int f = first; f < carry[1]; f += all) {
      const int b = row_of(cp, a.rows, f);
      const int blk = blocks_before(b) + f - cp[b];
      const int32_t* page = fresh(f);
      if (blk < a.max_blocks) a.bt[(int64_t)b * a.bt_stride + blk] = page ? *page : -1;
    }
    return;
  }
  for (int64_t t0 = ((int64_t)blockIdx.x * kThreads + tid) * kPerThread; t0 < a.total;
       t0 += (int64_t)a.token_groups * kThreads * kPerThread) {
    // first where each token's page is, then the pages together
    const int32_t* from[kPerThread];
    int row[kPerThread], page[kPerThread], depth[kPerThread], old[kPerThread], at[kPerThread];
    int b = 0, next = -1, have = 0;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
      const int t = (int)t0 + e;
      from[e] = nullptr;
      row[e] = old[e] = at[e] = depth[e] = 0;
      if (t >= a.total || t >= carry[0]) continue;  // past the last new token: no slot
      if (t >= next) {
        b = row_of(cq, a.rows, t);
        next = cq[b + 1];
        have = blocks_before(b);
      }
      old[e] = olds[b];
      at[e] = old[e] + t - cq[b];
      if (a.depth) depth[e] = a.depth[t];
      const int blk = whole((unsigned)at[e]);
      row[e] = at[e] - blk * a.block;
      if (blk < a.max_blocks) from[e] = blk >= have ? fresh(cp[b] + blk - have) : a.bt + (int64_t)b * a.bt_stride + blk;
    }
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) page[e] = from[e] ? *from[e] : -1;
    int64_t pos[kPerThread];
    int slot[kPerThread];
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
      const int64_t s = (int64_t)page[e] * a.block + row[e];
      slot[e] = page[e] >= 0 && s <= INT32_MAX ? (int)s : -1;
      pos[e] = a.depth ? (int64_t)old[e] + depth[e] : at[e];
    }
    if (t0 + kPerThread <= a.total) {
      *reinterpret_cast<int4*>(a.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<longlong2*>(a.pos + t0) = make_longlong2(pos[0], pos[1]);
      *reinterpret_cast<longlong2*>(a.pos + t0 + 2) = make_longlong2(pos[2], pos[3]);
    } else {
#pragma unroll
      for (int e = 0; e < kPerThread; ++e)
        if (t0 + e < a.total) {
          a.slots[t0 + e] = slot[e];
          a.pos[t0 + e] = pos[e];
        }
    }
  }
}

}  // namespace

extern "C" int xv_step_maps(const int32_t* seq_lens, const int32_t* new_lens, const int32_t* row_blocks, int rows, int32_t* block_tables,
                            int64_t bt_stride, int max_blocks_per_seq, int block_size, const int32_t* free_pages,
                            int num_free, const int32_t* free_head, const int32_t* depths, int total_tokens,
                            int32_t* cu_seqlens_q, int32_t* cu_seqlens_k, int32_t* cache_seqlens, int32_t* next_row_blocks,
                            int64_t* positions, int32_t* slot_mapping, int32_t* next_free_head, hipStream_t stream) {
  if (rows < 0 || rows > kMaxRows || block_size < 1 || max_blocks_per_seq < 1 || bt_stride < max_blocks_per_seq ||
      num_free < 0 || total_tokens < 0 || total_tokens > (1 << 30))
    return (int)hipErrorInvalidValue;
  if (((uintptr_t)positions | (uintptr_t)slot_mapping) & 15) return (int)hipErrorInvalidValue;
  MapsArgs a;
  a.old = seq_lens; a.add = new_lens; a.owned = row_blocks;
  a.bt = block_tables; a.bt_stride = bt_stride; a.max_blocks = max_blocks_per_seq;
  a.free = free_pages; a.num_free = num_free; a.head = free_head;
  a.depth = depths;
  a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k; a.ends = cache_seqlens; a.own = next_row_blocks;
  a.pos = positions; a.slots = slot_mapping; a.next_head = next_free_head;
  a.rows = rows; a.total = total_tokens; a.block = block_size;
  a.shift = block_size & (block_size - 1) ? -1 : __builtin_ctz(block_size);
  const int64_t per = kThreads * kPerThread;
  const int64_t pages = total_tokens / block_size + rows;  // about as many as there are: the loops take any number
  a.token_groups = (int)min((int64_t)kMaxGroups, (total_tokens + per - 1) / per);
  const int64_t page_groups = max((int64_t)1, min((int64_t)kMaxGroups, (pages + kThreads - 1) / kThreads));
  step_maps_kernel<<<(unsigned)(a.token_groups + page_groups), kThreads, (3 * rows + 2) * sizeof(int), stream>>>(a);
  XV_CHECK_LAUNCH();
  return 0;
}
