"""KV store by slot mapping (reference ``src/compute/kv_ops.py:35-62``), the
read back of 4-bit pages as bf16 rows, and a step's block tables, slots and
positions from its requests' lengths."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _C
from ._torch_glue import aligned16, call, ptr, require_bf16, require_cuda, stream_of

FP4_PAGES = torch.float4_e2m1fn_x2  # 4-bit pages: two e2m1 codes to a byte
FP4_SCALE = torch.float8_e8m0fnu
FP4_BLOCK = 32  # values that share one scale


def fp4_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, k_block_scale: torch.Tensor | None,
              v_block_scale: torch.Tensor | None) -> tuple[tuple, tuple, tuple[int, int, int, int]]:
    """Check a 4-bit cache: codes [NB, BS, Hkv, D/2] (or [num_slots, Hkv, D/2])
    and their scales [..., D/32], K and V in one layout each.  Returns the C
    ABI's (k, v, page, token, head stride) of the codes and of the scales, and
    the sizes (blocks, block size, heads, head_dim)."""
    if k_block_scale is None or v_block_scale is None:
        raise ValueError("a 4-bit cache needs k_block_scale and v_block_scale")
    if v_cache.dtype != FP4_PAGES or k_block_scale.dtype != FP4_SCALE or v_block_scale.dtype != FP4_SCALE:
        raise TypeError(f"a 4-bit cache holds {FP4_PAGES} codes and {FP4_SCALE} scales, got {v_cache.dtype}, "
                        f"{k_block_scale.dtype}, {v_block_scale.dtype}")
    shape, sshape, st, ss = k_cache.shape, k_block_scale.shape, k_cache.stride(), k_block_scale.stride()
    if v_cache.shape != shape or v_block_scale.shape != sshape or v_cache.stride() != st or v_block_scale.stride() != ss:
        raise ValueError("k_cache and v_cache, and their scales, must share one layout")
    dims = len(shape)
    if (dims not in (3, 4) or sshape[:-1] != shape[:-1] or shape[-1] * 2 != sshape[-1] * FP4_BLOCK or st[-1] != 1
            or ss[-1] != 1):
        raise ValueError(f"codes {tuple(shape)} and scales {tuple(sshape)} are not [..., Hkv, D/2] and [..., Hkv, D/32] "
                         "of unit last stride")
    dev = k_cache.get_device()  # -1 on the CPU
    if dev < 0 or v_cache.get_device() != dev or k_block_scale.get_device() != dev or v_block_scale.get_device() != dev:
        raise RuntimeError("xvllm ops run on the GPU only (HIP kernels), a cache and its scales on one device")
    if dims == 4:
        strides, sstrides, bs = st[:3], ss[:3], shape[1]
    else:
        strides, sstrides, bs = (st[0], 0, st[1]), (ss[0], 0, ss[1]), 1
    return ((k_cache.data_ptr(), v_cache.data_ptr(), *strides),
            (k_block_scale.data_ptr(), v_block_scale.data_ptr(), *sstrides),
            (shape[0], bs, shape[-2], shape[-1] * 2))


def as_int32(t: torch.Tensor) -> torch.Tensor:
    """t as contiguous-enough int32 indexes (t itself where it is that already)."""
    return t if t.dtype == torch.int32 else t.to(torch.int32)


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t [N, Hkv, D] with 16-byte aligned rows of unit stride."""
    if t.stride(-1) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or not aligned16(t):
        return t.clone(memory_format=torch.contiguous_format)  # fresh, aligned allocation
    return t


def _store_fp4(key, value, k_cache, v_cache, slot_mapping, k_block_scale, v_block_scale) -> None:
    require_bf16(key, value)
    codes, scales, (_, bs, hkv, d) = fp4_pages(k_cache, v_cache, k_block_scale, v_block_scale)
    n = slot_mapping.numel()
    if key.shape != (n, hkv, d) or value.shape != (n, hkv, d):
        raise ValueError(f"key {tuple(key.shape)}, value {tuple(value.shape)}: a cache of {hkv} heads of {d} takes "
                         f"[{n}, {hkv}, {d}] for {n} slots")
    dev = k_cache.get_device()
    if key.get_device() != dev or value.get_device() != dev or slot_mapping.get_device() != dev:
        raise RuntimeError("key, value, slot_mapping and the cache must be on one device")
    key, value = _readable(key), _readable(value)
    slots = as_int32(slot_mapping).contiguous()
    call("xv_store_kvcache_fp4", dev, ptr(key), key.stride(0), key.stride(1), ptr(value), value.stride(0),
         value.stride(1), *codes, *scales, bs, ptr(slots), n, hkv, d)


def store_kvcache(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    k_block_scale: torch.Tensor | None = None,
    v_block_scale: torch.Tensor | None = None,
) -> None:
    """k_cache[slot[i]] = key[i]; v_cache[slot[i]] = value[i]; slot -1 is skipped.

    An fp8 cache (torch.float8_e4m3fn, this build's optional pool format)
    stores e4m3fn(key * (1/k_scale)) and e4m3fn(value * (1/v_scale)); the
    scales are ignored for a bf16 cache.

    A 4-bit cache (torch.float4_e2m1fn_x2 codes [NB, BS, Hkv, D/2], OCP MXFP4)
    also takes its scales k_block_scale / v_block_scale (torch.float8_e8m0fnu,
    [NB, BS, Hkv, D/32]): every 32 values of a row are stored with the power of
    two that brings their largest magnitude to 6 (or within 6/7 of it), rounded
    to the nearest code, ties to even; a run with an infinity or NaN reads back
    as NaN.  Slots other than -1 are distinct.

    key/value: [N, Hkv, D].  The kernel reads strided views directly when
    every head row starts 16-byte aligned with a unit last stride (the q/k/v
    views of a fused qkv GEMM output); any other layout is first copied to a
    fresh contiguous tensor, as the reference does for every input
    (kv_ops.py:42-45).  k_cache/v_cache: paged [NB, BS, Hkv, D] views of the
    pool (any strides, written in place) or flat [num_slots, Hkv, D].
    """
    require_cuda(key, value, k_cache, v_cache, slot_mapping)
    if k_cache.dtype == FP4_PAGES:
        _store_fp4(key, value, k_cache, v_cache, slot_mapping, k_block_scale, v_block_scale)
        return
    fp8 = k_cache.dtype == torch.float8_e4m3fn
    require_bf16(key, value, *(() if fp8 else (k_cache, v_cache)))
    if fp8 and v_cache.dtype != torch.float8_e4m3fn:
        raise TypeError("k_cache and v_cache must share one dtype")
    n, num_heads, head_dim = key.shape
    assert slot_mapping.numel() == n
    if head_dim % 8:
        raise ValueError(f"head_dim must be a multiple of 8 (16-byte rows), got {head_dim}")

    key, value = _readable(key), _readable(value)
    kc, vc = k_cache, v_cache
    if kc.stride() != vc.stride() or kc.shape != vc.shape:
        raise ValueError("k_cache and v_cache must share one layout")
    if kc.dim() == 4:  # [NB, BS, Hkv, D]
        assert kc.shape[2] == num_heads and kc.shape[3] == head_dim
        ps, ts, hs, bs = kc.stride(0), kc.stride(1), kc.stride(2), kc.shape[1]
    else:  # [num_slots, Hkv, D]
        kc = kc.view(-1, num_heads, head_dim)
        vc = vc.view(-1, num_heads, head_dim)
        ps, ts, hs, bs = kc.stride(0), 0, kc.stride(1), 1
    slots = slot_mapping if slot_mapping.dtype == torch.int32 else slot_mapping.to(torch.int32)
    slots = slots.contiguous()
    if fp8:
        _C.check(
            _C.lib().xv_store_kvcache_fp8(
                ptr(key), key.stride(0), key.stride(1), ptr(value), value.stride(0), value.stride(1),
                ptr(kc), ptr(vc), ps, ts, hs, bs, ptr(slots), n, num_heads, head_dim,
                float(k_scale), float(v_scale), stream_of(key),
            ),
            "xv_store_kvcache_fp8",
        )
        return
    _C.check(
        _C.lib().xv_store_kvcache(
            ptr(key), key.stride(0), key.stride(1), ptr(value), value.stride(0), value.stride(1),
            ptr(kc), ptr(vc), ps, ts, hs, bs, ptr(slots), n, num_heads, head_dim,
            stream_of(key),
        ),
        "xv_store_kvcache",
    )


def gather_kvcache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    total_tokens: int,
    *,
    k_block_scale: torch.Tensor,
    v_block_scale: torch.Tensor,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
    cu_seqlens_q: torch.Tensor | None = None,
    window: int = 0,
    sink_tokens: int = 0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of whole sequences out of 4-bit pages: rows
    cu_seqlens_k[b] .. cu_seqlens_k[b+1] of the two bf16 [total_tokens, Hkv, D]
    outputs are sequence b's cached tokens 0, 1, ... through block_tables[b]
    (what prefill_attention takes as varlen k and v).  Every 4-bit value times
    its scale is an exact bf16.

    The cache as store_kvcache writes it, [NB, BS, Hkv, D/2] with its scales;
    block_tables int32 [B, max_blocks]; total_tokens = cu_seqlens_k[B], as the
    host knows it.  Rows from cu_seqlens_k[B] on are left as they were (out:
    the two outputs to write into, of total_tokens rows).

    window > 0: for prefill_attention with this window and sink_tokens, whose
    queries are sequence b's last cu_seqlens_q[b+1] - cu_seqlens_q[b] tokens:
    rows of keys that none of them sees are left as they were, and block-table
    entries that hold only such keys are not read."""
    require_cuda(k_cache, v_cache, block_tables, cu_seqlens_k)
    if k_cache.dtype != FP4_PAGES:
        raise TypeError(f"gather_kvcache reads 4-bit pages ({FP4_PAGES}), got {k_cache.dtype}")
    codes, scales, (_, bs, hkv, d) = fp4_pages(k_cache, v_cache, k_block_scale, v_block_scale)
    if k_cache.dim() != 4:
        raise ValueError(f"gather_kvcache needs a paged cache [NB, BS, Hkv, D/2], got {tuple(k_cache.shape)}")
    dev = k_cache.get_device()
    if block_tables.get_device() != dev or cu_seqlens_k.get_device() != dev:
        raise RuntimeError("the cache, block_tables and cu_seqlens_k must be on one device")
    bsz = cu_seqlens_k.shape[0] - 1
    if cu_seqlens_k.dim() != 1 or bsz < 0 or block_tables.dim() != 2 or block_tables.shape[0] < bsz:
        raise ValueError(f"cu_seqlens_k {tuple(cu_seqlens_k.shape)} and block_tables {tuple(block_tables.shape)} "
                         "are not [B + 1] and [B, max_blocks]")
    if total_tokens < 0:
        raise ValueError("total_tokens must not be negative")
    if window or sink_tokens or cu_seqlens_q is not None:
        if not 1 <= window < 1 << 31 or not 0 <= sink_tokens < 1 << 31:
            raise ValueError(f"window {window}, sink_tokens {sink_tokens}: a window is at least 1, sinks and cu_seqlens_q go with "
                             "one, sinks are not negative, both below 2^31")
        if cu_seqlens_q is None or cu_seqlens_q.shape != cu_seqlens_k.shape:
            raise ValueError("a windowed read back needs cu_seqlens_q, as long as cu_seqlens_k")
        if cu_seqlens_q.get_device() != dev:
            raise RuntimeError("cu_seqlens_q must be on the cache's device")
    if out is None:
        ko, vo = torch.empty((2, total_tokens, hkv, d), dtype=torch.bfloat16, device=k_cache.device).unbind(0)
        row = hkv * d
    else:
        ko, vo = out
        require_bf16(ko, vo)
        for t in (ko, vo):
            if (t.shape != (total_tokens, hkv, d) or t.get_device() != dev or t.stride() != ko.stride() or t.stride(2) != 1
                    or t.stride(1) != d or t.stride(0) % 8 or t.stride(0) < hkv * d or not aligned16(t)):
                raise ValueError(f"out: two bf16 [{total_tokens}, {hkv}, {d}] of contiguous, 16-byte aligned rows")
        row = ko.stride(0)
    if total_tokens == 0 or bsz == 0:
        return ko, vo
    bt = as_int32(block_tables)
    if bt.stride(-1) != 1:
        bt = bt.contiguous()
    cu = as_int32(cu_seqlens_k).contiguous()
    if window:
        cuq = as_int32(cu_seqlens_q).contiguous()
        call("xv_window_gather_kv_fp4", dev, *codes, *scales, bs, ptr(bt), bt.stride(0), bt.shape[1], ptr(cuq), ptr(cu), bsz,
             int(total_tokens), hkv, d, int(window), int(sink_tokens), ptr(ko), ptr(vo), row)
        return ko, vo
    call("xv_gather_kv_fp4", dev, *codes, *scales, bs, ptr(bt), bt.stride(0), bt.shape[1], ptr(cu), bsz,
         int(total_tokens), hkv, d, ptr(ko), ptr(vo), row)
    return ko, vo


class StepMaps(NamedTuple):
    cu_seqlens_q: torch.Tensor   # int32 [B + 1]: new tokens before each request
    cu_seqlens_k: torch.Tensor   # int32 [B + 1]: tokens in the cache after the step, before each request
    cache_seqlens: torch.Tensor  # int32 [B]: tokens of each request in the cache after the step
    positions: torch.Tensor      # int64 [total_tokens]
    slot_mapping: torch.Tensor   # int32 [total_tokens], -1: none
    free_head: torch.Tensor      # int32 [1]: the free list's first page after the step
    row_blocks: torch.Tensor     # int32 [B]: blocks of each request's row after the step


MAX_STEP_ROWS = 4096


def step_maps(
    seq_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_pages: torch.Tensor,
    block_size: int,
    total_tokens: int,
    *,
    free_head: torch.Tensor | None = None,
    depths: torch.Tensor | None = None,
    row_blocks: torch.Tensor | None = None,
) -> StepMaps:
    """The maps of a step whose request b has seq_lens[b] tokens in the cache and
    adds new_lens[b] (int32 [B], on the GPU), in one launch and without a look at
    the lengths on the host (which builds the same in Batch.build_decode and
    build_prefill):

    - block_tables int32 [B, max_blocks], in place: each row's blocks from those
      it has to ceil((seq_lens + new_lens) / block_size) are taken from
      free_pages[free_head:] (int32; free_head int32 [1], 0 where None), row after
      row; its other entries stay as they are.  A row has ceil(seq_lens /
      block_size) blocks, or row_blocks (int32 [B]) where that is more: blocks of
      drafted tokens that were rejected stay the row's.  StepMaps.row_blocks are
      the next step's.
    - StepMaps.free_head: free_head and the pages taken; larger than
      len(free_pages) where the list ran out (such blocks get -1).
    - positions and slot_mapping of the new tokens, request after request
      (StepMaps.cu_seqlens_q), total_tokens rows in all, which the host knows:
      rows past the last new token get slot -1 and position 0, tokens past
      total_tokens none.  A token without a page (no block in its row, free list
      run out) gets slot -1, which store_kvcache skips.
    - depths int32 [total_tokens]: the new tokens are nodes of drafted trees, at
      position seq_lens + depth instead of their index (tree_attention).

    The running sums stay below 2^31, and so do the pool's slots."""
    if not 1 <= block_size <= 1 << 30 or not 0 <= total_tokens <= 1 << 30:
        raise ValueError(f"block_size {block_size}, total_tokens {total_tokens}")
    dev = block_tables.get_device()
    rows, i32 = seq_lens.numel(), torch.int32
    if dev < 0 or seq_lens.get_device() != dev or new_lens.get_device() != dev or free_pages.get_device() != dev:
        raise RuntimeError("xvllm ops run on the GPU only (HIP kernels), all operands on one device")
    if seq_lens.dtype != i32 or new_lens.dtype != i32 or free_pages.dtype != i32 or block_tables.dtype != i32:
        raise TypeError(f"lengths, pages and block tables are int32, got {seq_lens.dtype}, {new_lens.dtype}, {free_pages.dtype}, "
                        f"{block_tables.dtype}")
    if (seq_lens.dim() != 1 or new_lens.shape != seq_lens.shape or free_pages.dim() != 1 or rows > MAX_STEP_ROWS
            or not (seq_lens.is_contiguous() and new_lens.is_contiguous() and free_pages.is_contiguous())):
        raise ValueError(f"seq_lens {tuple(seq_lens.shape)}, new_lens {tuple(new_lens.shape)}, free_pages "
                         f"{tuple(free_pages.shape)}: contiguous vectors, as many lengths of each, at most {MAX_STEP_ROWS}")
    if block_tables.dim() != 2:
        raise ValueError(f"block_tables {tuple(block_tables.shape)} is not [{rows}, max_blocks]")
    max_blocks = block_tables.shape[1]
    bt_st, inner = block_tables.stride()
    if block_tables.shape[0] < rows or max_blocks < 1 or (inner != 1 and max_blocks > 1) or (bt_st < max_blocks and rows > 1):
        raise ValueError(f"block_tables {tuple(block_tables.shape)} of strides {block_tables.stride()} is not [{rows}, max_blocks] of "
                         "unit last stride")
    for name, t, n in (("free_head", free_head, 1), ("depths", depths, total_tokens), ("row_blocks", row_blocks, rows)):
        if t is not None:
            if t.dtype != i32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 vector of {n}, got {t.dtype} {tuple(t.shape)}")
            if t.get_device() != dev:
                raise RuntimeError(f"{name} must be on the block tables' device")
    # one allocation: positions (int64), slots, both running sums, the lengths, the rows' blocks, the list's head
    total_tokens = int(total_tokens)
    buf = block_tables.new_empty(3 * total_tokens + total_tokens % 2 * 2 + 4 * rows + 3)
    wide = 2 * total_tokens + total_tokens % 2 * 2  # the slots start 16-byte aligned
    # (unsafe: pieces that autograd does not relate to each other, a microsecond less for these integers)
    pos, slots, cu_q, cu_k, ends, own, head = buf.unsafe_split_with_sizes((wide, total_tokens, rows + 1, rows + 1, rows, rows, 1))
    base = buf.data_ptr()
    at = base + 4 * (wide + total_tokens)
    call("xv_step_maps", dev, seq_lens.data_ptr(), new_lens.data_ptr(), ptr(row_blocks), rows, block_tables.data_ptr(),
         max(bt_st, max_blocks), max_blocks, block_size, free_pages.data_ptr(), free_pages.shape[0], ptr(free_head), ptr(depths),
         total_tokens, at, at + 4 * (rows + 1), at + 8 * (rows + 1), at + 12 * rows + 8, base, base + 4 * wide, at + 16 * rows + 8)
    pos = pos.view(torch.int64)
    return StepMaps(cu_q, cu_k, ends, pos[:total_tokens] if total_tokens % 2 else pos, slots, head, own)
