"""``vllm::attention`` custom op (reference ``src/compute/layers/attention.py:13-143``):
stores this step's K/V at ``slot_mapping`` (kv_ops.store_kvcache), then runs
paged GQA decode attention or varlen causal prefill attention, both as gfx950
HIP kernels.  Same signature (and three optional arguments more), same module-global ``attention_context`` pool
handle, same ``AttnInputs`` record.
"""
from __future__ import annotations

import math
from contextlib import contextmanager
from dataclasses import dataclass
from functools import lru_cache
from typing import NamedTuple, Optional, Sequence

import torch
import torch.nn as nn

from .. import _C
from .._torch_glue import aligned16, call, ptr, require_bf16, require_cuda, stream_of
from ..kv_ops import FP4_PAGES, as_int32, fp4_pages, gather_kvcache, store_kvcache


@dataclass
class CascadePlan:
    """Shared-prefix groups of a decode batch (device int32 tensors): row b's
    first prefix_tokens[b] tokens are its group's shared blocks; group g's
    record group_info[g] is (first index into group_rows, rows, first batch
    row, prefix tokens).  num_groups and max_prefix_blocks fix the prefix
    pass's grid (empty groups allowed)."""
    prefix_tokens: torch.Tensor
    group_info: torch.Tensor
    group_rows: torch.Tensor
    num_groups: int
    max_prefix_blocks: int


@dataclass
class TreePlan:
    """Trees of drafted tokens of a step (device tensors): rows cu_seqlens_q[b]
    .. cu_seqlens_q[b+1] - 1 are sequence b's nodes, the last of its
    cache_seqlens tokens, and row t sees the nodes of mask[t] (tree_attention).
    max_nodes: those of the largest tree at most."""
    cu_seqlens_q: torch.Tensor
    mask: torch.Tensor
    max_nodes: int


class AttnInputs(NamedTuple):
    slot_mapping: torch.Tensor
    is_prefill: bool
    cu_seqlens_q: Optional[torch.Tensor] = None
    cu_seqlens_k: Optional[torch.Tensor] = None
    max_seqlen_q: int = 0
    max_seqlen_k: int = 0
    block_tables: Optional[torch.Tensor] = None
    cache_seqlens: Optional[torch.Tensor] = None
    cascade: Optional[CascadePlan] = None  # decode only: shared-prefix groups (no reference counterpart)
    total_seqlen_k: int = 0  # prefill: the keys of all sequences, cu_seqlens_k's last, where the host knows it
    tree: Optional[TreePlan] = None  # not prefill: the rows are trees of drafted tokens (no reference counterpart)


@dataclass
class AttnMetadata:
    kv_cache: torch.Tensor  # [2, L, NB, BS, Hkv, D]
    # fp8 (e4m3fn) pools only: the dequantisation scales of K and V (this
    # build's optional pool format; the reference's pool holds the model dtype)
    k_scale: float = 1.0
    v_scale: float = 1.0
    # 4-bit pools only (kv_cache [..., D/2] of two codes to a byte): the block scales [2, L, NB, BS, Hkv, D/32]
    block_scale: Optional[torch.Tensor] = None


# Active metadata, innermost context last (the reference keeps one module
# global, attention.py:29-40; a stack gives the same nesting behaviour).
_META_STACK: list[AttnMetadata] = []


@contextmanager
def attention_context(meta: AttnMetadata):
    """Makes `meta.kv_cache` the pool that vllm::attention reads and writes
    for the duration of the block (nesting restores the outer one)."""
    _META_STACK.append(meta)
    try:
        yield meta
    finally:
        _META_STACK.pop()


def kv_scales() -> tuple[float, float]:
    """(k_scale, v_scale) of the active pool (1, 1 for a bf16 pool)."""
    if not _META_STACK:
        raise RuntimeError("vllm::attention needs an active attention_context(AttnMetadata(kv_cache=...))")
    m = _META_STACK[-1]
    return m.k_scale, m.v_scale


def _layer_caches(layer_id: int) -> tuple[torch.Tensor, torch.Tensor]:
    if not _META_STACK:
        raise RuntimeError("vllm::attention needs an active attention_context(AttnMetadata(kv_cache=...))")
    pool = _META_STACK[-1].kv_cache
    return pool[0, layer_id], pool[1, layer_id]


def _layer_scales(layer_id: int) -> dict:
    """The scales of a layer's cache, as store_kvcache and paged_decode_attention take them."""
    ks, vs = kv_scales()
    meta = _META_STACK[-1]
    if meta.kv_cache.dtype != FP4_PAGES:
        return {"k_scale": ks, "v_scale": vs}
    if meta.block_scale is None:
        raise ValueError("a 4-bit pool needs its block scales: AttnMetadata(block_scale=...)")
    return {"k_block_scale": meta.block_scale[0, layer_id], "v_block_scale": meta.block_scale[1, layer_id]}


def _refuse_cascade(k_cache: torch.Tensor) -> None:
    if k_cache.dtype == FP4_PAGES:
        raise TypeError("no cascade decode over 4-bit pages: paged_decode_attention reads them")


_WORKSPACE: dict[tuple[str, int | None], torch.Tensor] = {}


# Workspaces replaced by a larger one stay allocated: a hipGraph captured
# earlier keeps the old pointer and replays onto it.
_RETIRED: list[torch.Tensor] = []


def decode_workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Per-device decode workspace, grown on demand outside graph capture (the
    kernels need no initial contents: partial counts and partials are written
    before they are read).  The size query never decreases with the batch, so
    a decode graph set captured largest bucket first allocates it once; a
    workspace that is outgrown anyway is kept alive for the graphs that hold
    it.  Calls on one device share it: they must be ordered on one stream."""
    key = (device.type, device.index)
    ws = _WORKSPACE.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _RETIRED.append(ws)
        with torch.inference_mode(False):  # a plain tensor: later callers outside inference mode may use it
            ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _WORKSPACE[key] = ws
    return ws


def _q_view(q: torch.Tensor, num_heads: int, head_dim: int) -> tuple[torch.Tensor, int, int]:
    q3 = q.view(q.shape[0], num_heads, head_dim) if q.dim() == 2 else q
    if q3.stride(-1) != 1 or q3.stride(0) % 8 or q3.stride(1) % 8 or not aligned16(q3):
        q3 = q3.clone(memory_format=torch.contiguous_format)  # whole rows may be unaligned too: a fresh allocation
    return q3, q3.stride(0), q3.stride(1)


def _paged_decode_fp4(q, k_cache, v_cache, block_tables, cache_seqlens, hq, hkv, d, softmax_scale, out,
                      k_block_scale, v_block_scale) -> torch.Tensor:
    require_bf16(q)
    codes, scales, (_, bs, heads, dim) = fp4_pages(k_cache, v_cache, k_block_scale, v_block_scale)
    if k_cache.dim() != 4 or heads != hkv or dim != d:
        raise ValueError(f"cache {tuple(k_cache.shape)} is not 4-bit pages [NB, BS, {hkv}, {d} / 2]")
    q3, qs0, qs1 = _q_view(q, hq, d)
    bsz = q3.shape[0]
    if q3.shape[1:] != (hq, d) or block_tables.dim() != 2 or block_tables.shape[0] < bsz or cache_seqlens.numel() < bsz:
        raise ValueError(f"q {tuple(q.shape)}, block_tables {tuple(block_tables.shape)}, cache_seqlens "
                         f"{tuple(cache_seqlens.shape)}: not {hq} heads of {d} with a table row and a length each")
    dev = k_cache.get_device()
    if q.get_device() != dev or block_tables.get_device() != dev or cache_seqlens.get_device() != dev:
        raise RuntimeError("q, the cache, block_tables and cache_seqlens must be on one device")
    bt = as_int32(block_tables)
    max_blocks = bt.shape[1]
    bt_st, inner = bt.stride()
    if inner != 1 or (bsz > 1 and bt_st < max_blocks):
        bt = bt.contiguous()
        bt_st = max_blocks
    sl = as_int32(cache_seqlens).contiguous()
    if out is None:
        out = torch.empty((bsz, hq * d), dtype=q.dtype, device=q.device)
        out_st = hq * d
    elif out.shape != (bsz, hq * d) or out.dtype != q.dtype or out.get_device() != dev or out.stride(-1) != 1:
        raise ValueError(f"out must be bf16 [{bsz}, {hq * d}] of unit last stride on the cache's device")
    else:
        out_st = out.stride(0)
    if bsz == 0:
        return out
    # a workspace of the call's own, from the caching allocator: calls on several streams and captured graphs share none
    ws_bytes = _C.lib().xv_paged_decode_fp4_workspace_size(bsz, hq, hkv)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
    scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    call("xv_paged_decode_attention_fp4", dev, q3.data_ptr(), qs0, qs1, *codes, *scales, bt.data_ptr(),
         max(bt_st, max_blocks), sl.data_ptr(), out.data_ptr(), out_st, ws.data_ptr(), ws_bytes, bsz, hq, hkv, d, bs,
         max_blocks, scale)
    return out


def _windowed(window: int, sink_tokens: int) -> bool:
    """Whether a call has a sliding window (0: none), after checking its sizes."""
    if not window and not sink_tokens:
        return False
    if not 1 <= window < 1 << 31 or not 0 <= sink_tokens < 1 << 31:
        raise ValueError(f"window {window}, sink_tokens {sink_tokens}: a window is at least 1, sinks go with one and are not "
                         "negative, both below 2^31")
    return True


def _hides(window: int, block_tables: torch.Tensor | None, k_cache: torch.Tensor) -> bool:
    """Whether a window (0: none) may hide a token: one as long as all that a table row has room for hides none."""
    return window > 0 and (block_tables is None or window < block_tables.shape[-1] * k_cache.shape[1])


def _paged_rows(q, k_cache, v_cache, block_tables, cache_seqlens, hq, hkv, d, bsz, out, what):
    """Operands of the attention kernels that take bf16 pages and a workspace
    per call: the C ABI's q, cache, table and length arguments, the output and
    its row stride."""
    require_bf16(q)
    if k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise TypeError(f"{what} reads bf16 pages, got {k_cache.dtype} and {v_cache.dtype}")
    ks, st = k_cache.shape, k_cache.stride()
    if len(ks) != 4 or ks[2] != hkv or ks[3] != d or v_cache.shape != ks or v_cache.stride() != st or st[3] != 1:
        raise ValueError(f"caches {tuple(k_cache.shape)} and {tuple(v_cache.shape)} are not pages [NB, BS, {hkv}, {d}] of one "
                         "layout")
    shape, qs = q.shape, q.stride()
    usual = len(shape) == 2 and shape[1] == hq * d and qs[1] == 1 and not (qs[0] | d) % 8 and aligned16(q)
    if usual:
        q3, qs0, qs1 = q, qs[0], d  # without the cost of a view
    else:
        q3, qs0, qs1 = _q_view(q, hq, d)
        if q3.dim() != 3 or q3.shape[1:] != (hq, d):
            raise ValueError(f"q {tuple(q.shape)} is not rows of {hq} heads of {d}")
    tables = block_tables.shape
    if len(tables) != 2 or tables[0] < bsz or cache_seqlens.dim() != 1 or cache_seqlens.shape[0] < bsz:
        raise ValueError(f"block_tables {tuple(block_tables.shape)}, cache_seqlens {tuple(cache_seqlens.shape)}: not a row and a "
                         f"length for each of {bsz} sequences")
    dev = k_cache.get_device()
    if (dev < 0 or v_cache.get_device() != dev or q.get_device() != dev or block_tables.get_device() != dev
            or cache_seqlens.get_device() != dev):
        raise RuntimeError("xvllm ops run on the GPU only (HIP kernels), q, the cache, block_tables and cache_seqlens on one device")
    bt = as_int32(block_tables)
    max_blocks = tables[1]
    bt_st, inner = bt.stride()
    if inner != 1 or (bsz > 1 and bt_st < max_blocks):
        bt = bt.contiguous()
        bt_st = max_blocks
    sl = as_int32(cache_seqlens).contiguous()
    if out is None:
        out = torch.empty_like(q) if usual and qs[0] == hq * d else q.new_empty((shape[0], hq * d))
        out_st = hq * d
    elif out.shape != (shape[0], hq * d) or out.dtype != q.dtype or out.get_device() != dev or out.stride(-1) != 1:
        raise ValueError(f"out must be bf16 [{shape[0]}, {hq * d}] of unit last stride on the cache's device")
    else:
        out_st = out.stride(0)
    head = (q3.data_ptr(), qs0, qs1, k_cache.data_ptr(), v_cache.data_ptr(), *st[:3], bt.data_ptr(), max(bt_st, max_blocks),
            sl.data_ptr())
    return dev, head, (q3, bt, sl), out, out_st, ks[1], max_blocks


@lru_cache(maxsize=1024)
def _rows_workspace_size(batch: int, max_nodes: int, hq: int, hkv: int) -> int:
    return _C.lib().xv_tree_attention_workspace_size(batch, max_nodes, hq, hkv)


def _window_decode(q, k_cache, v_cache, block_tables, cache_seqlens, hq, hkv, d, softmax_scale, out, window,
                   sink_tokens) -> torch.Tensor:
    bsz = q.shape[0]
    dev, head, keep, out, out_st, bs, max_blocks = _paged_rows(q, k_cache, v_cache, block_tables, cache_seqlens, hq, hkv, d, bsz,
                                                               out, "a windowed decode")
    if bsz == 0:
        return out
    ws_bytes = _rows_workspace_size(bsz, 1, hq, hkv)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8)
    scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    call("xv_window_decode_attention", dev, *head, out.data_ptr(), out_st, ws.data_ptr(), ws_bytes, bsz, hq, hkv, d, bs,
         max_blocks, window, sink_tokens, scale)
    return out


MAX_TREE_NODES = 1024


def tree_masks(parents: Sequence[int]) -> tuple[torch.Tensor, torch.Tensor]:
    """(mask int64 [n, words], depths int32 [n]) of a tree of drafted tokens by
    its nodes' parents (a node before its children; -1: a child of the last
    token before the tree): a node sees its ancestors and itself (tree_attention),
    and its position is the context's length plus its depth (step_maps)."""
    n = len(parents)
    rows, depths = [], []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"node {i}: parent {p} is not -1 or a node before it")
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
        depths.append(depths[p] + 1 if p >= 0 else 0)
    words = max(1, -(-n // 64))
    signed = lambda w: w - (1 << 64) if w >> 63 else w
    mask = [[signed(r >> 64 * w & (1 << 64) - 1) for w in range(words)] for r in rows]
    return torch.tensor(mask, dtype=torch.int64).view(n, words), torch.tensor(depths, dtype=torch.int32)


def tree_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    cache_seqlens: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    tree_mask: torch.Tensor,
    max_seqlen_q: int,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of trees of drafted tokens over the paged cache: q [T, Hq*D] (or
    [T, Hq, D]) -> [T, Hq*D].

    Sequence b holds cache_seqlens[b] tokens (int32 [B]), the last n =
    cu_seqlens_q[b+1] - cu_seqlens_q[b] of them its drafted nodes, whose K and V
    are in the cache already (bf16 pages [NB, BS, Hkv, D]).  Its node i is row
    cu_seqlens_q[b] + i and sees every token before the nodes and node j where
    bit j % 64 of tree_mask[row, j // 64] is set (int64 [T, words] or, up to 64
    nodes, [T]; a node's own bit is set by the caller too: tree_masks).
    max_seqlen_q: nodes of the largest tree, at most 64 * words and 1024.  Rows
    that see nothing are zeros; rows from cu_seqlens_q[B] on are left as they
    are in `out`.  Takes a workspace of its own per call."""
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] < 1:
        raise ValueError(f"cu_seqlens_q {tuple(cu_seqlens_q.shape)} is not [B + 1]")
    bsz = cu_seqlens_q.shape[0] - 1
    dev, head, keep, out, out_st, bs, max_blocks = _paged_rows(q, k_cache, v_cache, block_tables, cache_seqlens, num_qo_heads,
                                                               num_kv_heads, head_dim, bsz, out, "tree attention")
    mask = tree_mask if tree_mask.dim() == 2 else tree_mask.unsqueeze(-1)
    if mask.dtype != torch.int64 or mask.dim() != 2 or mask.shape[0] != q.shape[0] or mask.shape[1] < 1:
        raise ValueError(f"tree_mask {tree_mask.dtype} {tuple(tree_mask.shape)} is not int64 [{q.shape[0]}, words]")
    if mask.get_device() != dev or cu_seqlens_q.get_device() != dev:
        raise RuntimeError("tree_mask and cu_seqlens_q must be on the cache's device")
    words = mask.shape[1]
    if not 0 <= max_seqlen_q <= min(64 * words, MAX_TREE_NODES):
        raise ValueError(f"max_seqlen_q {max_seqlen_q}: {words} mask words hold {64 * words} nodes, a tree at most {MAX_TREE_NODES}")
    if bsz == 0 or max_seqlen_q == 0 or q.shape[0] == 0:
        return out
    if (words > 1 and mask.stride(1) != 1) or mask.stride(0) < words:
        mask = mask.contiguous()
    cu = as_int32(cu_seqlens_q).contiguous()
    ws_bytes = _rows_workspace_size(bsz, max_seqlen_q, num_qo_heads, num_kv_heads)
    ws = q.new_empty(ws_bytes, dtype=torch.uint8)
    scale = 1.0 / math.sqrt(head_dim) if softmax_scale is None else float(softmax_scale)
    call("xv_tree_attention", dev, *head, cu.data_ptr(), mask.data_ptr(), max(mask.stride(0), words), words, out.data_ptr(), out_st,
         ws.data_ptr(), ws_bytes, bsz, max_seqlen_q, num_qo_heads, num_kv_heads, head_dim, bs, max_blocks, scale)
    return out


def paged_decode_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    cache_seqlens: torch.Tensor,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
    *,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
    k_block_scale: torch.Tensor | None = None,
    v_block_scale: torch.Tensor | None = None,
    window: int = 0,
    sink_tokens: int = 0,
) -> torch.Tensor:
    """Causal decode over the paged cache: q [B, Hq*D] (or [B, Hq, D]),
    k_cache/v_cache [NB, BS, Hkv, D], block_tables int32 [B, max_blocks],
    cache_seqlens int32 [B] (0 = padding row) -> [B, Hq*D].  An fp8 cache
    (torch.float8_e4m3fn, written by store_kvcache with the same scales)
    attends to k_cache * k_scale and v_cache * v_scale; a 4-bit cache
    (torch.float4_e2m1fn_x2 [NB, BS, Hkv, D/2]) to its codes times the block
    scales k_block_scale / v_block_scale [NB, BS, Hkv, D/32].

    window > 0: the query sees the last `window` tokens of its sequence, itself
    among them, and the first sink_tokens; block-table entries that hold none of
    these are not read.  Caches are bf16, unless the window is as long as all
    that the table has room for and so hides nothing.

    The 4-bit and the windowed form take a workspace of their own per call; the
    others share one per device (decode_workspace)."""
    if _windowed(window, sink_tokens) and (k_cache.dtype == torch.bfloat16 or _hides(window, block_tables, k_cache)):
        return _window_decode(q, k_cache, v_cache, block_tables, cache_seqlens, num_qo_heads, num_kv_heads, head_dim,
                              softmax_scale, out, window, sink_tokens)
    if k_cache.dtype == FP4_PAGES:
        return _paged_decode_fp4(q, k_cache, v_cache, block_tables, cache_seqlens, num_qo_heads, num_kv_heads, head_dim,
                                 softmax_scale, out, k_block_scale, v_block_scale)
    require_cuda(q, k_cache, v_cache, block_tables, cache_seqlens)
    fp8 = k_cache.dtype == torch.float8_e4m3fn
    require_bf16(q, *(() if fp8 else (k_cache, v_cache)))
    if fp8 and v_cache.dtype != torch.float8_e4m3fn:
        raise TypeError("k_cache and v_cache must share one dtype")
    q3, qs0, qs1 = _q_view(q, num_qo_heads, head_dim)
    bsz = q3.shape[0]
    nb, page, hkv, d = k_cache.shape
    assert hkv == num_kv_heads and d == head_dim and v_cache.stride() == k_cache.stride()
    bt = block_tables if block_tables.dtype == torch.int32 else block_tables.to(torch.int32)
    if bt.stride(-1) != 1:
        bt = bt.contiguous()
    sl = cache_seqlens.to(torch.int32).contiguous()
    assert bt.shape[0] >= bsz and sl.shape[0] >= bsz
    if out is None:
        out = torch.empty((bsz, num_qo_heads * head_dim), dtype=q.dtype, device=q.device)
    L = _C.lib()
    max_blocks = bt.shape[1]
    ws_bytes = L.xv_paged_decode_workspace_size(bsz, num_qo_heads, num_kv_heads, max_blocks, page, head_dim)
    ws = decode_workspace(q.device, ws_bytes)
    scale = 1.0 / math.sqrt(head_dim) if softmax_scale is None else softmax_scale
    if fp8:
        _C.check(
            L.xv_paged_decode_attention_fp8(
                ptr(q3), qs0, qs1, ptr(k_cache), ptr(v_cache), k_cache.stride(0), k_cache.stride(1),
                k_cache.stride(2), ptr(bt), bt.stride(0), ptr(sl), ptr(out), out.stride(0), ptr(ws), ws.numel(),
                bsz, num_qo_heads, num_kv_heads, head_dim, page, max_blocks, float(scale), float(k_scale),
                float(v_scale), stream_of(q),
            ),
            "xv_paged_decode_attention_fp8",
        )
        return out
    _C.check(
        L.xv_paged_decode_attention(
            ptr(q3), qs0, qs1, ptr(k_cache), ptr(v_cache), k_cache.stride(0), k_cache.stride(1),
            k_cache.stride(2), ptr(bt), bt.stride(0), ptr(sl), ptr(out), out.stride(0), ptr(ws), ws.numel(),
            bsz, num_qo_heads, num_kv_heads, head_dim, page, max_blocks, float(scale), stream_of(q),
        ),
        "xv_paged_decode_attention",
    )
    return out


_CASCADE_WS: dict[tuple[str, int | None], torch.Tensor] = {}


def cascade_decode_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    cache_seqlens: torch.Tensor,
    plan: CascadePlan,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
    *,
    k_scale: float = 1.0,
    v_scale: float = 1.0,
) -> torch.Tensor:
    """paged_decode_attention with the shared prefixes of `plan` read once per
    group (xv_cascade_decode_attention, or _fp8 on an fp8 cache with the
    scales of paged_decode_attention).  Same output as the plain decode up
    to fp32 summation order.  Not over 4-bit pages."""
    _refuse_cascade(k_cache)
    require_cuda(q, k_cache, v_cache, block_tables, cache_seqlens, plan.prefix_tokens)
    fp8 = k_cache.dtype == torch.float8_e4m3fn
    require_bf16(q, *(() if fp8 else (k_cache, v_cache)))
    if fp8 and v_cache.dtype != torch.float8_e4m3fn:
        raise TypeError("k_cache and v_cache must share one dtype")
    q3, qs0, qs1 = _q_view(q, num_qo_heads, head_dim)
    bsz = q3.shape[0]
    nb, page, hkv, d = k_cache.shape
    assert hkv == num_kv_heads and d == head_dim and v_cache.stride() == k_cache.stride()
    bt = block_tables if block_tables.dtype == torch.int32 else block_tables.to(torch.int32)
    if bt.stride(-1) != 1:
        bt = bt.contiguous()
    sl = cache_seqlens.to(torch.int32).contiguous()
    if out is None:
        out = torch.empty((bsz, num_qo_heads * head_dim), dtype=q.dtype, device=q.device)
    L = _C.lib()
    max_blocks = bt.shape[1]
    nbytes = L.xv_cascade_decode_workspace_size(bsz, num_qo_heads, num_kv_heads, max_blocks, page, head_dim)
    key = (q.device.type, q.device.index)
    ws = _CASCADE_WS.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _RETIRED.append(ws)  # a recorded graph may still hold it
        with torch.inference_mode(False):  # a plain tensor: later callers outside inference mode may use it
            ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=q.device)
        _CASCADE_WS[key] = ws
    scale = 1.0 / math.sqrt(head_dim) if softmax_scale is None else softmax_scale
    args = (
        ptr(q3), qs0, qs1, ptr(k_cache), ptr(v_cache), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
        ptr(bt), bt.stride(0), ptr(sl), ptr(plan.prefix_tokens), ptr(plan.group_info), ptr(plan.group_rows),
        plan.num_groups, min(plan.max_prefix_blocks, max_blocks), ptr(out), out.stride(0), ptr(ws), ws.numel(),
        bsz, num_qo_heads, num_kv_heads, head_dim, page, max_blocks, float(scale),
    )
    if fp8:
        _C.check(L.xv_cascade_decode_attention_fp8(*args, float(k_scale), float(v_scale), stream_of(q)),
                 "xv_cascade_decode_attention_fp8")
    else:
        _C.check(L.xv_cascade_decode_attention(*args, stream_of(q)), "xv_cascade_decode_attention")
    return out


def _check_prefill(q3, cu_seqlens_q, cu_seqlens_k, hq, hkv, d, k, v, k_cache, v_cache, block_tables) -> None:
    """What the prefill kernels take on trust: one device, a length for every sequence, rows of hq and hkv heads, and
    caches of one layout (they are given one set of strides)."""
    if q3.dim() != 3 or q3.shape[1:] != (hq, d):
        raise ValueError(f"q {tuple(q3.shape)} is not rows of {hq} heads of {d}")
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] < 1 or cu_seqlens_k.dim() != 1 or cu_seqlens_k.shape[0] < cu_seqlens_q.shape[0]:
        raise ValueError(f"cu_seqlens_q {tuple(cu_seqlens_q.shape)} and cu_seqlens_k {tuple(cu_seqlens_k.shape)} are not [B + 1]")
    dev, bsz = q3.get_device(), cu_seqlens_q.shape[0] - 1
    operands = (k, v) if block_tables is None else (k_cache, v_cache, block_tables)
    if any(t is None for t in operands):
        raise ValueError("prefill needs k and v, or k_cache, v_cache and block_tables")
    if any(t.get_device() != dev for t in (cu_seqlens_q, cu_seqlens_k, *operands)):
        raise RuntimeError("xvllm ops run on the GPU only (HIP kernels), all operands on one device")
    if block_tables is None:
        return
    if block_tables.dim() != 2 or block_tables.shape[0] < bsz:
        raise ValueError(f"block_tables {tuple(block_tables.shape)} has no row for each of {bsz} sequences")
    if k_cache.dtype != FP4_PAGES:
        ks, st = k_cache.shape, k_cache.stride()
        if len(ks) != 4 or ks[2] != hkv or ks[3] != d or st[3] != 1 or v_cache.shape != ks or v_cache.stride() != st or v_cache.dtype != k_cache.dtype:
            raise ValueError(f"caches {tuple(ks)} and {tuple(v_cache.shape)} are not pages [NB, BS, {hkv}, {d}] of one type and layout")


def prefill_attention(
    q: torch.Tensor,
    k: torch.Tensor | None,
    v: torch.Tensor | None,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    k_cache: torch.Tensor | None = None,
    v_cache: torch.Tensor | None = None,
    block_tables: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    max_seqlen_k: int = 0,
    kv_scale: tuple[float, float] | None = None,
    k_block_scale: torch.Tensor | None = None,
    v_block_scale: torch.Tensor | None = None,
    total_seqlen_k: int = 0,
    *,
    window: int = 0,
    sink_tokens: int = 0,
) -> torch.Tensor:
    """Varlen causal attention, bottom-right aligned.  With block_tables the
    keys come from the paged cache (cached prefix + this chunk), otherwise
    from k/v rows cu_seqlens_k[b] .. cu_seqlens_k[b+1].  An fp8 paged cache
    needs max_seqlen_k and its (k_scale, v_scale) (default: the active
    attention_context's), a 4-bit one its block scales and total_seqlen_k, the
    keys of all sequences (cu_seqlens_k's last): they are read back as so many
    bf16 rows.  With max_seqlen_k alone room is made for B of the longest run.

    window > 0: a query sees the last `window` keys up to itself and the
    sequence's first sink_tokens (softmax_scale > 0); block-table entries that
    hold no key some query sees are not read."""
    windowed = _windowed(window, sink_tokens)
    if windowed and softmax_scale is not None and not softmax_scale > 0:
        raise ValueError(f"a windowed prefill needs softmax_scale > 0, got {softmax_scale}")
    q3, qs0, qs1 = _q_view(q, num_qo_heads, head_dim)
    require_cuda(q3, cu_seqlens_q, cu_seqlens_k)
    require_bf16(q3)
    _check_prefill(q3, cu_seqlens_q, cu_seqlens_k, num_qo_heads, num_kv_heads, head_dim, k, v, k_cache, v_cache, block_tables)
    bsz = cu_seqlens_q.shape[0] - 1
    cuq = cu_seqlens_q.to(torch.int32).contiguous()
    cuk = cu_seqlens_k[: bsz + 1].to(torch.int32).contiguous()  # it may be a larger batch's buffer
    out = torch.empty((q3.shape[0], num_qo_heads * head_dim), dtype=q.dtype, device=q.device)
    scale = 1.0 / math.sqrt(head_dim) if softmax_scale is None else softmax_scale
    if block_tables is not None and k_cache is not None and k_cache.dtype == FP4_PAGES:
        # 4-bit pages: the sequences' keys and values as varlen bf16 rows (exact), then the dense path
        if max_seqlen_k <= 0 and total_seqlen_k <= 0:
            raise ValueError("prefill over a 4-bit paged cache needs total_seqlen_k (the keys of all sequences) or "
                             "max_seqlen_k (the longest key run)")
        if total_seqlen_k < 0 or (total_seqlen_k and max_seqlen_k > 0 and not max_seqlen_k <= total_seqlen_k <= bsz * max_seqlen_k):
            raise ValueError(f"total_seqlen_k {total_seqlen_k} is not the keys of {bsz} sequences of up to {max_seqlen_k}")
        if k_cache.dim() != 4 or k_cache.shape[2] != num_kv_heads or k_cache.shape[3] * 2 != head_dim:
            raise ValueError(f"cache {tuple(k_cache.shape)} is not 4-bit pages [NB, BS, {num_kv_heads}, {head_dim} / 2]")
        seen = dict(cu_seqlens_q=cuq, window=window, sink_tokens=sink_tokens) if windowed else {}
        kd, vd = gather_kvcache(k_cache, v_cache, block_tables, cuk, int(total_seqlen_k) or bsz * int(max_seqlen_k),
                                k_block_scale=k_block_scale, v_block_scale=v_block_scale, **seen)
        return prefill_attention(q, kd, vd, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, num_qo_heads, num_kv_heads,
                                 head_dim, softmax_scale=softmax_scale, window=window, sink_tokens=sink_tokens)
    if block_tables is not None and k_cache is not None and k_cache.dtype == torch.float8_e4m3fn:
        # fp8 pages: the sequences' keys dequantized into varlen bf16 rows, then the dense path
        k_scale, v_scale = kv_scales() if kv_scale is None else kv_scale
        if max_seqlen_k <= 0:
            raise ValueError("prefill over an fp8 paged cache needs max_seqlen_k (the longest key run)")
        hkv = k_cache.shape[2]
        bt = block_tables.to(torch.int32)
        if bt.stride(-1) != 1:
            bt = bt.contiguous()
        rows = bsz * int(max_seqlen_k)
        kd = torch.empty((max(rows, 1), hkv, head_dim), dtype=torch.bfloat16, device=q.device)
        vd = torch.empty_like(kd)
        pages = (ptr(k_cache), ptr(v_cache), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), ptr(bt), bt.stride(0),
                 k_cache.shape[1])
        rows_out = (float(k_scale), float(v_scale), ptr(kd), ptr(vd), kd.stride(0))
        if windowed:
            call("xv_window_gather_kv_fp8", q3.get_device(), *pages, ptr(cuq), ptr(cuk), bsz, int(max_seqlen_k), hkv, head_dim,
                 int(window), int(sink_tokens), *rows_out)
        else:
            _C.check(_C.lib().xv_gather_kv_fp8(*pages, ptr(cuk), bsz, int(max_seqlen_k), hkv, head_dim, *rows_out,
                                               stream_of(q)), "xv_gather_kv_fp8")
        return prefill_attention(q, kd, vd, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, num_qo_heads, num_kv_heads,
                                 head_dim, softmax_scale=softmax_scale, window=window, sink_tokens=sink_tokens)
    if block_tables is not None:
        require_bf16(k_cache, v_cache)
        bt = block_tables.to(torch.int32)
        if bt.stride(-1) != 1:
            bt = bt.contiguous()
        kd = vd = None
        kvs0 = kvs1 = 0
        kc, vc = k_cache, v_cache
        ps, ts, hs = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
        page = k_cache.shape[1]
        bts = bt.stride(0)
    else:
        k3 = k.view(k.shape[0], num_kv_heads, head_dim) if k.dim() == 2 else k
        v3 = v.view(v.shape[0], num_kv_heads, head_dim) if v.dim() == 2 else v
        if (k3.stride() != v3.stride() or k3.stride(-1) != 1 or k3.stride(0) % 8 or k3.stride(1) % 8
                or not aligned16(k3) or not aligned16(v3)):
            # whole rows may be unaligned too: fresh allocations
            k3, v3 = (t.clone(memory_format=torch.contiguous_format) for t in (k3, v3))
        require_bf16(k3, v3)
        if k3.shape != v3.shape or k3.dim() != 3 or k3.shape[1:] != (num_kv_heads, head_dim):
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} are not rows of {num_kv_heads} heads of {head_dim}")
        kd, vd = k3, v3
        kvs0, kvs1 = k3.stride(0), k3.stride(1)
        kc = vc = bt = None
        ps = ts = hs = bts = 0
        page = 16
    if windowed:
        call("xv_window_prefill_attention", q3.get_device(), ptr(q3), qs0, qs1, ptr(kd), ptr(vd), kvs0, kvs1, ptr(kc), ptr(vc), ps,
             ts, hs, ptr(bt), bts, ptr(cuq), ptr(cuk), ptr(out), out.stride(0), bsz, int(max_seqlen_q), q3.shape[0], num_qo_heads,
             num_kv_heads, head_dim, page, int(window), int(sink_tokens), float(scale))
        return out
    _C.check(
        _C.lib().xv_prefill_attention(
            ptr(q3), qs0, qs1, ptr(kd), ptr(vd), kvs0, kvs1, ptr(kc), ptr(vc), ps, ts, hs, ptr(bt), bts,
            ptr(cuq), ptr(cuk), ptr(out), out.stride(0), bsz, int(max_seqlen_q), num_qo_heads, num_kv_heads,
            head_dim, page, float(scale), stream_of(q),
        ),
        "xv_prefill_attention",
    )
    return out


@torch.library.custom_op("vllm::attention", mutates_args=())
def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    slot_mapping: Optional[torch.Tensor],
    is_prefill: bool,
    cu_seqlens_q: Optional[torch.Tensor],
    cu_seqlens_k: Optional[torch.Tensor],
    max_seqlen_q: int,
    max_seqlen_k: int,
    block_tables: Optional[torch.Tensor],
    cache_seqlens: Optional[torch.Tensor],
    layer_id: int,
    num_qo_heads: int,
    num_kv_heads: int,
    head_dim: int,
    total_seqlen_k: int = 0,
    window: int = 0,
    sink_tokens: int = 0,
) -> torch.Tensor:
    """The reference's arguments and, at their end, AttnInputs' total_seqlen_k
    and the layer's sliding window and sinks (0: none)."""
    k_cache, v_cache = _layer_caches(layer_id)
    k3 = k.view(-1, num_kv_heads, head_dim)
    v3 = v.view(-1, num_kv_heads, head_dim)
    scales = _layer_scales(layer_id)
    if slot_mapping is not None:  # None: this step's K/V are already in the cache (fused store)
        store_kvcache(k3, v3, k_cache, v_cache, slot_mapping, **scales)  # paged view, in place
    if is_prefill:
        if block_tables is not None:
            return prefill_attention(
                q, None, None, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, num_qo_heads, num_kv_heads,
                head_dim, k_cache=k_cache, v_cache=v_cache, block_tables=block_tables, max_seqlen_k=max_seqlen_k,
                total_seqlen_k=total_seqlen_k, window=window, sink_tokens=sink_tokens,
                **(scales if k_cache.dtype == FP4_PAGES else {"kv_scale": kv_scales()}),
            )
        return prefill_attention(
            q, k3, v3, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, num_qo_heads, num_kv_heads, head_dim, window=window,
            sink_tokens=sink_tokens,
        )
    return paged_decode_attention(
        q, k_cache, v_cache, block_tables, cache_seqlens, num_qo_heads, num_kv_heads, head_dim, window=window,
        sink_tokens=sink_tokens, **scales,
    )


@attention.register_fake
def _attention_fake(
    q, k, v, slot_mapping, is_prefill, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
    max_seqlen_k, block_tables, cache_seqlens, layer_id, num_qo_heads,
    num_kv_heads, head_dim, total_seqlen_k=0, window=0, sink_tokens=0,
):
    return torch.empty((q.shape[0], num_qo_heads * head_dim), dtype=q.dtype, device=q.device)


def kv_cache_of(layer_id: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(k_cache, v_cache) [NB, BS, Hkv, D] views of the active pool for a layer."""
    return _layer_caches(layer_id)


class Attention(nn.Module):
    """window > 0: a query sees the last `window` tokens of its sequence, itself
    among them, and the first sink_tokens; else every one before it."""

    def __init__(self, num_heads: int, head_dim: int, num_kv_heads: int, layer_id: int = 0, window: int = 0,
                 sink_tokens: int = 0) -> None:
        super().__init__()
        _windowed(window, sink_tokens)
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.layer_id = layer_id
        self.window, self.sink_tokens = window, sink_tokens

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, attn: AttnInputs) -> torch.Tensor:
        if attn.tree is not None and attn.is_prefill:
            raise ValueError("a prefill step takes no tree plan")
        if not attn.is_prefill and (attn.cascade is not None or attn.tree is not None):
            # shared-prefix decode, or trees of drafted tokens: the plan does not fit the vllm::attention schema
            k_cache, v_cache = _layer_caches(self.layer_id)
            if _hides(self.window, attn.block_tables, k_cache) or (attn.cascade is not None and attn.tree is not None):
                raise ValueError("a sliding window, a shared-prefix plan and a tree plan exclude each other")
            if attn.tree is None:
                _refuse_cascade(k_cache)
            scales = _layer_scales(self.layer_id)
            if attn.slot_mapping is not None:
                store_kvcache(k.view(-1, self.num_kv_heads, self.head_dim), v.view(-1, self.num_kv_heads, self.head_dim),
                              k_cache, v_cache, attn.slot_mapping, **scales)
            if attn.tree is not None:
                return tree_attention(q, k_cache, v_cache, attn.block_tables, attn.cache_seqlens, attn.tree.cu_seqlens_q,
                                      attn.tree.mask, attn.tree.max_nodes, self.num_heads, self.num_kv_heads, self.head_dim)
            return cascade_decode_attention(q, k_cache, v_cache, attn.block_tables, attn.cache_seqlens, attn.cascade,
                                            self.num_heads, self.num_kv_heads, self.head_dim, **scales)
        return torch.ops.vllm.attention(
            q, k, v, attn.slot_mapping, attn.is_prefill, attn.cu_seqlens_q, attn.cu_seqlens_k,
            attn.max_seqlen_q, attn.max_seqlen_k, attn.block_tables, attn.cache_seqlens,
            self.layer_id, self.num_heads, self.num_kv_heads, self.head_dim, attn.total_seqlen_k, self.window,
            self.sink_tokens,
        )
