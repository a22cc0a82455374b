"""KV tensor pool (reference src/compute/kv_pool.py:18-83): one tensor
kv_cache[2, L, NB, BS, Hkv, D] holding K (index 0) and V (index 1) pages of
every layer, indexed exactly as the reference's.  Every xvllm kernel reads it
through explicit (page, token, head) strides, so the order in memory is the
pool's choice:

- layout "hnd" (the default): memory is [2, L, NB, Hkv, BS, D] and kv_cache is
  the permuted view with the reference's logical shape; one kv head's page is
  one contiguous BS*D*2 = 4 KB piece, which the decode kernel streams 1-4 %
  faster and with less run-to-run spread than the reference's order.
- layout "nhd" (the reference's memory order, kv_pool.py:49-51): a page is
  [BS, Hkv, D]; one kv head's 16 rows of a page are 256 B pieces at a
  Hkv*D*2 B stride.  Code outside xvllm that needs a contiguous pool (a
  .view() over pages) takes this one.

A 4-bit pool (dtype torch.float4_e2m1fn_x2, no reference counterpart) holds
MXFP4 pages: kv_cache[2, L, NB, BS, Hkv, D/2] of two codes to a byte, and
beside it block_scale[2, L, NB, BS, Hkv, D/32], a power of two for every 32
values, in the same layout.  Its blocks take 17/64 of the bytes of bf16 ones.
"""
from __future__ import annotations

import torch

from .config import head_dim as _head_dim
from .kv_ops import FP4_BLOCK, FP4_PAGES, FP4_SCALE


def get_kv_dims(cfg) -> tuple[int, int, int]:
    """(layers, kv heads, head_dim) at tp = pp = 1 (kv_pool.py:9-15)."""
    return cfg.num_hidden_layers, max(1, cfg.num_key_value_heads), _head_dim(cfg)


def _row_bytes(head_dim: int, dtype: torch.dtype) -> int:
    """Bytes of one head's row in a pool of `dtype` (4-bit: with its scales)."""
    if dtype != FP4_PAGES:
        return head_dim * dtype.itemsize
    if head_dim % FP4_BLOCK:
        raise ValueError(f"a 4-bit pool needs a head_dim of whole blocks of {FP4_BLOCK}, got {head_dim}")
    return head_dim // 2 + head_dim // FP4_BLOCK


class KVPool:
    def __init__(self, hf_config, *, num_blocks: int, block_size: int, device, dtype: torch.dtype,
                 num_layers: int | None = None, layout: str = "hnd", k_scale: float = 1.0,
                 v_scale: float = 1.0) -> None:
        """dtype torch.float8_e4m3fn selects this build's fp8 page format (no
        reference counterpart): K and V are stored as e4m3fn(x / k_scale) and
        e4m3fn(x / v_scale) and attended to as value * scale.
        torch.float4_e2m1fn_x2 selects 4-bit pages, whose scales the store
        takes from the values (block_scale; k_scale and v_scale stay 1)."""
        if num_blocks < 1:
            raise ValueError(f"num_blocks must be > 0, got {num_blocks}")
        if layout not in ("nhd", "hnd"):
            raise ValueError(f"layout must be 'nhd' or 'hnd', got {layout!r}")
        model_layers, nkv, hd = get_kv_dims(hf_config)
        # num_layers: a pool for fewer layers than the model (layer aliasing)
        layers = model_layers if num_layers is None else num_layers
        if not (k_scale > 0 and v_scale > 0):
            raise ValueError("k_scale and v_scale must be > 0")
        row_bytes = _row_bytes(hd, dtype)
        fp4 = dtype == FP4_PAGES
        if fp4 and not (k_scale == v_scale == 1.0):
            raise ValueError("a 4-bit pool takes its scales from the values stored: k_scale and v_scale must be 1")
        vars(self).update(hf_config=hf_config, num_blocks=num_blocks, block_size=block_size, device=device,
                          dtype=dtype, num_layers=layers, layout=layout, k_scale=float(k_scale),
                          v_scale=float(v_scale))
        # bytes of one block across K and V of every layer (kv_pool.py:48)
        self.block_bytes = 2 * layers * block_size * nkv * row_bytes
        self.kv_cache = self._pages(layers, nkv, hd // 2 if fp4 else hd, dtype)
        self.block_scale = self._pages(layers, nkv, hd // FP4_BLOCK, FP4_SCALE) if fp4 else None

    def _pages(self, layers: int, nkv: int, width: int, dtype: torch.dtype) -> torch.Tensor:
        nb, bs = self.num_blocks, self.block_size
        if self.layout == "nhd":
            return torch.empty(2, layers, nb, bs, nkv, width, dtype=dtype, device=self.device)
        return torch.empty(2, layers, nb, nkv, bs, width, dtype=dtype, device=self.device).transpose(3, 4)

    @property
    def num_blocks_total(self) -> int:
        return self.num_blocks

    @classmethod
    def auto_num_blocks(cls, hf_config, *, block_size: int, dtype: torch.dtype, device,
                        gpu_memory_utilization: float, reserve_bytes: int = 0) -> int:
        """Blocks that fit in gpu_memory_utilization of the device (kv_pool.py:62-83)."""
        torch.cuda.empty_cache()
        torch.cuda.synchronize(device)
        layers, nkv, hd = get_kv_dims(hf_config)
        block_bytes = 2 * layers * block_size * nkv * _row_bytes(hd, dtype)
        free, total = torch.cuda.mem_get_info(device)
        available = int(total * gpu_memory_utilization) - (total - free) - reserve_bytes
        return max(4, available // block_bytes)
