"""Seeded 4-bit (MXFP4) caches and weights for the parity tests, numpy on the CPU."""
from __future__ import annotations

import numpy as np
import torch

import oracle.ops as O


def codes(arr: np.ndarray) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(arr)).view(torch.float4_e2m1fn_x2)


def scales(arr: np.ndarray) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(arr)).view(torch.float8_e8m0fnu)


def random_pages(rng, nb, page, hkv, d, low=122, high=128):
    """Codes [nb, page, hkv, d/2] of every value and scales [nb, page, hkv, d/32]."""
    return (rng.integers(0, 256, (nb, page, hkv, d // 2), dtype=np.uint8),
            rng.integers(low, high + 1, (nb, page, hkv, d // O.FP4_BLOCK)).astype(np.uint8))


def tables(rng, ctx, page, extra=4):
    """Block tables of a random permutation of the pool; (table int32, blocks in the pool)."""
    need = [-(-c // page) for c in ctx]
    nb = sum(need) + extra
    perm = rng.permutation(nb).astype(np.int32)
    bt = np.full((len(ctx), max(1, max(need, default=1))), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        bt[b, :k] = perm[at : at + k]
        at += k
    return bt, nb


def on_device(arr: np.ndarray, dev, layout: str) -> torch.Tensor:
    """arr [nb, page, hkv, n] bytes on the device in the memory order `layout`
    (hnd: heads outermost; wide: token rows with room behind them), logical
    order kept."""
    t = torch.from_numpy(np.ascontiguousarray(arr)).to(dev)
    if layout == "hnd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "wide":
        nb, page, hkv, n = arr.shape
        room = torch.zeros((nb, page, hkv + 1, n), dtype=torch.uint8, device=dev)
        room[:, :, :hkv] = t
        return room[:, :, :hkv]
    return t


def as_codes(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.float4_e2m1fn_x2)


def as_scales(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.float8_e8m0fnu)
