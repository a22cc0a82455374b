"""Inputs and 64-bit oracles of the windowed, prefill and tree attention tests.

Tolerance, for outputs o of weights p over values v (bf16 kernels, fp32 sums):
  2^-8 |o|                the rounding of the output to bf16 (half a step)
  2^-8 sum p |v - o|      the weights' rounding to bf16, each by half a step at
                          most; the sum that divides them takes the rounded
                          ones, so an error moves o by its distance to v only
  2^-11 sum p |v - o|     scores: 128-term fp32 sums are off by 128 * 2^-24 of
                          sum |q k| scale (<= 20 here) at most, 2^-12.7, the
                          exponential's argument and result by less, and both
                          enter a weight and the sum of all
"""
import numpy as np
import torch

D = 128
NAN = float("nan")


def paged(lens, block, hkv, seed, layout="hnd", dev="cuda", extra=3):
    """A pool whose rows of no sequence hold NaN, permuted block tables (entries past a sequence's end: a page of
    NaN), and each sequence's K and V [tokens, hkv, D]."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in lens]
    pool = sum(need) + extra
    perm = torch.randperm(pool, generator=g)
    shape = (2, pool, hkv, block, D) if layout == "hnd" else (2, pool, block, hkv, D)
    kv = torch.full(shape, NAN, dtype=torch.bfloat16)
    if layout == "hnd":
        kv = kv.transpose(2, 3)  # [2, pool, block, hkv, D]
    bt = torch.full((len(lens), max(1, *need)), int(perm[-1]), dtype=torch.int32)
    seqs, at = [], 0
    for b, (n, k) in enumerate(zip(lens, need)):
        bt[b, :k] = perm[at : at + k].to(torch.int32)
        at += k
        x = torch.randn(2, n, hkv, D, generator=g).to(torch.bfloat16)
        pos = torch.arange(n)
        kv[:, bt[b].long()[pos // block], pos % block] = x
        seqs.append(x.to(dev))
    d = kv.to(dev)  # keeps the strides
    return d[0], d[1], bt.to(dev), seqs


def attend(q, k, v, seen, scale=None):
    """q [n, hq, D], k and v [keys, hkv, D], seen [n, keys] -> the outputs [n, hq, D] and their tolerances, fp64."""
    n, hq, _ = q.shape
    hkv = k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(n, hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    if k.shape[0] == 0:
        return out, tol
    k = torch.nan_to_num(k.double()).transpose(0, 1).contiguous()
    v = torch.nan_to_num(v.double()).transpose(0, 1).contiguous()
    for h in range(hq):
        s = q[:, h].double() @ k[h * hkv // hq].t().contiguous() * scale
        s = s.masked_fill(~seen, -float("inf"))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top.isinf(), 0.0, top)) * seen
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        vv = v[h * hkv // hq]
        o = p @ vv
        out[:, h] = o
        for i in range(n):
            spread = p[i] @ (vv - o[i]).abs()
            tol[i, h] = o[i].abs() * 2.0 ** -8 + spread * (2.0 ** -8 + 2.0 ** -11) + 1e-30
    return out, tol


def window_mask(pos, keys, window, sinks, dev="cuda"):
    j = torch.arange(keys, device=dev)[None]
    p = torch.as_tensor(pos, device=dev)[:, None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def check(got, want, tol, what=""):
    got = got.double().reshape(want.shape)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float(((got - want).abs() / tol)[bad].max()):.3g} x, first at {bad.nonzero()[0].tolist()}")


def random_tree(n, seed):
    """Parents of n nodes (-1: a child of the last token before the tree)."""
    r = np.random.RandomState(seed)
    return [int(r.randint(-1, i)) if i else -1 for i in range(n)]


def tree_seen(parents):
    """[n, n] whether node i sees node j: its ancestors and itself."""
    n = len(parents)
    seen = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def pack_mask(seen, words):
    """[n, m] truth values -> int64 [n, words]."""
    m = np.zeros((seen.shape[0], words), np.uint64)
    for i, j in seen.nonzero().tolist():
        m[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return torch.from_numpy(m.view(np.int64))
