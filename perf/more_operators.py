"""Attention over the visible part of a paged cache, and the maps that lead to
it, as cases that can be timed and checked: decode and prefill attention with
a sliding window and first tokens that stay visible, attention of a tree of
drafted tokens, and the block tables, slots and positions of a step built from
its requests' lengths.

Kinds (the "kind" of a case):
  maps     a step's maps: every request's block-table row grown by pages of a
           free list, and slot, position and running lengths of its new tokens
  decode   one query token per sequence: it sees the first `sinks` tokens and
           the last `window`, itself among them
  prefill  causal attention of prompts (dense keys) or of prompt chunks (keys
           through the block table) with the same window and sinks
  tree     the last tokens of each sequence are a tree of drafted ones: a node
           sees every token before the tree and the nodes of its mask
"""
import math
import random

import numpy as np
import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
D = 128  # head_dim of every supported shape

# what run() calls where own is true
FUNCS = None


def _api():
    """The framework's entry points (imported only by a tree that has them)."""
    global FUNCS
    if FUNCS is None:
        import sys
        from pathlib import Path

        sys.path.insert(0, str(Path("xixi-vllm_amd").resolve()))
        from xvllm.kv_ops import step_maps
        from xvllm.layers.attention import paged_decode_attention, prefill_attention, tree_attention

        FUNCS = {"maps": step_maps, "decode": paged_decode_attention, "prefill": prefill_attention, "tree": tree_attention}
    return FUNCS


def listed():
    return [
        # one user chatting: the smallest step there is
        dict(name="maps_one", kind="maps", rows=1, lo=1937, hi=1937, new_lo=1, new_hi=1, chunks=0, chunk=0, block=16, tree=False, mix=1),
        # a mixed step: 180 decoding requests and the chunks of 20 prompts
        dict(name="maps_mixed_200", kind="maps", rows=200, lo=100, hi=6000, new_lo=1, new_hi=1, chunks=20, chunk=400, block=16,
             tree=False, mix=2),
        # drafted trees of a full batch, every tree of its own size, a padded batch
        dict(name="maps_trees_256", kind="maps", rows=256, lo=0, hi=9000, new_lo=0, new_hi=64, chunks=0, chunk=0, block=48, tree=True,
             mix=3),
        # one user deep in a long chat: launch latency and the split of one window over the chip
        dict(name="decode_one", kind="decode", rows=1, lo=60001, hi=60001, window=4096, sinks=4, hq=32, hkv=8, block=16, empty=0, mix=4),
        # a decode batch of uneven context, some of it shorter than the window
        dict(name="decode_64", kind="decode", rows=64, lo=512, hi=16000, window=2048, sinks=16, hq=32, hkv=8, block=16, empty=0, mix=5),
        # a padded batch with eight query heads per kv head, window and sinks that end inside pages
        dict(name="decode_padded_200", kind="decode", rows=200, lo=1, hi=9000, window=1000, sinks=5, hq=64, hkv=8, block=48, empty=9,
             mix=6),
        # a prefill step of new prompts
        dict(name="prefill_prompts", kind="prefill", rows=12, q_lo=40, q_hi=2500, lo=0, hi=0, window=512, sinks=4, hq=32, hkv=8, block=0,
             mix=7),
        # one long document, two query heads per kv head
        dict(name="prefill_document", kind="prefill", rows=1, q_lo=16001, q_hi=16001, lo=0, hi=0, window=4096, sinks=64, hq=16, hkv=8,
             block=0, mix=8),
        # prompt chunks over what the pool holds of each prompt, eight query heads per kv head
        dict(name="prefill_chunks", kind="prefill", rows=16, q_lo=300, q_hi=512, lo=0, hi=12000, window=2000, sinks=4, hq=64, hkv=8,
             block=16, mix=9),
        # one user with a small tree: latency
        dict(name="tree_one", kind="tree", rows=1, lo=1937, hi=1937, n_lo=16, n_hi=16, hq=32, hkv=8, block=16, empty=0, mix=10),
        # a batch with trees of their own sizes, some rows of it without a request
        dict(name="tree_32", kind="tree", rows=32, lo=300, hi=4096, n_lo=5, n_hi=64, hq=32, hkv=8, block=16, empty=2, mix=11),
        # few users with long documents, more than 64 nodes each
        dict(name="tree_long", kind="tree", rows=4, lo=30000, hi=90001, n_lo=40, n_hi=90, hq=16, hkv=8, block=256, empty=0, mix=12),
    ]


HEADS = [(16, 8), (32, 8), (32, 8), (64, 8), (8, 8), (8, 1), (6, 3)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["maps", "decode", "decode", "prefill", "prefill", "tree", "tree"])
    mix = rng.randrange(1 << 20)
    block = rng.choice([16, 16, 48, 256])
    hq, hkv = rng.choice(HEADS)
    if kind == "maps":
        rows = _log_int(rng, 1, 512)
        new = _log_int(rng, 1, max(2, 16384 // rows))
        tree = rng.random() < 0.4
        return dict(kind=kind, rows=rows, lo=0, hi=_log_int(rng, 1, 30000),
                    new_lo=rng.choice([0, 1]) if rows > 4 else 1, new_hi=min(new, 64) if tree else new,
                    chunks=0, chunk=0, block=block, tree=tree, mix=mix)
    if kind == "decode":
        rows = _log_int(rng, 1, 256)
        window = min(_log_int(rng, 1, 16000), 180000 // rows)
        hi = min(_log_int(rng, 1, 100000), 400000 // rows)
        return dict(kind=kind, rows=rows, lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, window=window, sinks=rng.choice([0, 1, 4, 16, 100]),
                    hq=hq, hkv=hkv, block=block, empty=rng.choice([0, 0, 1, rows // 3]) if rows > 1 else 0, mix=mix)
    if kind == "prefill":
        rows = _log_int(rng, 1, 24)
        paged = rng.random() < 0.5
        q = min(_log_int(rng, 1, 2000), 8000 // rows)
        hi = min(_log_int(rng, 1, 12000), 60000 // rows, 4000000000 // (rows * q * hq)) if paged else 0
        window = _log_int(rng, 1, min(5000, 900000000 // (rows * q * hq)))
        return dict(kind=kind, rows=rows, q_lo=max(1, q // rng.choice([1, 3, 10])), q_hi=q, lo=0, hi=hi, window=window,
                    sinks=rng.choice([0, 1, 4, 16, 100]), hq=hq, hkv=hkv, block=block if paged else 0, mix=mix)
    rows = _log_int(rng, 1, 48)
    hi = min(_log_int(rng, 1, 80000), 120000 // rows)
    n = min(_log_int(rng, 1, 128), 2048 // rows)
    return dict(kind=kind, rows=rows, lo=rng.choice([0, hi // 2]), hi=hi, n_lo=max(1, n // rng.choice([1, 2, 8])), n_hi=n, hq=hq, hkv=hkv,
                block=block, empty=rng.choice([0, 0, 1, rows // 3]) if rows > 1 else 0, mix=mix)


# ---------------------------------------------------------------- sizes of a case
def _sizes(c):
    """(tokens already there, new tokens) of each sequence; the empty rows of a padded batch have neither."""
    r = random.Random(c["mix"])
    old = [r.randint(c["lo"], c["hi"]) for _ in range(c["rows"])]
    if c["kind"] == "maps":
        new = [r.randint(c["new_lo"], c["new_hi"]) for _ in old]
        for b in r.sample(range(c["rows"]), c["chunks"]):
            new[b] = r.randint(c["chunk"] // 2, c["chunk"])
    elif c["kind"] == "prefill":
        new = [r.randint(c["q_lo"], c["q_hi"]) for _ in old]
    elif c["kind"] == "tree":
        new = [r.randint(c["n_lo"], c["n_hi"]) for _ in old]
    else:
        new = [0] * len(old)  # the token of this step is counted in lo .. hi
    for b in r.sample(range(c["rows"]), c.get("empty", 0)):
        old[b] = new[b] = 0
    return old, new


def _trees(c, new):
    """Each sequence's drafted tree: the parent of every node, -1 for a child of the last token before the tree."""
    r = random.Random(c["mix"] + 1)
    return [[r.choice([-1, max(-1, i - r.randint(1, 8)), i - 1]) if i else -1 for i in range(n)] for n in new]


def _visible(p, window, sinks):
    """Keys that a query at position p sees."""
    return min(p + 1, window + min(sinks, max(0, p + 1 - window)))


def work(c):
    old, new = _sizes(c)
    if c["kind"] == "maps":
        pages = sum(-(-(o + n) // c["block"]) - -(-o // c["block"]) for o, n in zip(old, new))
        # lengths and pages read; tables, running lengths, positions and slots written
        return {"bytes": c["rows"] * 20 + pages * 8 + sum(new) * (16 if c["tree"] else 12), "flops": 0}
    hq, row = c["hq"], 2 * c["hkv"] * D * 2  # K and V of a token
    io = 2 * hq * D * 2                      # a query and its output
    if c["kind"] == "decode":
        seen = sum(_visible(o - 1, c["window"], c["sinks"]) for o in old if o)
        return {"bytes": seen * row + c["rows"] * io, "flops": 4 * hq * D * seen}
    if c["kind"] == "prefill":
        pairs = sum(_visible(p, c["window"], c["sinks"]) for o, n in zip(old, new) for p in range(o, o + n))
        keys = sum(n + _visible(o, c["window"], c["sinks"]) - 1 for o, n in zip(old, new))
        return {"bytes": keys * row + sum(new) * io, "flops": 4 * hq * D * pairs}
    pairs = sum(n * o for o, n in zip(old, new)) + sum(len(p) for t in _trees(c, new) for p in _paths(t))
    return {"bytes": (sum(old) + sum(new)) * row + sum(new) * (io + 8), "flops": 4 * hq * D * pairs}


def _paths(parents):
    """Each node's path: its ancestors in the tree, and itself."""
    paths = []
    for i, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else []) + [i])
    return paths


# ---------------------------------------------------------------- inputs, from the seed alone
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F32).to(BF16)


def _tables(lens, block, seed, width=0):
    """Block tables of sequences of `lens` tokens out of a random permutation
    of a pool a quarter larger than needed (entries past a sequence's end hold
    -1), the pages that are left, and the size of the pool."""
    need = [-(-s // block) for s in lens]
    pool = max(4, int(1.25 * sum(need)) + 1, width * len(lens) + 4)
    perm = np.random.RandomState(seed % (1 << 31)).permutation(pool).astype(np.int32)
    bt = np.full((len(lens), max(1, width, max(need))), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        bt[b, :k] = perm[at : at + k]
        at += k
    return bt, perm[at:], pool


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to("cuda")


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def prepare(case, seed):
    g = _gen(seed)
    old, new = _sizes(case)
    ends = [o + n for o, n in zip(old, new)]
    block = case["block"]
    st = {"case": case}
    if case["kind"] == "maps":
        bt, free, _ = _tables(old, block, seed, width=max(1, max(-(-e // block) for e in ends)))
        st.update(seq_lens=_dev(old), new_lens=_dev(new), bt=_dev(bt), free=_dev(free), head=_dev([seed % 3]), total=sum(new))
        if case["tree"]:
            st["depths"] = _dev([len(p) - 1 for t in _trees(case, new) for p in _paths(t)])
        return st
    hq, hkv = case["hq"], case["hkv"]
    if case["kind"] == "prefill" and not block:  # q, k and v are views of one qkv product
        qkv = _randn(g, sum(new), (hq + 2 * hkv) * D)
        st.update(q=qkv[:, : hq * D], k=qkv[:, hq * D : (hq + hkv) * D], v=qkv[:, (hq + hkv) * D :])
    else:
        bt, _, pool = _tables(ends, block, seed)
        # one head's block of tokens is contiguous; keys have a few loud channels, as after a rotary embedding
        k = torch.randn(pool, hkv, block, D, generator=g, device="cuda", dtype=F32)
        loud = torch.randint(0, D, (4,), generator=g, device="cuda")
        k[..., loud] *= 4
        st.update(k=k.to(BF16).transpose(1, 2), v=_randn(g, pool, hkv, block, D).transpose(1, 2), bt=_dev(bt), lens=_dev(ends))
        st["q"] = _randn(g, sum(new) if case["kind"] != "decode" else case["rows"], hq * D)
    if case["kind"] != "decode":
        st.update(cu_q=_dev(_cu(new)), cu_k=_dev(_cu(ends)), max_q=max(new), max_k=max(ends), total_k=sum(ends), new=new, ends=ends)
    if case["kind"] == "tree":
        words = -(-max(new) // 64)
        mask = np.zeros((sum(new), words), np.uint64)
        at = 0
        for tree in _trees(case, new):
            for path in _paths(tree):
                for j in path:
                    mask[at, j // 64] |= np.uint64(1 << (j % 64))
                at += 1
        st["mask"] = _dev(mask.view(np.int64), np.int64)
    return st


# ---------------------------------------------------------------- the plain forms
def _plain_maps(st):
    block, total = st["case"]["block"], st["total"]
    old, new, bt, free = st["seq_lens"].long(), st["new_lens"].long(), st["bt"], st["free"]
    ends = old + new
    zero = old.new_zeros(1)
    cu_q, cu_k = torch.cat([zero, new.cumsum(0)]), torch.cat([zero, ends.cumsum(0)])
    have, need = (old + block - 1) // block, (ends + block - 1) // block
    cu_p = torch.cat([zero, (need - have).cumsum(0)])
    head = st["head"].long()
    col = torch.arange(bt.shape[1], device=bt.device)
    at = (head + cu_p[:-1] - have)[:, None] + col
    fresh = (col >= have[:, None]) & (col < need[:, None])
    bt.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], bt))
    t = torch.arange(total, device=bt.device)
    row = torch.searchsorted(cu_q, t, right=True) - 1
    pos = old[row] + t - cu_q[row]
    slots = bt[row, pos // block] * block + pos % block
    if st["case"]["tree"]:
        pos = old[row] + st["depths"]
    i32 = torch.int32
    return cu_q.to(i32), cu_k.to(i32), ends.to(i32), pos, slots.to(i32), (head + cu_p[-1]).to(i32), bt


def _softmax_product(q, k, v, seen):
    """softmax over the seen keys of q k^T / sqrt(D), times v; q [..., n, D], k and v [..., keys, D], fp32."""
    s = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(D)
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top > -math.inf, top, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def _plain_decode(st):
    c = st["case"]
    rows, hq, hkv, block, window, sinks = c["rows"], c["hq"], c["hkv"], c["block"], c["window"], c["sinks"]
    lens = st["lens"].long()[:, None]
    first = (lens - window).clamp(min=0)  # the first key of the window
    width = min(window, st["bt"].shape[1] * block)
    pos = torch.cat([torch.arange(sinks, device="cuda").expand(rows, sinks), first + torch.arange(width, device="cuda")], dim=1)
    seen = pos < lens
    seen[:, :sinks] &= pos[:, :sinks] < first
    pos = torch.where(seen, pos, 0)
    page = torch.gather(st["bt"].long(), 1, pos // block).clamp(min=0)
    k = st["k"][page, pos % block].to(F32).permute(0, 2, 1, 3)
    v = st["v"][page, pos % block].to(F32).permute(0, 2, 1, 3)
    q = st["q"].to(F32).view(rows, hkv, hq // hkv, D)
    return _softmax_product(q, k, v, seen[:, None, None, :]).reshape(rows, -1).to(BF16)


def _keys(st, b):
    """Sequence b's keys and values [hkv, tokens, D] in fp32."""
    c, n = st["case"], st["ends"][b]
    if not c["block"]:
        at = sum(st["ends"][:b])
        return [st[x][at : at + n].to(F32).view(n, c["hkv"], D).transpose(0, 1) for x in ("k", "v")]
    pages = st["bt"][b, : -(-n // c["block"])].long()
    return [st[x][pages].to(F32).reshape(-1, c["hkv"], D)[:n].transpose(0, 1) for x in ("k", "v")]


def _plain_rows(st):
    """prefill and tree: a sequence and a kv head at a time."""
    c = st["case"]
    hq, hkv = c["hq"], c["hkv"]
    out = torch.empty(sum(st["new"]), hq * D, dtype=BF16, device="cuda")
    at = 0
    for b, (n, end) in enumerate(zip(st["new"], st["ends"])):
        if n == 0:
            continue
        k, v = _keys(st, b)
        key = torch.arange(end, device="cuda")
        pos = torch.arange(end - n, end, device="cuda")[:, None]
        if c["kind"] == "prefill":
            seen = (key <= pos) & ((key > pos - c["window"]) | (key < c["sinks"]))
        else:
            node = (key - (end - n)).clamp(min=0)
            seen = (key < end - n) | ((st["mask"][at : at + n][:, node // 64] >> (node % 64)) & 1).bool()
        q = st["q"][at : at + n].to(F32).view(n, hkv, hq // hkv, D)
        o = out[at : at + n].view(n, hkv, hq // hkv, D)
        for h in range(hkv):
            o[:, h] = _softmax_product(q[:, h].transpose(0, 1), k[h], v[h], seen).transpose(0, 1).to(BF16)
        at += n
    return out


def run(state):
    c = state["case"]
    if not own:
        return {"maps": _plain_maps, "decode": _plain_decode, "prefill": _plain_rows, "tree": _plain_rows}[c["kind"]](state)
    f = _api()[c["kind"]]
    if c["kind"] == "maps":
        m = f(state["seq_lens"], state["new_lens"], state["bt"], state["free"], c["block"], state["total"], free_head=state["head"],
              depths=state.get("depths"))
        return m.cu_seqlens_q, m.cu_seqlens_k, m.cache_seqlens, m.positions, m.slot_mapping, m.free_head, state["bt"]
    heads = (c["hq"], c["hkv"], D)
    if c["kind"] == "decode":
        return f(state["q"], state["k"], state["v"], state["bt"], state["lens"], *heads, window=c["window"], sink_tokens=c["sinks"])
    if c["kind"] == "tree":
        return f(state["q"], state["k"], state["v"], state["bt"], state["lens"], state["cu_q"], state["mask"], state["max_q"], *heads)
    if c["block"]:
        return f(state["q"], None, None, state["cu_q"], state["cu_k"], state["max_q"], *heads, k_cache=state["k"], v_cache=state["v"],
                 block_tables=state["bt"], window=c["window"], sink_tokens=c["sinks"])
    return f(state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"], state["max_q"], *heads, window=c["window"],
             sink_tokens=c["sinks"])


# ---------------------------------------------------------------- the definition, in 64 bits
def _exact_maps(st):
    """Request by request, on the host."""
    block = st["case"]["block"]
    old, new = st["seq_lens"].tolist(), st["new_lens"].tolist()
    bt, free, head = st["bt"].tolist(), st["free"].tolist(), st["head"].tolist()[0]
    depths = st["depths"].tolist() if st["case"]["tree"] else None
    cu_q, cu_k, pos, slots = [0], [0], [], []
    for b, (o, n) in enumerate(zip(old, new)):
        for blk in range((o + block - 1) // block, (o + n + block - 1) // block):
            bt[b][blk] = free[head]
            head += 1
        for p in range(o, o + n):
            pos.append(o + depths[len(pos)] if depths else p)
            slots.append(bt[b][p // block] * block + p % block)
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + o + n)
    ends = [o + n for o, n in zip(old, new)]
    return tuple(torch.tensor(x, dtype=torch.int64, device="cuda") for x in (cu_q, cu_k, ends, pos, slots, [head], bt))


def _attend64(q, k, v, bias):
    return torch.softmax(q @ k.t().contiguous() * D ** -0.5 + bias, dim=-1) @ v


def _bias64(seen):
    return torch.zeros(seen.shape, dtype=F64, device="cuda").masked_fill_(~seen, -math.inf)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "maps":
        return _exact_maps(st)
    hq, hkv, block = case["hq"], case["hkv"], case["block"]
    group = hq // hkv
    old, new = _sizes(case)
    if case["kind"] == "prefill" and sum(n * (o + n) for o, n in zip(old, new)) * hq > 5 << 30:
        return None
    out = torch.zeros(st["q"].shape[0], hq, D, dtype=F64, device="cuda")
    at = dense = 0
    for b, (o, n) in enumerate(zip(old, new)):
        end = o + n
        count = 1 if case["kind"] == "decode" else n
        if end == 0 or count == 0:
            at += count
            continue
        if block:
            slot = torch.arange(end, device="cuda")
            page = st["bt"][b].long()[slot // block]
            k, v = st["k"][page, slot % block].to(F64), st["v"][page, slot % block].to(F64)
        else:
            k, v = (st[x][dense : dense + end].to(F64).view(end, hkv, D) for x in ("k", "v"))
            dense += end
        j = torch.arange(end, device="cuda")[None, :]
        if case["kind"] == "tree":
            seen = torch.ones(n, end, dtype=torch.bool, device="cuda")
            seen[:, o:] = False
            for i, path in enumerate(_paths(_trees(case, new)[b])):
                seen[i, [o + p for p in path]] = True
        else:
            p = torch.arange(end - count, end, device="cuda")[:, None]
            seen = (p - j >= 0) & ((p - j < case["window"]) | (j < case["sinks"]))
        q = st["q"][at : at + count].to(F64).view(count, hq, D)
        bias = _bias64(seen)
        for h in range(hq):
            out[at : at + count, h] = _attend64(q[:, h], k[:, h // group], v[:, h // group], bias)
        at += count
    return out.reshape(out.shape[0], -1)
