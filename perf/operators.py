"""The 4-bit operators of the serving path as cases that can be timed and
checked: K and V quantised as the paged cache is written and read back, decode
attention over the 4-bit pages, and the products of a decode batch with 4-bit
weights.

Everything is held as OCP MXFP4: a block of 32 values along the contiguous
axis is 32 e2m1 codes (two a byte, the lower index in the low half) and one
e8m0 scale byte s, and stands for code * 2^(s - 127).  A block is quantised
with the exponent of its largest magnitude (carried up where the mantissa is
1.75 or more) minus 2, between -126 and 125, then each value to the nearest
code, ties to the even one, past 6 to 6.

Kinds (the "kind" of a case):
  kv      KV store of a step's new tokens into 4-bit pages, then every
          sequence's keys and values read back as bf16 rows (what a chunked
          prefill attends to)
  attn    paged decode attention over 4-bit pages
  linear  x @ w^T with a 4-bit weight, bf16 activations; silu: w is a
          gate / up weight and the result silu(gate) * up
"""
import math
import random

import numpy as np
import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
D = 128     # head_dim of every supported shape
BLOCK = 32  # values that share one scale
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)

# what run() calls where own is true
FUNCS = None


def _api():
    """The framework's entry points (imported only by a tree that has them)."""
    global FUNCS
    if FUNCS is None:
        import sys
        from pathlib import Path

        sys.path.insert(0, str(Path("xixi-vllm_amd").resolve()))
        from xvllm.kv_ops import gather_kvcache, store_kvcache
        from xvllm.layers.attention import paged_decode_attention
        from xvllm.layers.linear import mxfp4_linear

        FUNCS = {"store": store_kvcache, "gather": gather_kvcache, "decode": paged_decode_attention, "linear": mxfp4_linear}
    return FUNCS


def listed():
    return [
        # a short prompt of one user: the smallest cache write and read there is
        dict(name="kv_one_prompt", kind="kv", rows=1, q=77, lo=0, hi=0, hkv=8, block=16, mix=1),
        # a chunked-prefill step: 512-token chunks of 16 prompts over what the pool holds of each
        dict(name="kv_chunks", kind="kv", rows=16, q=512, lo=0, hi=1536, hkv=8, block=16, mix=2),
        # the last chunks of long documents: the read back of the prefix outweighs the write
        dict(name="kv_long_prefix", kind="kv", rows=3, q=2048, lo=20000, hi=33000, hkv=8, block=256, mix=3),
        # one user chatting: launch latency and the split of one sequence over the chip
        dict(name="attn_one", kind="attn", rows=1, lo=1937, hi=1937, hq=32, hkv=8, block=16, empty=0, mix=4),
        # the headline decode batch: 64 sequences of uneven context
        dict(name="attn_64", kind="attn", rows=64, lo=512, hi=4096, hq=32, hkv=8, block=16, empty=0, mix=5),
        # eight query heads per kv head, a padded batch (rows of length 0)
        dict(name="attn_padded_48", kind="attn", rows=48, lo=700, hi=6000, hq=64, hkv=8, block=16, empty=5, mix=6),
        # few users with long documents, large cache blocks, two query heads per kv head
        dict(name="attn_long", kind="attn", rows=4, lo=40000, hi=130001, hq=16, hkv=8, block=256, empty=0, mix=7),
        # one user's attention output projection: the smallest weight there is
        dict(name="linear_one", kind="linear", rows=1, n=4096, k=4096, silu=False),
        # one user's gate / up product of the same model, with its SiLU
        dict(name="linear_one_gate_up", kind="linear", rows=1, n=24576, k=4096, silu=True),
        # a small serving batch through a down projection
        dict(name="linear_8_down", kind="linear", rows=8, n=4096, k=12288, silu=False),
        # odd sizes: rows, columns and blocks that fill no tile
        dict(name="linear_odd", kind="linear", rows=37, n=5003, k=4704, silu=False),
        # a full decode batch through a large model's gate / up weight
        dict(name="linear_200_gate_up", kind="linear", rows=200, n=51200, k=5120, silu=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["kv", "attn", "attn", "linear", "linear"])
    mix = rng.randrange(1 << 20)
    if kind == "kv":
        rows = _log_int(rng, 1, 32)
        q = min(_log_int(rng, 1, 4096), 8192 // rows)
        hi = min(_log_int(rng, 1, 40000), 98304 // rows)
        return dict(kind=kind, rows=rows, q=q, lo=0, hi=hi, hkv=rng.choice([1, 2, 4, 5, 8]), block=rng.choice([16, 16, 48, 256]), mix=mix)
    if kind == "attn":
        rows = _log_int(rng, 1, 300)
        hi = min(_log_int(rng, 1, 130000), 300000 // rows)
        hq, hkv = rng.choice([(16, 8), (32, 8), (32, 8), (64, 8), (8, 8), (8, 1), (6, 3)])
        return dict(kind=kind, rows=rows, lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, hq=hq, hkv=hkv,
                    block=rng.choice([16, 16, 48, 256]), empty=rng.choice([0, 0, 1, rows // 3]) if rows > 1 else 0, mix=mix)
    rows = _log_int(rng, 1, 256)
    silu = rng.random() < 0.4
    n = _log_int(rng, 16, 51200) // (2 if silu else 1) * (2 if silu else 1)
    k = BLOCK * _log_int(rng, 1, min(800, 262144000 // n // BLOCK))
    return dict(kind=kind, rows=rows, n=n, k=k, silu=silu)


# ---------------------------------------------------------------- sizes of a case
def _lens(c):
    """Tokens of each sequence (kv: those already in the pool); every few rows of a padded batch are empty."""
    r = random.Random(c["mix"])
    lens = [r.randint(c["lo"], c["hi"]) for _ in range(c["rows"])]
    for b in r.sample(range(c["rows"]), c.get("empty", 0)):
        lens[b] = 0
    return lens


def work(c):
    if c["kind"] == "linear":
        m, n, k = c["rows"], c["n"], c["k"]
        out = n // 2 if c["silu"] else n
        return {"bytes": n * (k // 2 + k // BLOCK) + m * (k + out) * 2, "flops": 2 * m * n * k}
    lens = _lens(c)
    row = 2 * c["hkv"] * (D // 2 + D // BLOCK)  # K and V of a cached token
    if c["kind"] == "attn":
        return {"bytes": sum(lens) * row + c["rows"] * 2 * c["hq"] * D * 2, "flops": 4 * c["hq"] * D * sum(lens)}
    new, every = c["rows"] * c["q"], sum(lens) + c["rows"] * c["q"]
    bf = 2 * c["hkv"] * D * 2
    # a step's new rows need not be read again from the cache that they were just written to
    return {"bytes": new * (bf + row) + (every - new) * row + every * bf, "flops": 0}


# ---------------------------------------------------------------- inputs, from the seed alone
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(g, *shape):
    """Bytes of two codes each, every code alike."""
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def _scales(g, *shape, low, high):
    return torch.randint(low, high + 1, shape, generator=g, device="cuda", dtype=torch.uint8)


def _tables(lens, block, seed):
    """Block tables of sequences of `lens` tokens: a random permutation of a
    pool a quarter larger than needed; entries past a sequence's end hold -1."""
    need = [-(-s // block) for s in lens]
    pool = max(4, int(1.25 * sum(need)) + 1)
    perm = np.random.RandomState(seed % (1 << 31)).permutation(pool).astype(np.int32)
    bt = np.full((len(lens), max(1, max(need))), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        bt[b, :k] = perm[at : at + k]
        at += k
    return bt, pool


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to("cuda")


def _pages(g, pool, block, hkv, low, high):
    """Codes and scales [blocks, tokens, heads, ...] of a filled pool, one head's block of tokens contiguous."""
    data = _codes(g, pool, hkv, block, D // 2).transpose(1, 2)
    return data, _scales(g, pool, hkv, block, D // BLOCK, low=low, high=high).transpose(1, 2)


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        x = torch.randn(m, k, generator=g, device="cuda", dtype=F32).to(BF16)
        # weights of a trained size: blocks whose largest code stands for 0.01 .. 0.1
        return {"case": case, "x": x, "w": _codes(g, n, k // 2), "s": _scales(g, n, k // BLOCK, low=118, high=121)}
    lens, block, hkv = _lens(case), case["block"], case["hkv"]
    if case["kind"] == "attn":
        bt, pool = _tables(lens, block, seed)
        k, ks = _pages(g, pool, block, hkv, 124, 126)
        v, vs = _pages(g, pool, block, hkv, 122, 127)
        q = torch.randn(case["rows"], case["hq"] * D, generator=g, device="cuda", dtype=F32).to(BF16)
        return {"case": case, "q": q, "k": k, "ks": ks, "v": v, "vs": vs, "bt": _dev(bt), "lens": _dev(lens)}
    ends = [s + case["q"] for s in lens]
    bt, pool = _tables(ends, block, seed)
    k, ks = _pages(g, pool, block, hkv, 120, 129)
    v, vs = _pages(g, pool, block, hkv, 120, 129)
    n = case["rows"] * case["q"]
    # keys have a few loud channels, as after a rotary embedding; k and v are views of one qkv product
    qkv = torch.randn(n, 2, hkv, D, generator=g, device="cuda", dtype=F32)
    loud = torch.randint(0, D, (hkv, 4), generator=g, device="cuda")
    qkv[:, 0].scatter_(2, loud.expand(n, hkv, 4), torch.randn(n, hkv, 4, generator=g, device="cuda", dtype=F32) * 12)
    qkv = qkv.to(BF16)
    pos = [np.arange(s, e) for s, e in zip(lens, ends)]
    slots = np.concatenate([bt[b, p // block] * block + p % block for b, p in enumerate(pos)])
    cu = np.concatenate([[0], np.cumsum(ends)])
    return {"case": case, "new_k": qkv[:, 0], "new_v": qkv[:, 1], "k": k, "ks": ks, "v": v, "vs": vs, "bt": _dev(bt),
            "slots": _dev(slots), "cu": _dev(cu), "total": int(cu[-1])}


# ---------------------------------------------------------------- the plain forms
def _power(scale):
    """2^(s - 127) of scale bytes 1 .. 254 in fp32, exactly: the byte is its exponent field."""
    return (scale.to(torch.int32) << 23).view(F32)


def _value(data, scale):
    """The fp32 values of codes [..., n / 2] and scales [..., n / 32]."""
    table = torch.tensor(CODES, dtype=F32, device=data.device)
    pair = torch.stack((data & 15, data >> 4), dim=-1)
    codes = table[pair.reshape(*data.shape[:-1], -1, BLOCK).int()]
    return (codes * _power(scale)[..., None]).flatten(-2)


def _quantise(x):
    """Codes and scales of x [..., n], fp32 arithmetic that is exact throughout."""
    blocks = x.to(F32).unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 1 + (mantissa >= 0.875).to(exponent.dtype) - 2
    e = torch.where(top > 0, e, -126).clamp(-126, 125)
    scale = (e + 127).to(torch.uint8)
    a = blocks.abs() / _power(scale)[..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (blocks < 0)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _plain_write(new, data, scale, slots, block):
    page, row = slots.long() // block, slots.long() % block
    data[page, row], scale[page, row] = _quantise(new)


def _plain_kv(st):
    block = st["case"]["block"]
    _plain_write(st["new_k"], st["k"], st["ks"], st["slots"], block)
    _plain_write(st["new_v"], st["v"], st["vs"], st["slots"], block)
    cu = st["cu"].long()
    at = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(cu, at, right=True) - 1
    pos = at - cu[seq]
    page, row = st["bt"].long()[seq, pos // block], pos % block
    return _value(st["k"][page, row], st["ks"][page, row]).to(BF16), _value(st["v"][page, row], st["vs"][page, row]).to(BF16)


def _plain_attn(st):
    c = st["case"]
    rows, hq, hkv, block = c["rows"], c["hq"], c["hkv"], c["block"]
    bt = st["bt"].long().clamp(min=0)
    keys = bt.shape[1] * block
    shape = (rows, keys, hkv, -1)
    k = _value(st["k"][bt].reshape(shape), st["ks"][bt].reshape(shape)).permute(0, 2, 3, 1)
    v = _value(st["v"][bt].reshape(shape), st["vs"][bt].reshape(shape)).permute(0, 2, 1, 3)
    q = st["q"].to(F32).view(rows, hkv, hq // hkv, D)
    s = torch.matmul(q, k) / math.sqrt(D)
    seen = (torch.arange(keys, device="cuda") < st["lens"][:, None])[:, None, None, :]
    s = torch.where(seen, s, -math.inf)
    p = torch.where(seen, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return torch.where(st["lens"][:, None] > 0, o.reshape(rows, -1), 0.0).to(BF16)


def _plain_linear(st):
    y = torch.matmul(st["x"].to(F32), _value(st["w"], st["s"]).t())
    if st["case"]["silu"]:
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(BF16)


def run(state):
    c = state["case"]
    if own:
        f = _api()
        if c["kind"] == "linear":
            return f["linear"](state["x"], state["w"].view(FP4), state["s"].view(E8M0), silu_mul=c["silu"])
        k, v, ks, vs = state["k"].view(FP4), state["v"].view(FP4), state["ks"].view(E8M0), state["vs"].view(E8M0)
        if c["kind"] == "attn":
            return f["decode"](state["q"], k, v, state["bt"], state["lens"], c["hq"], c["hkv"], D, k_block_scale=ks, v_block_scale=vs)
        f["store"](state["new_k"], state["new_v"], k, v, state["slots"], k_block_scale=ks, v_block_scale=vs)
        return f["gather"](k, v, state["bt"], state["cu"], state["total"], k_block_scale=ks, v_block_scale=vs)
    return {"kv": _plain_kv, "attn": _plain_attn, "linear": _plain_linear}[c["kind"]](state)


# ---------------------------------------------------------------- the definition, in 64 bits
def _power64(e):
    """2^e of whole numbers, built from the bits."""
    return ((e + 1023) << 52).view(F64)


def _decode64(data, scale):
    """Values of codes and scales from the bits: sign, 2 exponent bits, 1 mantissa bit."""
    code = torch.empty(*data.shape, 2, dtype=torch.int64, device=data.device)
    code[..., 0], code[..., 1] = data.long() % 16, data.long() // 16
    code = code.flatten(-2)
    sign, e, m = 1 - 2 * (code // 8), code // 2 % 4, code % 2
    mag = torch.where(e == 0, m.to(F64) / 2, (1 + m.to(F64) / 2) * _power64(e - 1))
    return sign * mag * _power64(scale.long() - 127).repeat_interleave(BLOCK, dim=-1)


def _nearest64(x):
    """x [..., n] rounded to its MXFP4 blocks: the nearest multiple of the code spacing around each value."""
    b = x.to(F64).reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0))).long()
    e = torch.where(_power64(e) > top, e - 1, e)  # a logarithm that rounded up
    e = torch.where(top / _power64(e) >= 1.75, e + 1, e) - 2
    unit = _power64(torch.where(top > 0, e, -126).clamp(-126, 125))
    a = (b / unit).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(F64)
    return (torch.sign(b) * torch.clamp(torch.round(a / step) * step, max=6.0) * unit).reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "linear":
        if case["rows"] * case["n"] * case["k"] > 1 << 37:
            return None
        parts = [st["x"].to(F64) @ _decode64(st["w"][i : i + 2048], st["s"][i : i + 2048]).t().contiguous() for i in range(0, case["n"], 2048)]
        y = torch.cat(parts, dim=1)
        half = case["n"] // 2
        return y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:] if case["silu"] else y
    block = case["block"]
    if case["kind"] == "attn":
        out = torch.zeros(case["rows"], case["hq"], D, dtype=F64, device="cuda")
        group = case["hq"] // case["hkv"]
        for b, n in enumerate(st["lens"].tolist()):
            pages = st["bt"][b, : -(-n // block)].long()
            for h in range(case["hkv"] if n else 0):
                k = _decode64(st["k"][pages, :, h], st["ks"][pages, :, h]).reshape(-1, D)[:n]
                v = _decode64(st["v"][pages, :, h], st["vs"][pages, :, h]).reshape(-1, D)[:n]
                q = st["q"][b].view(-1, D)[h * group : (h + 1) * group].to(F64)
                w = torch.softmax(q @ k.t().contiguous() * D ** -0.5, dim=-1)
                out[b, h * group : (h + 1) * group] = w @ v
        return out.reshape(case["rows"], -1)
    res = []
    n, q = case["rows"], case["q"]
    for new, data, scale in ((st["new_k"], st["k"], st["ks"]), (st["new_v"], st["v"], st["vs"])):
        rows = []
        for b, end in enumerate((st["cu"][1:] - st["cu"][:-1]).tolist()):
            pages = st["bt"][b, : -(-end // block)].long()
            old = _decode64(data[pages], scale[pages]).reshape(-1, case["hkv"], D)[: end - q]
            rows += [old, _nearest64(new[b * q : (b + 1) * q])]
        res.append(torch.cat(rows))
    return tuple(res)
