"""The 4-bit (MXFP4) operators as they are used together: a pool's store, read
back, chunked prefill and decode, and the model and runner on a 4-bit pool.

Each stage is held to the oracle's for the very inputs that it had, so that a
code that falls the other way (one unit in the last place of a key before it)
is no difference: the store and read back are exact; decode is held to 4 * 2^-9
of the weighted mean magnitude (roundings of the weights and of the output,
2^-8 each at most); products to 2^-8 of the value
and (K + 8) 2^-24 of the sum of magnitudes; the dense prefill and the layer's
other kernels to the bf16 tolerance that their own tests have."""
import numpy as np
import pytest
import torch

import oracle.model as OM
import oracle.ops as O
from helpers import f32, gen, randn_bf16
from fp4_cases import as_codes, as_scales

pytestmark = pytest.mark.gpu

D = 128


def _bytes(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def _values(kv, i, layer):
    """What pool half i (0 keys, 1 values) of a layer holds, in 64 bits."""
    return O.dequantize_fp4(_bytes(kv.kv_cache[i, layer]), _bytes(kv.block_scale[i, layer]))


def _pool(dev, hq, hkv, blocks, page, layout, layers=1):
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool

    kv = KVPool(Qwen3Shape(256, hq, hkv, D, 512, layers), num_blocks=blocks, block_size=page, device=dev,
                dtype=torch.float4_e2m1fn_x2, layout=layout)
    kv.block_scale.view(torch.uint8).fill_(255)  # NaN: rows are read only where a store wrote them
    kv.kv_cache.view(torch.uint8).fill_(0x77)
    return kv


def _attend(q, k, v, scale=D ** -0.5):
    """softmax(q k^T) v of one sequence's rows q [n, Hq, D], the last n of the keys, in 64 bits, with the weighted
    mean magnitudes."""
    n, hq, _ = q.shape
    total, hkv = k.shape[:2]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    seen = np.arange(total)[None] <= total - n + np.arange(n)[:, None]
    for h in range(hq):
        s = np.where(seen, q[:, h] @ k[:, h // (hq // hkv)].T * scale, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[:, h], mag[:, h] = w @ v[:, h // (hq // hkv)], w @ np.abs(v[:, h // (hq // hkv)])
    return out, mag


def _close(got, want, tolerance):
    got = got.detach().double().cpu().numpy().reshape(want.shape)
    assert np.isfinite(got).all()
    excess = np.abs(got - want) - tolerance
    assert (excess <= 0).all(), f"max excess {excess.max():.4g} at {np.unravel_index(excess.argmax(), excess.shape)}"


@pytest.mark.parametrize("layout,page,hq,hkv", [("hnd", 16, 8, 2), ("nhd", 16, 8, 2), ("hnd", 64, 6, 3)])
def test_store_prefill_decode_product(dev, layout, page, hq, hkv):
    """Two chunks of ragged prompts through the pool, then decode steps whose
    outputs go through a 4-bit weight, replayed from a graph on another stream:
    every stage against the oracle for its inputs."""
    from xvllm.batch import slots_for_range
    from xvllm.kv_ops import gather_kvcache, store_kvcache
    from xvllm.layers.attention import AttnInputs, AttnMetadata, Attention, attention_context, paged_decode_attention
    from xvllm.layers.linear import mxfp4_linear

    rng, g = np.random.default_rng(page + hq), gen(page + hq)
    chunks = [[37, 0, 200, 1, 64], [20, 5, 1, 0, 130]]
    lens = np.sum(chunks, 0)
    need = [-(-(int(n) + 4) // page) for n in lens]  # room for four decoded tokens
    kv = _pool(dev, hq, hkv, sum(need) + 3, page, layout)
    perm = rng.permutation(kv.num_blocks)
    table, at = np.full((len(lens), max(need)), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at : at + n]
        at += n
    bt = torch.from_numpy(table).to(dev)
    attn = Attention(hq, D, hkv, layer_id=0)
    meta = AttnMetadata(kv.kv_cache, block_scale=kv.block_scale)
    k_cache, v_cache, k_scale, v_scale = *kv.kv_cache[:, 0], *kv.block_scale[:, 0]

    done = np.zeros(len(lens), int)
    for step, new in enumerate(chunks):
        rows = [b for b in range(len(lens)) if new[b]]
        total = sum(new)
        q, k, v = (randn_bf16((total, h, D), g) for h in (hq, hkv, hkv))
        slots = np.concatenate([slots_for_range(table[b], done[b], done[b] + new[b], page) for b in rows])
        ends = [int(done[b] + new[b]) for b in rows]
        cu_q = torch.tensor([0, *np.cumsum([new[b] for b in rows])], dtype=torch.int32, device=dev)
        cu_k = torch.tensor([0, *np.cumsum(ends)], dtype=torch.int32, device=dev)
        a = AttnInputs(torch.from_numpy(slots).to(dev), True, cu_q, cu_k, max(new), max(ends),
                       block_tables=bt[rows] if step else None)
        with attention_context(meta):
            out = attn(q.to(dev).flatten(1), k.to(dev).flatten(1), v.to(dev).flatten(1), a)
        for i, t in enumerate((k, v)):  # the store: codes and scales of these slots
            c, s = O.quantize_fp4(f32(t))
            assert np.array_equal(_bytes(kv.kv_cache[i, 0]).reshape(-1, hkv, D // 2)[slots], c)
            assert np.array_equal(_bytes(kv.block_scale[i, 0]).reshape(-1, hkv, D // 32)[slots], s)
        if step:  # over the pages: the read back's values, what is behind it untouched
            kd, vd = gather_kvcache(k_cache, v_cache, bt[rows], cu_k, sum(ends), k_block_scale=k_scale,
                                    v_block_scale=v_scale)
            kd, vd = (t.double().cpu().numpy() for t in (kd, vd))
            pools = [_values(kv, i, 0) for i in (0, 1)]
            for j, b in enumerate(rows):
                ids = slots_for_range(table[b], 0, ends[j], page)
                span = slice(int(cu_k[j]), int(cu_k[j + 1]))
                for got, pool in ((kd, pools[0]), (vd, pools[1])):
                    assert np.array_equal(got[span], pool.reshape(-1, hkv, D)[ids])
        else:
            kd, vd = k.double().numpy(), v.double().numpy()
        for j, b in enumerate(rows):
            want, _ = _attend(q.double().numpy()[int(cu_q[j]) : int(cu_q[j + 1])], kd[int(cu_k[j]) : int(cu_k[j + 1])],
                              vd[int(cu_k[j]) : int(cu_k[j + 1])])
            _close(out.view(total, hq, D)[int(cu_q[j]) : int(cu_q[j + 1])], want, 2e-2 + 2e-2 * np.abs(want))
        done += new

    # decode: rows 1 .. n and a padding row, the static buffers of a graph
    n, bsz = 200, len(lens) + 1
    wc = rng.integers(0, 256, (n, hq * D // 2), dtype=np.uint8)
    ws = rng.integers(118, 123, (n, hq * D // 32)).astype(np.uint8)
    w, s = as_codes(torch.from_numpy(wc).to(dev)), as_scales(torch.from_numpy(ws).to(dev))
    pad = torch.full((1, bt.shape[1]), -1, dtype=torch.int32, device=dev)
    q, k, v = (torch.zeros((bsz, h, D), dtype=torch.bfloat16, device=dev) for h in (hq, hkv, hkv))
    slots = torch.full((bsz,), -1, dtype=torch.int32, device=dev)
    ctx = torch.zeros(bsz, dtype=torch.int32, device=dev)
    tables = torch.cat([bt, pad])

    def step():
        store_kvcache(k, v, k_cache, v_cache, slots, k_block_scale=k_scale, v_block_scale=v_scale)
        o = paged_decode_attention(q, k_cache, v_cache, tables, ctx, hq, hkv, D, k_block_scale=k_scale,
                                   v_block_scale=v_scale)
        return o, mxfp4_linear(o, w, s)

    step()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        o, y = step()
    for t in range(4):
        new = [randn_bf16((bsz, h, D), g) for h in (hq, hkv, hkv)]
        for to, x in zip((q, k, v), new):
            to.copy_(x)
        slots[:-1] = torch.tensor([slots_for_range(table[b], int(done[b]), int(done[b]) + 1, page)[0]
                                   for b in range(len(lens))], dtype=torch.int32)
        ctx[:-1] = torch.from_numpy(done + 1)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        done += 1
        eager = step()  # the same store again, the same outputs
        torch.cuda.synchronize()
        assert torch.equal(o, eager[0]) and torch.equal(y, eager[1])
        assert not o[-1].any()
        pools = [_values(kv, i, 0).reshape(-1, hkv, D) for i in (0, 1)]
        for b in range(len(lens)):
            ids = slots_for_range(table[b], 0, int(done[b]), page)
            want, mag = _attend(new[0][b : b + 1].double().numpy(), pools[0][ids], pools[1][ids])
            _close(o[b], want, 4 * 2.0 ** -9 * mag)
        x, dense = o.double().cpu().numpy(), O.dequantize_fp4(wc, ws)
        want = x @ dense.T
        _close(y, want, 2.0 ** -8 * np.abs(want) + 1.01 * (hq * D + 8) * 2.0 ** -24 * (np.abs(x) @ np.abs(dense).T))


def test_prefill_over_pages_refuses_what_it_cannot_size(dev):
    from xvllm.layers.attention import prefill_attention

    kv = _pool(dev, 8, 2, 4, 16, "hnd")
    q = torch.zeros((3, 8 * D), dtype=torch.bfloat16, device=dev)
    cu = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    bt = torch.zeros((1, 2), dtype=torch.int32, device=dev)
    args = (q, None, None, cu, cu, 3, 8, 2, D, kv.kv_cache[0, 0], kv.kv_cache[1, 0], bt)
    scales = dict(k_block_scale=kv.block_scale[0, 0], v_block_scale=kv.block_scale[1, 0])
    with pytest.raises(ValueError, match="max_seqlen_k"):
        prefill_attention(*args, **scales)
    with pytest.raises(ValueError, match="block_scale"):
        prefill_attention(*args, max_seqlen_k=3)
    with pytest.raises(ValueError, match="not 4-bit pages"):
        prefill_attention(*args[:7], 4, *args[8:], max_seqlen_k=3, **scales)


def test_layer_decode_on_a_4bit_pool(dev):
    """A decoder layer over 4-bit pages: what it stores is the oracle's
    quantisation of the keys and values that Attention was given, other rows
    stay, attention and the rest of the layer match the oracle."""
    from test_gpu_model import D as HEAD, EPS, FFN, HIDDEN, HKV, HQ, _layer_case
    from xvllm.config import Qwen3Shape
    from xvllm.layers.attention import AttnInputs, AttnMetadata, attention_context
    from xvllm.layers.rotary import build_cos_sin_cache
    from xvllm.models.qwen3 import Qwen3DecoderLayer

    ctx, bt, w, kc, vc, hidden, pos, slots = _layer_case(seed=8)
    stored = [O.quantize_fp4(f32(t)) for t in (kc, vc)]
    cfg = Qwen3Shape(HIDDEN, HQ, HKV, HEAD, FFN, 1, max_position_embeddings=4096)
    with torch.device(dev):
        layer = Qwen3DecoderLayer(cfg, 0).to(torch.bfloat16)
        layer.self_attn.rotary_emb.cos_sin_cache = build_cos_sin_cache(HEAD, 4096, 1e6).to(dev)
    with torch.no_grad():
        for name, mod in (("qkv_proj", layer.self_attn), ("o_proj", layer.self_attn), ("gate_up_proj", layer.mlp),
                          ("down_proj", layer.mlp)):
            getattr(mod, name).copy_(w[name])
        layer.self_attn.q_norm.weight.copy_(w["q_norm"])
        layer.self_attn.k_norm.weight.copy_(w["k_norm"])
        layer.input_layernorm.weight.copy_(w["input_layernorm"])
        layer.post_attention_layernorm.weight.copy_(w["post_attention_layernorm"])
    pool = torch.stack([torch.from_numpy(c) for c, _ in stored])[:, None].to(dev)
    scale = torch.stack([torch.from_numpy(s) for _, s in stored])[:, None].to(dev)
    attn_in = AttnInputs(slot_mapping=slots.to(dev), is_prefill=False,
                         cache_seqlens=torch.tensor(ctx, dtype=torch.int32, device=dev), block_tables=bt.to(dev))
    seen = {}
    orig = layer.self_attn.attn.forward

    def spy(q, k, v, a):
        seen.update(q=q, k=k, v=v, out=orig(q, k, v, a))
        return seen["out"]

    layer.self_attn.attn.forward = spy
    with torch.no_grad(), attention_context(AttnMetadata(as_codes(pool), block_scale=as_scales(scale))):
        h, res = layer(pos.to(dev), hidden.to(dev), None, attn_in)
    torch.cuda.synchronize()
    for i, name in enumerate("kv"):
        c, s = (a.copy() for a in stored[i])
        qc, qs = O.quantize_fp4(f32(seen[name]).reshape(-1, HKV, HEAD))
        c.reshape(-1, HKV, HEAD // 2)[slots], s.reshape(-1, HKV, HEAD // 32)[slots] = qc, qs
        assert np.array_equal(_bytes(pool[i, 0]), c) and np.array_equal(_bytes(scale[i, 0]), s)
    pages = [O.dequantize_fp4(_bytes(pool[i, 0]), _bytes(scale[i, 0])).reshape(-1, HKV, HEAD) for i in (0, 1)]
    q = seen["q"].double().cpu().numpy().reshape(-1, HQ, HEAD)
    for b, n in enumerate(ctx):
        ids = (bt[b].numpy()[np.arange(n) // 16] * 16 + np.arange(n) % 16)
        want, mag = _attend(q[b : b + 1], pages[0][ids], pages[1][ids])
        _close(seen["out"][b], want, 4 * 2.0 ** -9 * mag)
    # q, k, v from the oracle's layer, and the rest of the layer from the attention's own output
    wn = {name: f32(t) for name, t in w.items()}
    x = O.rmsnorm(f32(hidden), wn["input_layernorm"], EPS)
    qkv = OM.linear(x, wn["qkv_proj"])
    qo, ko = O.qk_norm_rope(qkv[:, : HQ * HEAD].reshape(-1, HQ, HEAD),
                            qkv[:, HQ * HEAD : (HQ + HKV) * HEAD].reshape(-1, HKV, HEAD), wn["q_norm"], wn["k_norm"], EPS,
                            pos.numpy(), O.build_cos_sin_cache(HEAD, 4096, 1e6))
    for name, want in (("q", qo), ("k", ko), ("v", qkv[:, (HQ + HKV) * HEAD :])):
        want = np.asarray(want, np.float64)
        _close(seen[name].reshape(want.shape), want, 2e-2 + 2e-2 * np.abs(want))
    h_ref, r_ref = OM.post_attention(wn, f32(seen["out"]), f32(hidden), EPS)
    for got, want in ((h, h_ref), (res, r_ref)):
        _close(got, np.asarray(want, np.float64), 2e-2 + 2e-2 * np.abs(want))


def test_serving_on_a_4bit_pool(dev):
    """A small model served from a 4-bit pool (chunked prefill over the pages,
    decode under graphs, unused rows NaN): greedy ids in range and the same
    on a second run, sampled steps equal the oracle on the device's logits,
    and the pool takes 17/64 of a bf16 pool's bytes."""
    from test_gpu_serving import V, _serve
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool
    from xvllm.models import Qwen3ForCausalLM

    cfg = Qwen3Shape(1024, 16, 8, 128, 2048, 2, vocab_size=V, max_position_embeddings=4096)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(dev):
            model = Qwen3ForCausalLM(cfg).random_init_(seed=13)
    finally:
        torch.set_default_dtype(torch.float32)
    kv = KVPool(cfg, num_blocks=512, block_size=16, device=dev, dtype=torch.float4_e2m1fn_x2)
    kv.block_scale.view(torch.uint8).fill_(255)
    assert kv.block_bytes * 64 == 17 * 2 * 2 * 16 * 8 * 128 * 2
    g = torch.Generator().manual_seed(404)
    prompts = [torch.randint(0, V, (int(n),), generator=g).tolist() for n in torch.randint(16, 301, (20,), generator=g)]
    greedy1, st = _serve(dev, model, kv, prompts, 12, None, 0, check=False)
    greedy2, _ = _serve(dev, model, kv, prompts, 12, None, 0, check=False)
    assert greedy1 == greedy2, "greedy serving on the 4-bit pool is not reproducible"
    assert st.steps > 12 and st.prefill_tokens == sum(len(p) for p in prompts)
    sampled, _ = _serve(dev, model, kv, prompts, 12, dict(temperature=0.7, top_p=0.9, top_k=50), 7, check=True)
    assert all(0 <= t < V for o in sampled + greedy1 for t in o)


@pytest.mark.parametrize("rows", [3, 64])
def test_decode_layer_takes_buffers_of_a_larger_batch(dev, rows):
    """Positions and slots longer than the batch: its own rows are read, as on the other pools."""
    from xvllm.config import Qwen3Shape
    from xvllm.layers.attention import AttnInputs, AttnMetadata, attention_context
    from xvllm.models.qwen3 import Qwen3Attention

    g = torch.Generator(device=dev).manual_seed(rows)
    with torch.device(dev):
        layer = Qwen3Attention(Qwen3Shape(1024, 16, 8, D, 2048, 1, max_position_embeddings=1024), 0).to(torch.bfloat16)
    with torch.no_grad():
        layer.qkv_proj.normal_(0.0, 0.02, generator=g)
        layer.o_proj.normal_(0.0, 0.02, generator=g)
        hidden = torch.randn((rows, 1024), generator=g, device=dev).to(torch.bfloat16)
    lens = torch.randint(1, 64, (rows,), generator=g, device=dev, dtype=torch.int32)
    bt = torch.arange(4 * rows, dtype=torch.int32, device=dev).view(rows, 4)
    last = (lens - 1).long()
    slots = bt.gather(1, (last // 16)[:, None])[:, 0] * 16 + (last % 16).to(torch.int32)
    outs = []
    for slack in (0, 9):
        kv = _pool(dev, 16, 8, 4 * rows, 16, "hnd")
        kv.block_scale.view(torch.uint8).fill_(124)
        attn = AttnInputs(torch.cat([slots, slots.new_full((slack,), -1)]), False, block_tables=bt, cache_seqlens=lens)
        with torch.no_grad(), attention_context(AttnMetadata(kv.kv_cache, block_scale=kv.block_scale)):
            out = layer(torch.cat([last, last.new_zeros(slack)]), hidden, attn)
        outs.append((getattr(out, "parts", out), kv.kv_cache.view(torch.uint8), kv.block_scale.view(torch.uint8)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
