"""Chunked prefill over 4-bit pages of very uneven sequences: what it reads back
is the keys there are.  Outputs against attention in 64 bits over the pages'
values, which the read back holds exactly.  Tolerance: the dense prefill rounds
weights to bf16 for the product and may sum the rounded ones, and rounds its
output, each at most 2^-8 of A, the weighted mean magnitude of the column; its
fp32 scores and sums add less than 2^-10 A (scores of |q k| scale < 100, whose
128 products are summed to 2^-24 136 of their magnitudes)."""
import numpy as np
import pytest
import torch

import oracle.ops as O
from fp4_cases import as_codes, as_scales, on_device, random_pages, tables
from helpers import gen, randn_bf16

pytestmark = pytest.mark.gpu

D = 128


@pytest.mark.parametrize("hq,hkv,page", [(8, 2, 16), (16, 8, 64)])
def test_one_long_prefix_among_short_ones(dev, hq, hkv, page):
    from xvllm.layers.attention import Attention, AttnInputs, AttnMetadata, attention_context

    rng = np.random.default_rng(hq)
    ctx = [int(c) for c in rng.integers(2, 41, 40)]
    ctx[17] = 12001
    new = [min(c, int(n)) for c, n in zip(ctx, rng.integers(1, 5, 40))]
    bt, nb = tables(rng, ctx, page)
    arrays = [*random_pages(rng, nb, page, hkv, D, 120, 124), *random_pages(rng, nb, page, hkv, D, 120, 130)]
    kc, ks, vc, vs = (on_device(a, dev, "hnd") for a in arrays)
    pool, scale = (torch.stack(pair)[:, None] for pair in ((kc, vc), (ks, vs)))
    q = randn_bf16((sum(new), hq, D), gen(hq))
    cu_q, cu_k = (torch.tensor([0, *np.cumsum(n)], dtype=torch.int32, device=dev) for n in (new, ctx))
    a = AttnInputs(None, True, cu_q, cu_k, max(new), max(ctx), block_tables=torch.from_numpy(bt).to(dev), total_seqlen_k=sum(ctx))
    qd, kv = q.to(dev).flatten(1), torch.zeros(sum(new), hkv * D, dtype=torch.bfloat16, device=dev)
    attn = Attention(hq, D, hkv)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with attention_context(AttnMetadata(as_codes(pool), block_scale=as_scales(scale))):
        out = attn(qd, kv, kv, a)
        torch.cuda.synchronize()
        # rows for 40 times the longest would take 37 times as much
        assert torch.cuda.max_memory_allocated() - before < 2 * sum(ctx) * hkv * D * 4
        every = attn(qd, kv, kv, a._replace(total_seqlen_k=0))
    torch.cuda.synchronize()
    assert torch.equal(out, every)
    got = out.double().cpu().numpy().reshape(-1, hq, D)
    at = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        ids = bt[b, : -(-c // page)]
        k, v = (O.dequantize_fp4(arrays[i][ids], arrays[i + 1][ids]).reshape(-1, hkv, D)[:c] for i in (0, 2))
        seen = np.arange(c)[None] <= c - n + np.arange(n)[:, None]
        for h in range(hq):
            x = q[at : at + n, h].double().numpy()
            s = np.where(seen, x @ k[:, h // (hq // hkv)].T * D ** -0.5, -np.inf)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            vh = v[:, h // (hq // hkv)]
            excess = float((np.abs(got[at : at + n, h] - w @ vh) - (3 * 2.0 ** -8 + 2.0 ** -10) * (w @ np.abs(vh))).max())
            assert excess <= 0, (b, h, excess)
        at += n


def test_the_runner_gives_the_keys_it_schedules(dev, monkeypatch):
    """Chunked prompts served from a 4-bit pool: every read back has as many rows as cu_seqlens_k says."""
    import xvllm.layers.attention as A
    from test_gpu_serving import V, _serve
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool
    from xvllm.models import Qwen3ForCausalLM

    cfg = Qwen3Shape(1024, 16, 8, 128, 2048, 2, vocab_size=V, max_position_embeddings=4096)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(dev):
            model = Qwen3ForCausalLM(cfg).random_init_(seed=21)
    finally:
        torch.set_default_dtype(torch.float32)
    kv = KVPool(cfg, num_blocks=512, block_size=16, device=dev, dtype=torch.float4_e2m1fn_x2)
    kv.block_scale.view(torch.uint8).fill_(255)
    rows, gather = [], A.gather_kvcache

    def spy(k_cache, v_cache, block_tables, cu_seqlens_k, total_tokens, **kw):
        rows.append((total_tokens, int(cu_seqlens_k[-1])))
        return gather(k_cache, v_cache, block_tables, cu_seqlens_k, total_tokens, **kw)

    monkeypatch.setattr(A, "gather_kvcache", spy)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, V, (int(n),), generator=g).tolist() for n in (300, 20, 400, 17, 350, 333, 200, 90)]
    _serve(dev, model, kv, prompts, 3, None, 0, check=False)
    assert len(rows) >= 2 and all(a == b for a, b in rows), rows
