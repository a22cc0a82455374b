"""Sliding windows and drafted trees on the framework's own path: the Attention
module over a pool, the Qwen3 model and its runner, and a draft step whose maps,
store and attention run one after the other on the device."""
import pytest
import torch

from rows_cases import D, attend, check, random_tree, tree_seen, window_mask

pytestmark = pytest.mark.gpu


def _qkv(n, hq, hkv, seed, dev):
    x = torch.randn(n, (hq + 2 * hkv) * D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)
    return x[:, : hq * D], x[:, hq * D : (hq + hkv) * D], x[:, (hq + hkv) * D :]


def _slots(bt, b, start, end, block=16):
    p = torch.arange(start, end)
    return (bt[b].cpu().long()[p // block] * block + p % block).to(torch.int32)


@pytest.mark.parametrize("hq,hkv", [(16, 8), (8, 1)])
def test_attention_module(dev, hq, hkv):
    """A prompt, a chunk over it and two decode steps of two sequences, stored and attended through vllm::attention."""
    from xvllm.layers import Attention, AttnInputs, AttnMetadata, attention_context

    window, sinks = 40, 5
    attn = Attention(hq, D, hkv, window=window, sink_tokens=sinks)
    pool = torch.full((2, 1, 40, 16, hkv, D), float("nan"), dtype=torch.bfloat16, device=dev)
    bt = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:36].view(2, 18).to(torch.int32).to(dev)
    kept = [[[], []], [[], []]]
    steps = [((70, 33), True), ((60, 1), True), ((1, 1), False), ((1, 1), False)]
    lens = [0, 0]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    with attention_context(AttnMetadata(pool)):
        for step, (new, prefill) in enumerate(steps):
            n = sum(new)
            q, k, v = _qkv(n, hq, hkv, step, dev)
            slots = torch.cat([_slots(bt, b, lens[b], lens[b] + new[b]) for b in range(2)]).to(dev)
            ends = [a + b for a, b in zip(lens, new)]
            cu = lambda x: i32([0, x[0], x[0] + x[1]])
            if prefill:
                inp = AttnInputs(slots, True, cu(new), cu(ends), max(new), max(ends), bt if step else None)
            else:
                inp = AttnInputs(slots, False, block_tables=bt, cache_seqlens=i32(ends))
            got = attn(q, k, v, inp)
            at = 0
            for b in range(2):
                rows = slice(at, at + new[b])
                kept[b][0].append(k[rows].reshape(-1, hkv, D))
                kept[b][1].append(v[rows].reshape(-1, hkv, D))
                kk, vv = (torch.cat(x) for x in kept[b])
                seen = window_mask(list(range(lens[b], ends[b])), ends[b], window, sinks, dev)
                want, tol = attend(q[rows].reshape(-1, hq, D), kk, vv, seen)
                check(got[rows], want, tol, f"step {step} sequence {b}")
                at += new[b]
            lens = ends


def _model(dev, seed=3, **kw):
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool
    from xvllm.models import Qwen3ForCausalLM

    cfg = Qwen3Shape(512, 8, 2, D, 1024, 2, vocab_size=1000, max_position_embeddings=2048, **kw)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(dev):
            model = Qwen3ForCausalLM(cfg).random_init_(seed=seed)
            kv = KVPool(cfg, num_blocks=256, block_size=16, device=dev, dtype=torch.bfloat16)
    finally:
        torch.set_default_dtype(torch.float32)
    kv.kv_cache.zero_()
    return model, kv


def test_serving_with_windows(dev):
    """One windowed layer of two, served over chunked prefills and decode graphs: what the eager runner generates."""
    from xvllm.model_runner import ModelRunner
    from xvllm.serving import serve

    model, kv = _model(dev, sliding_window=48, attention_sinks=4, max_window_layers=1)
    assert [layer.self_attn.attn.window for layer in model.model.layers] == [0, 48]
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (150, 9, 77, 200)]
    outs = []
    for eager in (True, False):
        runner = ModelRunner(model, kv, max_num_seqs=4, max_num_batched_tokens=96, context_len=256, enforce_eager=eager)
        outs.append(serve(runner, prompts, 12, max_num_seqs=4, max_num_batched_tokens=96, num_pages=128)[0])
        runner.destroy()
    assert outs[0] == outs[1]


def test_windowed_model_forgets(dev):
    """With both layers windowed, tokens more than two windows back leave the last hidden state as it is, bit by bit."""
    from xvllm.layers import AttnInputs, AttnMetadata, attention_context

    model, kv = _model(dev, sliding_window=20)
    n = 90
    ids = torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(2)).to(dev)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    inp = AttnInputs(torch.arange(n, dtype=torch.int32, device=dev), True, cu, cu, n, n)
    outs = []
    with torch.no_grad(), attention_context(AttnMetadata(kv.kv_cache)):
        for first in (ids[0], (ids[0] + 1) % 1000):
            x = ids.clone()
            x[: n - 39] = first  # the last token reaches 19 + 19 back
            outs.append(model(x, torch.arange(n, device=dev), inp)[-1])
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("block", [16, 48])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (8, 8)])
def test_draft_steps(dev, block, hq, hkv):
    """Two draft steps in a row: tables, slots and positions from lengths on the device, the nodes' K and V stored, the
    trees attended; in between the accepted path's length is all that the device is told."""
    from xvllm.kv_ops import store_kvcache, step_maps
    from xvllm.layers.attention import prefill_attention, tree_attention, tree_masks

    lens, rows = [100, 0, 37, 260], 4
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    width = 330 // block + 2
    bt = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(4 * width, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(dev)
    cache = torch.full((2, 4 * width, block, hkv, D), float("nan"), dtype=torch.bfloat16, device=dev)
    seq, head = torch.zeros(rows, dtype=torch.int32, device=dev), i32([0])
    # the prompts, through the same maps
    m = step_maps(seq, i32(lens), bt, free, block, sum(lens), free_head=head)
    q, k, v = _qkv(sum(lens), hq, hkv, 1, dev)
    heads = lambda t: t.unflatten(1, (hkv, D))
    store_kvcache(heads(k), heads(v), cache[0], cache[1], m.slot_mapping)
    got = prefill_attention(q, None, None, m.cu_seqlens_q, m.cu_seqlens_k, max(lens), hq, hkv, D, k_cache=cache[0], v_cache=cache[1],
                            block_tables=bt, window=64, sink_tokens=2)
    kept, at = [], 0
    for b, n in enumerate(lens):
        kept.append([heads(k[at : at + n]), heads(v[at : at + n])])
        if n:
            want, tol = attend(q[at : at + n].view(n, hq, D), *kept[b], window_mask(list(range(n)), n, 64, 2, dev))
            check(got[at : at + n], want, tol, f"prompt {b}")
        at += n
    seq, head, own = m.cache_seqlens, m.free_head, m.row_blocks
    for step in range(2):
        trees = [random_tree(n, 10 * step + n) for n in ((7, 30, 0, 12), (1, 16, 25, 20))[step]]
        nodes = [len(t) for t in trees]
        masks, depths = zip(*(tree_masks(t) for t in trees))
        mask, depth = torch.cat(masks).to(dev), torch.cat(depths).to(dev)
        m = step_maps(seq, i32(nodes), bt, free, block, sum(nodes), free_head=head, depths=depth, row_blocks=own)
        q, k, v = _qkv(sum(nodes), hq, hkv, 20 + step, dev)
        store_kvcache(heads(k), heads(v), cache[0], cache[1], m.slot_mapping)
        got = tree_attention(q, cache[0], cache[1], bt, m.cache_seqlens, m.cu_seqlens_q, mask, max(nodes), hq, hkv, D)
        at = 0
        for b, (n, tree) in enumerate(zip(nodes, trees)):
            ctx = kept[b][0].shape[0]
            assert m.positions[at : at + n].tolist() == [ctx + d for d in depths[b].tolist()]
            if n:
                seen = torch.cat([torch.ones(n, ctx, dtype=torch.bool), tree_seen(tree)], dim=1).to(dev)
                new = [heads(t[at : at + n]) for t in (k, v)]
                want, tol = attend(q[at : at + n].view(n, hq, D), *(torch.cat([a, b2]) for a, b2 in zip(kept[b], new)), seen)
                check(got[at : at + n], want, tol, f"step {step} sequence {b}")
                # the first nodes that form a chain are accepted: they are where the sequence's next tokens belong
                chain = 1
                while chain < n and tree[chain] == chain - 1:
                    chain += 1
                kept[b] = [torch.cat([a, b2[:chain]]) for a, b2 in zip(kept[b], new)]
            at += n
        # the device is told the lengths alone: blocks that held rejected nodes only stay the row's
        seq, head, own = i32([x[0].shape[0] for x in kept]), m.free_head, m.row_blocks
    taken = int(head)
    assert taken == sum(own.tolist()) and sorted(p for r, n in zip(bt.tolist(), own.tolist()) for p in r[:n]) == sorted(free[:taken].tolist())


def test_model_checks_a_tree(dev):
    """A step of the Qwen3 model over drafted trees: each node's hidden state is that of decoding its path token by token
    (to the framework's 2e-2, for a layer's sums run in another order)."""
    from xvllm.layers import AttnInputs, AttnMetadata, TreePlan, attention_context
    from xvllm.layers.attention import tree_masks

    model, kv = _model(dev)
    g = torch.Generator().manual_seed(8)
    ctx, parents = 50, [-1, 0, 0, 1, 1, 2, -1, 6, 3]
    n = len(parents)
    prompt = torch.randint(0, 1000, (ctx,), generator=g).to(dev)
    drafted = torch.randint(0, 1000, (n,), generator=g).to(dev)
    mask, depths = tree_masks(parents)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    bt = torch.arange(8, dtype=torch.int32, device=dev).view(1, 8)
    with torch.no_grad(), attention_context(AttnMetadata(kv.kv_cache)):
        cu = i32([0, ctx])
        model(prompt, torch.arange(ctx, device=dev), AttnInputs(torch.arange(ctx, dtype=torch.int32, device=dev), True, cu, cu, ctx, ctx))
        before = kv.kv_cache.clone()
        inp = AttnInputs(torch.arange(ctx, ctx + n, dtype=torch.int32, device=dev), False, block_tables=bt, cache_seqlens=i32([ctx + n]),
                         tree=TreePlan(i32([0, n]), mask.to(dev), n))
        got = model(drafted, ctx + depths.to(dev).long(), inp)
        for leaf in range(n):
            path = []
            while leaf >= 0:
                path.insert(0, leaf)
                leaf = parents[leaf]
            kv.kv_cache.copy_(before)
            for i, node in enumerate(path):
                p = ctx + i
                one = model(drafted[node : node + 1], torch.tensor([p], device=dev),
                            AttnInputs(i32([p]), False, block_tables=bt, cache_seqlens=i32([p + 1])))
            err = (got[path[-1]].float() - one[0].float()).abs()
            assert (err <= 2e-2 + 2e-2 * one[0].float().abs()).all(), f"node {path[-1]}: {float(err.max()):.3g}"
