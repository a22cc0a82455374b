"""Prefill attention with a sliding window and sinks against 64-bit attention
over the keys each query sees."""
import pytest
import torch

from rows_cases import D, NAN, attend, check, paged, window_mask

pytestmark = pytest.mark.gpu


def _case(dev, lens, new, hq, hkv, window, sinks, block, layout="hnd", seed=0, scale=None, spoil=False):
    """lens: keys of each sequence, new: its queries (the last ones).  block 0: dense keys."""
    from xvllm.layers.attention import prefill_attention

    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(new), hq * D, generator=g).to(torch.bfloat16).to(dev)
    cu = [torch.tensor([0] + x, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev) for x in (new, lens)]
    k, v, bt, seqs = paged(lens, block or 16, hkv, seed + 1, layout, dev)
    if spoil:  # keys that no query sees
        for b, (n, m) in enumerate(zip(lens, new)):
            hidden = torch.arange(min(sinks, n), max(sinks, n - m + 1 - window), device=dev)
            page = bt[b].long()[hidden // block]
            k[page, hidden % block] = NAN
            v[page, hidden % block] = float("inf")
    if block:
        got = prefill_attention(q, None, None, *cu, max(new), hq, hkv, D, k_cache=k, v_cache=v, block_tables=bt,
                                softmax_scale=scale, window=window, sink_tokens=sinks)
    else:
        kv = [torch.cat([x[i] for x in seqs]).reshape(sum(lens), hkv * D) for i in range(2)]
        got = prefill_attention(q, *kv, *cu, max(new), hq, hkv, D, softmax_scale=scale, window=window, sink_tokens=sinks)
    at = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        if m:
            seen = window_mask(list(range(n - m, n)), n, window, sinks, dev)
            want, tol = attend(q[at : at + m].view(m, hq, D), seqs[b][0], seqs[b][1], seen, scale)
            check(got[at : at + m], want, tol, f"sequence {b} of {lens} / {new}, {hq}/{hkv}, window {window}, sinks {sinks}, block {block}")
        at += m


@pytest.mark.parametrize("hq,hkv", [(2, 2), (6, 3), (8, 2), (8, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (64, 0), (65, 64), (40, 70), (100, 4), (1000, 4)])
def test_prompts(dev, hq, hkv, window, sinks):
    lens = [1, 33, 64, 200, 0, 131]
    _case(dev, lens, lens, hq, hkv, window, sinks, 0, seed=window)


@pytest.mark.parametrize("hq,hkv,layout", [(4, 4, "hnd"), (8, 2, "nhd"), (8, 1, "hnd")])
@pytest.mark.parametrize("window,sinks,block", [(1, 1, 16), (30, 4, 16), (100, 70, 48), (64, 0, 256), (500, 4, 16)])
def test_chunks(dev, hq, hkv, layout, window, sinks, block):
    _case(dev, [300, 64, 17, 450, 130], [40, 64, 1, 129, 7], hq, hkv, window, sinks, block, layout, seed=window)


@pytest.mark.parametrize("window,sinks", [(700, 4), (1500, 100)])
def test_long_chunk(dev, window, sinks):
    _case(dev, [4000, 2500], [300, 70], 8, 2, window, sinks, 16, seed=3)


@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2)])
@pytest.mark.parametrize("block", [16, 48])
def test_values_no_query_sees(dev, hq, hkv, block):
    """Before a chunk's windows the pages may hold anything (a query block at a time: the chunk is one)."""
    _case(dev, [300, 90], [32, 5], hq, hkv, 40, 6, block, seed=5, spoil=True)


def test_queries_before_the_first_key(dev):
    """More queries than keys: the first see nothing and are zeros."""
    _case(dev, [3, 40], [10, 64], 8, 2, 4, 1, 16, seed=6)


def test_window_past_the_sequence_is_plain_prefill(dev):
    from xvllm.layers.attention import prefill_attention

    q = torch.randn(300, 8 * D, device=dev).to(torch.bfloat16)
    k, v = (torch.randn(300, 2 * D, device=dev).to(torch.bfloat16) for _ in range(2))
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device=dev)
    plain = prefill_attention(q, k, v, cu, cu, 200, 8, 2, D)
    for window, sinks in ((200, 0), (1 << 30, 5), (2**31 - 1, 0), (60, 200)):
        assert torch.equal(prefill_attention(q, k, v, cu, cu, 200, 8, 2, D, window=window, sink_tokens=sinks), plain)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
def test_other_page_formats(dev, fmt):
    """8-bit and 4-bit pages are read back first: the same window over the values they stand for."""
    from xvllm.kv_ops import gather_kvcache, store_kvcache
    from xvllm.layers.attention import prefill_attention

    hq, hkv, lens, new, window, sinks = 16, 4, [100, 40], [30, 40], 25, 3
    n = sum(lens)
    kv = torch.randn(2, n, hkv, D, device=dev).to(torch.bfloat16)
    bt = torch.arange(14, dtype=torch.int32, device=dev).view(2, 7)
    pos = torch.cat([torch.arange(x) for x in lens])
    seq = torch.tensor([0] * lens[0] + [1] * lens[1])
    slots = (bt.cpu()[seq, pos // 16] * 16 + pos % 16).to(torch.int32).to(dev)
    q = torch.randn(sum(new), hq * D, device=dev).to(torch.bfloat16)
    cu_q, cu_k = (torch.tensor([0, x[0], sum(x)], dtype=torch.int32, device=dev) for x in (new, lens))
    if fmt == "fp8":
        pool = torch.zeros(2, 14, 16, hkv, D, device=dev).to(torch.float8_e4m3fn)
        store_kvcache(kv[0], kv[1], pool[0], pool[1], slots, k_scale=0.02, v_scale=0.02)
        rows = pool.view(2, -1, hkv, D)[:, slots.long()].float() * 0.02
        kd, vd = rows.to(torch.bfloat16)
        kw = dict(max_seqlen_k=100, kv_scale=(0.02, 0.02))
    else:
        pool = torch.zeros(2, 14, 16, hkv, D // 2, dtype=torch.uint8, device=dev).view(torch.float4_e2m1fn_x2)
        sc = torch.zeros(2, 14, 16, hkv, D // 32, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
        kw = dict(k_block_scale=sc[0], v_block_scale=sc[1])
        store_kvcache(kv[0], kv[1], pool[0], pool[1], slots, **kw)
        kd, vd = gather_kvcache(pool[0], pool[1], bt, cu_k, n, **kw)
        kw["total_seqlen_k"] = n
    got = prefill_attention(q, None, None, cu_q, cu_k, 40, hq, hkv, D, k_cache=pool[0], v_cache=pool[1], block_tables=bt,
                            window=window, sink_tokens=sinks, **kw)
    want = prefill_attention(q, kd, vd, cu_q, cu_k, 40, hq, hkv, D, window=window, sink_tokens=sinks)
    assert torch.equal(got, want)


def test_graph_replays(dev):
    from xvllm.layers.attention import prefill_attention

    hq, hkv = 8, 2
    q = torch.randn(200, hq * D, device=dev).to(torch.bfloat16)
    k, v = (torch.randn(200, hkv * D, device=dev).to(torch.bfloat16) for _ in range(2))
    cu = torch.tensor([0, 90, 200], dtype=torch.int32, device=dev)
    body = lambda: prefill_attention(q, k, v, cu, cu, 200, hq, hkv, D, window=33, sink_tokens=2)
    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body()
    for at in (90, 0, 150, 200):
        cu[1] = at
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, body())


@pytest.mark.parametrize("block", [0, 16])
def test_many_sequences(dev, block):
    """More than 64 and more than 128 sequences, some without queries, one of them long."""
    new = [600 if i == 133 else (11 * i) % 47 for i in range(150)]
    lens = [n + (17 * i) % 60 for i, n in enumerate(new)]
    _case(dev, lens, new, 2, 2, 30, 3, block, seed=9)


def test_rows_of_eight_byte_alignment(dev):
    """The C entry's output rows need only 8 bytes, and what is around them stays."""
    from xvllm._torch_glue import call
    from xvllm.layers.attention import prefill_attention

    hq, lens = 2, [90, 37]
    q, k, v = (torch.randn(sum(lens), hq * D, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(dev) for s in range(3))
    cu = torch.tensor([0, 90, 127], dtype=torch.int32, device=dev)
    want = prefill_attention(q, k, v, cu, cu, 90, hq, hq, D, window=20, sink_tokens=1)
    wide = torch.full((sum(lens) + 1, hq * D + 12), 7.0, dtype=torch.bfloat16, device=dev)
    out = wide[:-1, 4 : 4 + hq * D]
    assert out.data_ptr() % 16 == 8
    call("xv_window_prefill_attention", 0, q.data_ptr(), hq * D, D, k.data_ptr(), v.data_ptr(), hq * D, D, None, None, 0, 0, 0, None, 0,
         cu.data_ptr(), cu.data_ptr(), out.data_ptr(), out.stride(0), 2, 90, sum(lens), hq, hq, D, 16, 20, 1, D ** -0.5)
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert (wide == 7).all()
