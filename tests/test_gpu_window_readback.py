"""Windowed prefill over 8-bit and 4-bit pages reads back the keys that some
query sees and nothing else: entries of other blocks may be gone."""
import pytest
import torch

from rows_cases import D, NAN

pytestmark = pytest.mark.gpu

LENS, NEW = [300, 64, 17, 450, 40, 5], [40, 64, 1, 129, 0, 9]  # the last: more queries than keys
CASES = [(30, 4, 16), (1, 0, 16), (100, 70, 48), (25, 17, 48), (2**31 - 1, 0, 16), (500, 3, 16)]


def _pool(dev, fmt, block, hkv, seed=0):
    """Pages of random keys and values, a full table, and the keywords that go with the format."""
    from xvllm.kv_ops import store_kvcache

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in LENS]
    perm = torch.randperm(sum(need), generator=g).to(torch.int32)
    bt = torch.zeros(len(LENS), max(need), dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        bt[b, :k] = perm[at : at + k]
        at += k
    nb = sum(need)
    kv = torch.randn(2, nb * block, hkv, D, generator=g).to(torch.bfloat16).to(dev)
    slots = torch.arange(nb * block, dtype=torch.int32, device=dev)
    if fmt == "fp8":
        pool = torch.zeros(2, nb, block, hkv, D, device=dev).to(torch.float8_e4m3fn)
        store_kvcache(kv[0], kv[1], pool[0], pool[1], slots, k_scale=0.02, v_scale=0.02)
        kw = dict(max_seqlen_k=max(LENS), kv_scale=(0.02, 0.02))
    else:
        pool = torch.zeros(2, nb, block, hkv, D // 2, dtype=torch.uint8, device=dev).view(torch.float4_e2m1fn_x2)
        sc = torch.zeros(2, nb, block, hkv, D // 32, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
        kw = dict(k_block_scale=sc[0], v_block_scale=sc[1])
        store_kvcache(kv[0], kv[1], pool[0], pool[1], slots, **kw)
        kw["total_seqlen_k"] = sum(LENS)
    return pool, bt, kw


def _seen(window, sinks):
    """Each sequence's keys that some query sees."""
    out = []
    for n, m in zip(LENS, NEW):
        j = torch.arange(n)
        out.append(((j < sinks) | (j > n - m - window)) & (m > 0))
    return out


def _cu(x, dev):
    return torch.tensor([0] + x, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("window,sinks,block", CASES)
def test_blocks_that_no_query_sees_may_be_gone(dev, fmt, window, sinks, block):
    from xvllm.layers.attention import prefill_attention

    hq, hkv = 8, 4
    pool, bt, kw = _pool(dev, fmt, block, hkv)
    q = torch.randn(sum(NEW), hq * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    run = lambda table: prefill_attention(q, None, None, _cu(NEW, dev), _cu(LENS, dev), max(NEW), hq, hkv, D, k_cache=pool[0],
                                          v_cache=pool[1], block_tables=table.to(dev), window=window, sink_tokens=sinks, **kw)
    want = run(bt)
    gone, left = bt.clone(), 0
    for b, seen in enumerate(_seen(window, sinks)):
        for i in range(bt.shape[1]):
            if not seen[i * block : (i + 1) * block].any():
                gone[b, i] = -1
                left += i < -(-LENS[b] // block)
    assert left > 0
    rows = len(LENS) * max(LENS) if fmt == "fp8" else sum(LENS)
    junk = [torch.full((2, rows, hkv, D), NAN, dtype=torch.bfloat16, device=dev) for _ in range(3)]  # rows left as they are are NaN
    del junk
    assert torch.equal(run(gone), want) and torch.isfinite(want).all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("window,sinks,block", CASES)
def test_rows_that_no_query_sees_stay(dev, fmt, window, sinks, block):
    from xvllm._torch_glue import call, ptr
    from xvllm.kv_ops import gather_kvcache

    hkv = 4
    pool, bt, kw = _pool(dev, fmt, block, hkv, seed=2)
    bt, cu_q, cu_k = bt.to(dev), _cu(NEW, dev), _cu(LENS, dev)
    out = torch.full((2, sum(LENS), hkv, D), 7.0, dtype=torch.bfloat16, device=dev)
    if fmt == "fp8":
        pages = (ptr(pool[0]), ptr(pool[1]), *pool.stride()[1:4], ptr(bt), bt.stride(0), block)
        rest = (len(LENS), max(LENS), hkv, D)
        tail = (0.02, 0.02, ptr(out[0]), ptr(out[1]), hkv * D)
        call("xv_gather_kv_fp8", 0, *pages, ptr(cu_k), *rest, *tail)
        want = out.clone()
        out.fill_(7.0)
        call("xv_window_gather_kv_fp8", 0, *pages, ptr(cu_q), ptr(cu_k), *rest, window, sinks, *tail)
    else:
        sc = {k: v for k, v in kw.items() if k != "total_seqlen_k"}
        want = torch.stack(gather_kvcache(pool[0], pool[1], bt, cu_k, sum(LENS), **sc))
        got = gather_kvcache(pool[0], pool[1], bt, cu_k, sum(LENS), out=(out[0], out[1]), cu_seqlens_q=cu_q, window=window,
                             sink_tokens=sinks, **sc)
        assert got[0].data_ptr() == out.data_ptr()
    seen = torch.cat(_seen(window, sinks)).to(dev)
    assert torch.equal(out[:, seen], want[:, seen]) and (out[:, ~seen] == 7.0).all()


@pytest.mark.parametrize("fmt", ["fp8", "fp4"])
@pytest.mark.parametrize("window", [0, 30])
def test_lengths_in_a_larger_batch_s_buffer(dev, fmt, window):
    """cu_seqlens_k may be longer than the sequences there are."""
    from xvllm.layers.attention import prefill_attention

    hq, hkv = 8, 4
    pool, bt, kw = _pool(dev, fmt, 16, hkv, seed=4)
    q = torch.randn(sum(NEW), hq * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    run = lambda cu_k: prefill_attention(q, None, None, _cu(NEW, dev), cu_k, max(NEW), hq, hkv, D, k_cache=pool[0], v_cache=pool[1],
                                         block_tables=bt.to(dev), window=window, **kw)
    assert torch.equal(run(_cu(LENS + [7, 7], dev)), run(_cu(LENS, dev)))
