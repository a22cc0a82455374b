"""A sliding window as long as all that a block table's row has room for hides
nothing: 8-bit and 4-bit pools, shared-prefix plans and tree plans go with it
as without a window."""
import pytest
import torch

BF16, I32, D = torch.bfloat16, torch.int32, 128


@pytest.mark.parametrize("window,allowed", [(63, False), (64, True), (1 << 30, True)])
@pytest.mark.parametrize("plan", ["tree", "cascade"])
def test_plans(monkeypatch, plan, window, allowed):
    from xvllm.layers import AttnInputs, AttnMetadata, TreePlan, attention_context
    from xvllm.layers import attention as A

    for name in ("tree_attention", "cascade_decode_attention"):
        monkeypatch.setattr(A, name, lambda *a, _n=name, **k: _n)
    i = torch.zeros(3, dtype=I32)
    x, table = torch.zeros(2, 512, dtype=BF16), torch.zeros(2, 4, dtype=I32)
    kw = {"tree": TreePlan(i, i.long(), 2)} if plan == "tree" else {"cascade": A.CascadePlan(i, i, i, 1, 1)}
    inputs = AttnInputs(None, False, block_tables=table, cache_seqlens=i, **kw)
    with attention_context(AttnMetadata(torch.zeros(2, 1, 4, 16, 2, D, dtype=BF16))):
        attn = A.Attention(4, D, 2, window=window)
        if allowed:
            assert attn(x, x, x, inputs).startswith(plan)
        else:
            with pytest.raises(ValueError, match="exclude"):
                attn(x, x, x, inputs)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float4_e2m1fn_x2])
def test_other_pages(monkeypatch, dtype):
    from xvllm.layers import attention as A

    monkeypatch.setattr(A, "_window_decode", lambda *a: "window")
    monkeypatch.setattr(A, "_paged_decode_fp4", lambda *a: "plain")

    def plain(*t):
        raise KeyError("plain")

    monkeypatch.setattr(A, "require_cuda", plain)  # the plain fp8 path's first step
    cache = torch.zeros(4, 16, 2, D if dtype == torch.float8_e4m3fn else D // 2, dtype=torch.uint8).view(dtype)
    q, bt, sl = torch.zeros(1, 256, dtype=BF16), torch.zeros(1, 4, dtype=I32), torch.zeros(1, dtype=I32)
    run = lambda w, c=cache: A.paged_decode_attention(q, c, c, bt, sl, 2, 2, D, window=w, sink_tokens=3)
    assert run(63) == "window"
    assert run(64, torch.zeros(4, 16, 2, D, dtype=BF16)) == "window"
    if dtype == torch.float8_e4m3fn:
        with pytest.raises(KeyError, match="plain"):
            run(64)
    else:
        assert run(64) == "plain"


@pytest.mark.gpu
def test_fp8_decode_and_runner(dev):
    """The outputs of a call without a window, and a runner over an fp8 pool that serves what one without windows does."""
    from xvllm.config import Qwen3Shape
    from xvllm.kv_ops import store_kvcache
    from xvllm.kv_pool import KVPool
    from xvllm.layers.attention import paged_decode_attention
    from xvllm.model_runner import ModelRunner
    from xvllm.models import Qwen3ForCausalLM
    from xvllm.serving import serve

    cache = torch.zeros(2, 12, 16, 8, D, device=dev).to(torch.float8_e4m3fn)
    kv = torch.randn(2, 192, 8, D, device=dev).to(BF16)
    store_kvcache(kv[0], kv[1], cache[0], cache[1], torch.arange(192, dtype=I32, device=dev), k_scale=0.02, v_scale=0.02)
    q = torch.randn(3, 16 * D, device=dev).to(BF16)
    bt = torch.arange(12, dtype=I32, device=dev).view(3, 4)
    sl = torch.tensor([64, 1, 33], dtype=I32, device=dev)
    run = lambda **kw: paged_decode_attention(q, cache[0], cache[1], bt, sl, 16, 8, D, k_scale=0.02, v_scale=0.02, **kw)
    assert torch.equal(run(window=64, sink_tokens=2), run())
    with pytest.raises(TypeError, match="bf16"):
        run(window=63)

    prompts, outs = [[5, 6, 7], [9] * 40], []
    for window in (None, 160):
        cfg = Qwen3Shape(512, 8, 4, D, 512, 2, vocab_size=1000, max_position_embeddings=256, sliding_window=window)
        torch.set_default_dtype(BF16)
        try:
            with torch.device(dev):
                model = Qwen3ForCausalLM(cfg).random_init_(seed=3)
                pool = KVPool(cfg, num_blocks=32, block_size=16, device=dev, dtype=torch.float8_e4m3fn, k_scale=0.1, v_scale=0.1)
        finally:
            torch.set_default_dtype(torch.float32)
        runner = ModelRunner(model, pool, max_num_seqs=2, max_num_batched_tokens=64, context_len=150)
        outs.append(serve(runner, prompts, 20, max_num_seqs=2, max_num_batched_tokens=64)[0])
        runner.destroy()
        if window:
            with pytest.raises(ValueError, match="sliding window"):
                ModelRunner(model, pool, max_num_seqs=2, max_num_batched_tokens=64, context_len=161)
    assert outs[0] == outs[1]
