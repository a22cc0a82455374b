"""A runner whose context is longer than its model's max_position_embeddings:
the rotary tables grow with it, so that no step reads past one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(dev, positions):
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool
    from xvllm.models import Qwen3ForCausalLM

    cfg = Qwen3Shape(512, 8, 4, 128, 512, 2, vocab_size=1000, max_position_embeddings=positions)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(dev):
            model = Qwen3ForCausalLM(cfg).random_init_(seed=3)
            kv = KVPool(cfg, num_blocks=64, block_size=16, device=dev, dtype=torch.bfloat16)
    finally:
        torch.set_default_dtype(torch.float32)
    kv.kv_cache.zero_()
    return model, kv


def _serve(model, kv, prompts, context, **kw):
    from xvllm.model_runner import ModelRunner
    from xvllm.serving import serve

    runner = ModelRunner(model, kv, max_num_seqs=2, max_num_batched_tokens=256, context_len=context, **kw)
    outs, _ = serve(runner, prompts, 20, max_num_seqs=2, max_num_batched_tokens=256)
    tables = [layer.self_attn.rotary_emb.cos_sin_cache for layer in model.model.layers]
    return runner, outs, tables


@pytest.mark.parametrize("eager", [False, True])
def test_a_context_past_the_table(dev, eager):
    """Prompts of 120 and 30 tokens and 20 more each, of a model with 128 positions and of one with 160."""
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (120, 30)]
    runner, got, tables = _serve(*_model(dev, 128), prompts, 150, enforce_eager=eager)
    assert all(t.shape == (160, 128) and t.is_cuda for t in tables) and runner.batch.max_positions == 160
    longer, want, same = _serve(*_model(dev, 160), prompts, 150, enforce_eager=eager)
    assert all(torch.equal(a, b) for a, b in zip(tables, same))
    assert got == want
    for r in (runner, longer):
        r.destroy()


def test_an_earlier_runner_keeps_its_table(dev):
    """A second runner with a longer context grows the tables; the first one's recorded steps still read theirs."""
    model, kv = _model(dev, 64)
    prompts = [[5, 6, 7], [9] * 20]
    first, want, before = _serve(model, kv, prompts, 64)
    second, got, after = _serve(model, kv, prompts, 200)
    assert got == want and all(len(b) == 64 and len(a) == 208 for b, a in zip(before, after))
    del before
    junk = [torch.full((64, 128), float("nan"), device=dev) for _ in range(64)]  # takes what the allocator has free
    from xvllm.serving import serve

    assert serve(first, prompts, 20, max_num_seqs=2, max_num_batched_tokens=256)[0] == want
    del junk
    for r in (first, second):
        r.destroy()
