"""Rotary tables reach every position that a runner's block tables have room
for, and a batch refuses positions past them (no GPU)."""
import pytest
import torch


def _model(rows):
    from xvllm.config import Qwen3Shape
    from xvllm.models import Qwen3ForCausalLM

    return Qwen3ForCausalLM(Qwen3Shape(256, 2, 1, 128, 256, 2, vocab_size=64, max_position_embeddings=rows))


@pytest.mark.parametrize("rows,positions", [(64, 80), (4096, 4112), (1, 33)])
def test_reserved_rows_are_those_of_a_longer_table(rows, positions):
    from xvllm.layers.rotary import build_cos_sin_cache
    from xvllm.model_runner import reserve_positions

    model = _model(rows)
    old = [layer.self_attn.rotary_emb.cos_sin_cache for layer in model.model.layers]
    assert reserve_positions(model, positions) == positions
    for layer, before in zip(model.model.layers, old):
        rotary = layer.self_attn.rotary_emb
        assert torch.equal(rotary.cos_sin_cache, build_cos_sin_cache(128, positions, 1e6))
        assert rotary.cos_sin_cache.dtype == torch.float32 and dict(layer.named_buffers())["self_attn.rotary_emb.cos_sin_cache"] is rotary.cos_sin_cache
        assert rotary._outgrown[-1] is before  # a recorded graph may hold it


def test_tables_long_enough_stay():
    from xvllm.model_runner import reserve_positions

    model = _model(64)
    old = [layer.self_attn.rotary_emb.cos_sin_cache for layer in model.model.layers]
    assert reserve_positions(model, 64) == 64 and reserve_positions(model, 3) == 64
    assert all(layer.self_attn.rotary_emb.cos_sin_cache is t for layer, t in zip(model.model.layers, old))
    assert reserve_positions(object(), 9) is None and reserve_positions(torch.nn.Linear(2, 2), 9) is None


def _batch(max_positions):
    from xvllm.batch import Batch

    return Batch(max_bs=2, max_tokens=256, max_blocks=4, vocab_size=64, device=torch.device("cpu"), block_size=16,
                 max_positions=max_positions)


def test_batch_refuses_positions_past_the_table():
    from xvllm.batch import SeqSchedule

    pages = list(range(9))  # a prompt's own block list may be longer than the batch's rows
    prompt = lambda n: SeqSchedule(0, [1] * n, 0, pages)
    b = _batch(100)
    b.build_prefill([prompt(100)])
    assert int(b.positions[:100].max()) == 99
    with pytest.raises(ValueError, match="rotary table"):
        b.build_prefill([prompt(101)])
    _batch(None).build_prefill([prompt(101)])
    decode = lambda at: SeqSchedule(0, [1], at, pages[:4])
    b = _batch(60)
    b.build_decode([decode(59)])
    with pytest.raises(ValueError, match="rotary table"):
        b.build_decode([decode(60)])
