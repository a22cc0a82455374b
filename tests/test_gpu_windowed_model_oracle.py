"""A served model with a windowed layer against the same weights in plain 64-bit
operations, with the window as a mask: chunked prefill, captured decode steps."""
import pytest
import torch

from rows_cases import D, window_mask

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, V = 512, 8, 2, 1000
WINDOW, SINKS = 48, 4


def _rms(x, w, eps=1e-6):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def _rope(x, table):
    """x [tokens, heads, D], table [tokens, D]: cos, then sin, of each half's angles."""
    cos, sin = table[:, None, : D // 2], table[:, None, D // 2 :]
    a, b = x[..., : D // 2], x[..., D // 2 :]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _hidden64(model, ids, windows):
    """The model's final hidden state at every token of one sequence; windows: each layer's (window, sinks), window 0: none."""
    n = len(ids)
    x = model.model.embed_tokens[torch.tensor(ids, device=model.lm_head.device)].double()
    for layer, (window, sinks) in zip(model.model.layers, windows):
        a, m = layer.self_attn, layer.mlp
        qkv = _rms(x, layer.input_layernorm.weight) @ a.qkv_proj.double().t().contiguous()
        q, k, v = (t.view(n, -1, D) for t in qkv.split([HQ * D, HKV * D, HKV * D], -1))
        table = a.rotary_emb.cos_sin_cache[:n].double()
        q, k = _rope(_rms(q, a.q_norm.weight), table), _rope(_rms(k, a.k_norm.weight), table)
        seen = window_mask(list(range(n)), n, window or n, sinks, x.device)
        out = []
        for h in range(HQ):
            s = q[:, h] @ k[:, h * HKV // HQ].t().contiguous() * D ** -0.5
            out.append(torch.softmax(s.masked_fill(~seen, -float("inf")), -1) @ v[:, h * HKV // HQ])
        x = x + torch.cat(out, -1) @ a.o_proj.double().t().contiguous()
        gate, up = (_rms(x, layer.post_attention_layernorm.weight) @ m.gate_up_proj.double().t().contiguous()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ m.down_proj.double().t().contiguous()
    return _rms(x, model.model.norm.weight)


@torch.no_grad()
def test_served_windowed_model(dev):
    """Per step relative L2 error of the hidden state below 3e-2: some 28 roundings to bf16 on the way, each by 2^-8 of a
    value at most, add up to 1.2e-2 where they are independent.  Without the window it is several times further off."""
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool
    from xvllm.model_runner import ModelRunner
    from xvllm.models import Qwen3ForCausalLM
    from xvllm.serving import serve

    cfg = Qwen3Shape(HIDDEN, HQ, HKV, D, 1024, 2, vocab_size=V, max_position_embeddings=256, sliding_window=WINDOW,
                     attention_sinks=SINKS, max_window_layers=1)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(dev):
            model = Qwen3ForCausalLM(cfg).random_init_(seed=3)
            kv = KVPool(cfg, num_blocks=32, block_size=16, device=dev, dtype=torch.bfloat16)
    finally:
        torch.set_default_dtype(torch.float32)
    kv.kv_cache.fill_(float("nan"))
    prompt, gen = torch.randint(0, V, (150,), generator=torch.Generator().manual_seed(5)).tolist(), 12
    runner = ModelRunner(model, kv, max_num_seqs=1, max_num_batched_tokens=64, context_len=176)
    steps = []

    def keep(r, n_p, n_d):
        if n_d:
            torch.cuda.synchronize()
            steps.append(r._decode_out[0].double())

    out = serve(runner, [prompt], gen, max_num_seqs=1, max_num_batched_tokens=64, after_forward=keep)[0][0]
    runner.destroy()
    assert len(steps) == gen - 1
    got = torch.stack(steps)
    ids = prompt + out[:-1]
    error = lambda windows: ((got - (want := _hidden64(model, ids, windows)[len(prompt):])).norm(dim=-1) / want.norm(dim=-1)).tolist()
    windowed, plain, no_sinks = (error([(0, 0), w]) for w in ((WINDOW, SINKS), (0, 0), (WINDOW, 0)))
    print("relative errors", max(windowed), "without the window at least", min(plain), "without sinks", min(no_sinks))
    assert max(windowed) < 3e-2, windowed
    assert min(plain) > 6e-2 and min(no_sinks) > max(windowed), (plain, no_sinks)
