"""Windowed and tree attention and the step maps without a GPU: the refusals of
the C ABI (fake pointers, never dereferenced) and of the Python entry points,
masks of trees, and which layers of a config have a window."""
import pytest
import torch

INVALID = 1  # hipErrorInvalidValue
A = 0x10000
BF16, I32 = torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def lib():
    from xvllm import _C

    if not _C.lib_path().exists():
        pytest.fail("libxv_kernels.so is not built (run __graft_entry__.build())")
    return _C.lib()


ROWS = dict(q=A, qst=4096, qsh=128, kc=A, vc=A, ps=16384, ts=1024, hs=128, bt=A, bts=64, sl=A, out=A, ost=4096, ws=A, wsb=1 << 32,
            B=4, Hq=32, Hkv=8, D=128, BS=16, maxb=64, scale=0.1)
BAD_ROWS = (dict(D=64), dict(D=256), dict(BS=0), dict(BS=24), dict(Hq=12), dict(Hq=128), dict(Hq=0), dict(Hkv=0), dict(B=-1),
            dict(q=A + 8), dict(kc=A + 8), dict(vc=A + 2), dict(qst=4100), dict(qsh=130), dict(ps=16388), dict(ts=1028), dict(ts=64),
            dict(ts=1 << 27), dict(hs=132), dict(ps=-8), dict(ps=1 << 33), dict(hs=-8), dict(bts=63), dict(maxb=0),
            dict(maxb=1 << 25, bts=1 << 25), dict(bts=1 << 29), dict(out=A + 2), dict(ost=4097), dict(ws=None), dict(ws=A + 8),
            dict(wsb=1024))


def _window(lib, **kw):
    a = dict(ROWS, window=100, sinks=4)
    a.update(kw)
    return lib.xv_window_decode_attention(*[a[k] for k in ("q", "qst", "qsh", "kc", "vc", "ps", "ts", "hs", "bt", "bts", "sl", "out",
                                                           "ost", "ws", "wsb", "B", "Hq", "Hkv", "D", "BS", "maxb", "window",
                                                           "sinks", "scale")], None)


def test_window_decode_refusals(lib):
    for kw in (*BAD_ROWS, dict(window=0), dict(window=-5), dict(sinks=-1)):
        assert _window(lib, **kw) == INVALID, kw
    assert _window(lib, B=0) == 0


def _tree(lib, **kw):
    a = dict(ROWS, cu=A, mask=A, mst=1, words=1, nodes=16)
    a.update(kw)
    return lib.xv_tree_attention(*[a[k] for k in ("q", "qst", "qsh", "kc", "vc", "ps", "ts", "hs", "bt", "bts", "sl", "cu", "mask", "mst",
                                                  "words", "out", "ost", "ws", "wsb", "B", "nodes", "Hq", "Hkv", "D", "BS", "maxb",
                                                  "scale")], None)


def test_tree_refusals(lib):
    for kw in (*BAD_ROWS, dict(nodes=65), dict(nodes=-1), dict(nodes=1025, words=32, mst=32), dict(words=0), dict(words=2),
               dict(words=2, mst=1)):
        assert _tree(lib, **kw) == INVALID, kw
    assert _tree(lib, B=0) == 0 and _tree(lib, nodes=0) == 0


def test_workspace_sizes(lib):
    size = lib.xv_tree_attention_workspace_size
    for hq, hkv in ((8, 8), (32, 8), (64, 8)):
        group = hq // hkv
        last = 0
        for nodes in (1, 2, 4, 8, 16, 64, 128, 1024):
            rows = nodes * group
            n = size(16, nodes, hq, hkv)
            assert n >= rows * 512 and (rows <= 32 or n >= last // 2)  # smaller trees may take more ranges
            last = n
        assert size(300, 16, hq, hkv) == size(256, 16, hq, hkv)
    assert size(0, 16, 32, 8) == size(4, 0, 32, 8) == size(4, 16, 12, 8) == 256


def test_workspace_of_large_trees(lib):
    """As many partial rows as fill the GPU, whatever the tree's size."""
    for nodes, hq in ((33, 8), (128, 32), (300, 64), (1024, 64)):
        assert lib.xv_tree_attention_workspace_size(256, nodes, hq, 8) < 80 << 20


def _prefill(lib, **kw):
    a = dict(q=A, qst=4096, qsh=128, k=A, v=A, kvst=1024, kvsh=128, kc=None, vc=None, ps=0, ts=0, hs=0, bt=None, bts=0, cuq=A, cuk=A,
             out=A, ost=4096, B=4, maxq=512, total=900, Hq=32, Hkv=8, D=128, BS=16, window=100, sinks=4, scale=0.1)
    a.update(kw)
    return lib.xv_window_prefill_attention(*a.values(), None)


def test_window_prefill_refusals(lib):
    for kw in (dict(window=0), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(D=64), dict(Hq=24),
               dict(k=None), dict(k=A + 8), dict(kvst=1020), dict(q=A + 8), dict(qsh=130), dict(out=A + 4), dict(ost=4098),
               dict(bt=A, kc=A, vc=A, BS=40), dict(bt=A, kc=None, vc=A), dict(bt=A, kc=A + 8, vc=A), dict(maxq=32 * 65536),
               dict(B=70000), dict(B=-1), dict(total=-1), dict(total=1 << 31)):
        assert _prefill(lib, **kw) == INVALID, kw
    assert _prefill(lib, B=0) == 0 and _prefill(lib, maxq=0) == 0 and _prefill(lib, total=0) == 0


def _maps(lib, **kw):
    a = dict(old=A, new=A, own=None, rows=4, bt=A, bts=8, maxb=8, BS=16, free=A, nfree=9, head=None, depths=None, total=10, cuq=A, cuk=A, ends=A,
             own2=A, pos=A, slots=A, next=A)
    a.update(kw)
    return lib.xv_step_maps(*a.values(), None)


def test_step_maps_refusals(lib):
    for kw in (dict(rows=-1), dict(rows=4097), dict(BS=0), dict(maxb=0), dict(bts=7), dict(nfree=-1), dict(total=-1),
               dict(total=(1 << 30) + 1), dict(pos=A + 8), dict(slots=A + 4)):
        assert _maps(lib, **kw) == INVALID, kw


# ---------------------------------------------------------------- Python
def _decode(q=(2, 512), k=(4, 16, 2, 128), v=None, bt=(2, 3), sl=(2,), heads=(4, 2, 128), dtype=BF16, **kw):
    from xvllm.layers.attention import paged_decode_attention

    cache = [torch.zeros(s, dtype=dtype) for s in (k, v or k)]
    return paged_decode_attention(torch.zeros(q, dtype=kw.pop("qdtype", BF16)), *cache, torch.zeros(bt, dtype=I32),
                                  torch.zeros(sl, dtype=I32), *heads, **kw)


def test_window_decode_arguments():
    for err, kw in ((ValueError, dict(sink_tokens=4)), (ValueError, dict(window=-1)), (ValueError, dict(window=8, sink_tokens=-1)),
                    (TypeError, dict(window=8, dtype=torch.float8_e4m3fn)), (TypeError, dict(window=8, dtype=torch.float16)),
                    (TypeError, dict(window=8, qdtype=torch.float32)), (ValueError, dict(window=8, k=(4, 16, 3, 128))),
                    (ValueError, dict(window=8, k=(64, 2, 128))), (ValueError, dict(window=8, v=(4, 32, 2, 128))),
                    (ValueError, dict(window=8, q=(2, 4, 3, 64), heads=(4, 2, 128))), (ValueError, dict(window=8, bt=(1, 3))),
                    (ValueError, dict(window=8, sl=(1,))), (RuntimeError, dict(window=8))):
        with pytest.raises(err):
            _decode(**kw)


def _tree_py(t=6, b=2, mask=(6,), mdtype=torch.int64, cu=None, nodes=3, dtype=BF16, **kw):
    from xvllm.layers.attention import tree_attention

    kv = torch.zeros(4, 16, 2, 128, dtype=dtype)
    return tree_attention(torch.zeros(t, 512, dtype=BF16), kv, kv, torch.zeros(b, 3, dtype=I32), torch.zeros(b, dtype=I32),
                          torch.zeros(cu or (b + 1,), dtype=I32), torch.zeros(mask, dtype=mdtype), nodes, 4, 2, 128, **kw)


def test_tree_arguments():
    for err, kw in ((ValueError, dict(cu=(0,))), (ValueError, dict(cu=(2, 2))), (TypeError, dict(dtype=torch.float8_e4m3fn)),
                    (ValueError, dict(cu=(4,))), (RuntimeError, dict())):
        with pytest.raises(err):
            _tree_py(**kw)


def test_prefill_window_arguments():
    from xvllm.layers.attention import prefill_attention

    q, kv, cu = torch.zeros(4, 512, dtype=BF16), torch.zeros(4, 256, dtype=BF16), torch.tensor([0, 4], dtype=I32)
    for kw in (dict(sink_tokens=1), dict(window=-2), dict(window=4, sink_tokens=-1), dict(window=4, softmax_scale=0.0),
               dict(window=4, softmax_scale=-1.0)):
        with pytest.raises(ValueError):
            prefill_attention(q, kv, kv, cu, cu, 4, 4, 2, 128, **kw)


@pytest.mark.parametrize("window,sinks", [(0, 4), (-1, 0), (5, -1), (1 << 31, 0), ((1 << 32) + 5, 0), (5, 1 << 32)])
def test_window_sizes(window, sinks):
    """Sizes that a 32-bit argument would wrap are refused too."""
    from xvllm.layers.attention import Attention

    with pytest.raises(ValueError, match="window"):
        Attention(8, 128, 8, window=window, sink_tokens=sinks)


@pytest.mark.parametrize("block,total", [(0, 4), ((1 << 32) + 16, 4), (16, -1), (16, (1 << 32) + 4)])
def test_step_maps_sizes(block, total):
    from xvllm.kv_ops import step_maps

    x = torch.zeros(2, dtype=I32)
    with pytest.raises(ValueError, match="block_size"):
        step_maps(x, x, torch.zeros(2, 3, dtype=I32), x, block, total)


def test_step_maps_needs_the_gpu():
    from xvllm.kv_ops import step_maps

    x = torch.zeros(2, dtype=I32)
    with pytest.raises(RuntimeError):
        step_maps(x, x, torch.zeros(2, 3, dtype=I32), x, 16, 4)


def test_tree_masks():
    from xvllm.layers.attention import tree_masks

    mask, depths = tree_masks([-1, 0, 0, 1, -1])
    assert mask.tolist() == [[0b1], [0b11], [0b101], [0b1011], [0b10000]] and depths.tolist() == [0, 1, 1, 2, 0]
    chain, depths = tree_masks(range(-1, 69))
    assert chain.shape == (70, 2) and depths.tolist() == list(range(70))
    assert chain[63].tolist() == [-1, 0] and chain[69].tolist() == [-1, 63]
    empty, depths = tree_masks([])
    assert empty.shape == (0, 1) and depths.shape == (0,)
    for bad in ([0], [-1, 1], [-2], [-1, 0, 5]):
        with pytest.raises(ValueError):
            tree_masks(bad)


def test_layer_window():
    from types import SimpleNamespace as Cfg

    from xvllm.config import QWEN3_8B, Qwen3Shape, layer_window

    assert layer_window(QWEN3_8B, 0) == (0, 0)
    shape = Qwen3Shape(256, 2, 1, 128, 512, 4, sliding_window=64, max_window_layers=2, attention_sinks=4)
    assert [layer_window(shape, i) for i in range(4)] == [(0, 0), (0, 0), (64, 4), (64, 4)]
    # as transformers has them
    types = ["full_attention", "sliding_attention"]
    assert [layer_window(Cfg(sliding_window=64, use_sliding_window=True, layer_types=types), i) for i in range(2)] == [(0, 0), (64, 0)]
    assert layer_window(Cfg(sliding_window=64, use_sliding_window=False, max_window_layers=0), 3) == (0, 0)
    assert layer_window(Cfg(sliding_window=None, use_sliding_window=False, layer_types=["full_attention"] * 4), 3) == (0, 0)


def test_transformers_config():
    transformers = pytest.importorskip("transformers")
    from xvllm.config import layer_window

    cfg = transformers.Qwen3Config(num_hidden_layers=4, use_sliding_window=True, sliding_window=128, max_window_layers=3)
    assert [layer_window(cfg, i) for i in range(4)] == [(0, 0)] * 3 + [(128, 0)]
    assert layer_window(transformers.Qwen3Config(num_hidden_layers=4), 3) == (0, 0)


def test_attention_module_refusals():
    from xvllm.layers import Attention, AttnInputs, AttnMetadata, TreePlan, attention_context
    from xvllm.layers.attention import CascadePlan

    with pytest.raises(ValueError):
        Attention(4, 128, 2, window=0, sink_tokens=3)
    x, i = torch.zeros(2, 512, dtype=BF16), torch.zeros(3, dtype=I32)
    tree, cascade = TreePlan(i, i.long(), 2), CascadePlan(i, i, i, 1, 1)
    pool = torch.zeros(2, 1, 4, 16, 2, 128, dtype=BF16)
    with attention_context(AttnMetadata(pool)):
        for window, inputs in ((8, AttnInputs(None, False, tree=tree)), (8, AttnInputs(None, False, cascade=cascade)),
                               (0, AttnInputs(None, False, cascade=cascade, tree=tree)), (0, AttnInputs(None, True, tree=tree))):
            with pytest.raises(ValueError):
                Attention(4, 128, 2, window=window)(x, x, x, inputs)


@pytest.mark.parametrize("dtype,groups", [(torch.float8_e4m3fn, 0), (torch.float4_e2m1fn_x2, 0), (BF16, 2)])
def test_runner_refuses_windows_it_cannot_decode(dtype, groups):
    from types import SimpleNamespace

    from xvllm.config import Qwen3Shape
    from xvllm.model_runner import ModelRunner
    from xvllm.models import Qwen3ForCausalLM

    model = Qwen3ForCausalLM(Qwen3Shape(256, 2, 1, 128, 256, 1, vocab_size=64, max_position_embeddings=64, sliding_window=16))
    with pytest.raises(ValueError, match="sliding window"):
        ModelRunner(model, SimpleNamespace(dtype=dtype), cascade_groups=groups)
