"""4-bit (MXFP4) formats without a GPU: the oracle's quantiser against the
definition by exhaustive search, and the refusals of the C ABI (fake pointers,
never dereferenced) and of the Python entry points."""
import numpy as np
import pytest
import torch

import oracle.ops as O
from fp4_cases import codes, scales

INVALID = 1  # hipErrorInvalidValue
A = 0x10000


@pytest.fixture(scope="module")
def lib():
    from xvllm import _C

    if not _C.lib_path().exists():
        pytest.fail("libxv_kernels.so is not built (run __graft_entry__.build())")
    return _C.lib()


def test_oracle_quantiser_is_nearest_and_even():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 32)) * np.exp2(rng.integers(-130, 127, (500, 1)).astype(np.float64))
    x = torch.from_numpy(x).to(torch.bfloat16).double().numpy()
    x = np.where(np.isfinite(x), x, 0.0)
    x[0] = 0.0
    x[1] = 2.0 ** np.arange(-20, 12)
    x[2] = np.linspace(-6, 6, 32)
    q, s = O.quantize_fp4(x)
    v = O.dequantize_fp4(q, s)
    assert s.min() >= 1 and s.max() <= 252
    unit = np.exp2(s.astype(np.float64) - 127)[:, 0]
    for i in range(x.shape[0]):
        grid = np.concatenate([O.FP4_MAGNITUDES, -O.FP4_MAGNITUDES]) * unit[i]
        best = np.abs(grid[None, :] - x[i][:, None]).min(1)
        assert (np.abs(v[i] - x[i]) == best).all()
        top = np.abs(x[i]).max()
        if top > 0 and 1 < s[i, 0] < 252:
            assert 3.5 <= top / unit[i] < 7  # 1.75 .. 3.5 times two: the codes reach their largest or the one below
    # ties: to the even code
    ties = np.zeros((1, 32))
    ties[0, :8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    got = O.dequantize_fp4(*O.quantize_fp4(ties))[0, :8]
    assert got.tolist() == [6, 0, 1, 1, 2, 2, 4, 4]


def test_oracle_blocks_with_infinities_read_back_as_nan():
    x = np.ones((2, 64))
    x[0, 3], x[1, 40] = np.inf, np.nan
    v = O.dequantize_fp4(*O.quantize_fp4(x))
    assert np.isnan(v[0, :32]).all() and (v[0, 32:] == 1).all()
    assert (v[1, :32] == 1).all() and np.isnan(v[1, 32:]).all()


def _store(lib, **kw):
    a = dict(k=A, kst=1024, ksh=128, v=A, vst=1024, vsh=128, kc=A, vc=A, ps=8192, ts=512, hs=64, ks=A, vs=A, sps=512,
             sts=32, shs=4, BS=16, sl=A, n=4, H=8, D=128)
    a.update(kw)
    return lib.xv_store_kvcache_fp4(*a.values(), None)


def test_store_rejects_bad_arguments(lib):
    for kw in (dict(k=A + 8), dict(v=A + 2), dict(kst=1020), dict(vsh=132), dict(kc=A + 2), dict(kc=None), dict(ks=None),
               dict(ts=510), dict(hs=66), dict(BS=0), dict(BS=-16), dict(D=100), dict(D=16), dict(D=0), dict(H=0),
               dict(n=-1), dict(n=1 << 36)):
        assert _store(lib, **kw) == INVALID, kw
    assert _store(lib, n=0) == 0


def _gather(lib, **kw):
    a = dict(kc=A, vc=A, ps=8192, ts=512, hs=64, ks=A, vs=A, sps=512, sts=32, shs=4, BS=16, bt=A, bts=8, maxb=8, cu=A,
             B=4, T=100, H=8, D=128, ko=A, vo=A, ost=1024)
    a.update(kw)
    return lib.xv_gather_kv_fp4(*a.values(), None)


def test_gather_rejects_bad_arguments(lib):
    for kw in (dict(kc=None), dict(vc=A + 1), dict(ts=510), dict(BS=0), dict(D=48), dict(H=0), dict(B=-1), dict(T=-1),
               dict(T=1 << 31), dict(ko=A + 8), dict(ost=1020), dict(ost=512), dict(maxb=-1), dict(vs=None)):
        assert _gather(lib, **kw) == INVALID, kw
    assert _gather(lib, T=0) == 0 and _gather(lib, B=0) == 0


def test_python_entry_points_refuse_cpu_tensors_and_wrong_types():
    from xvllm.kv_ops import gather_kvcache, store_kvcache

    q = codes(np.zeros((4, 16, 2, 64), np.uint8))
    s = scales(np.zeros((4, 16, 2, 4), np.uint8))
    bt, cu = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    kv = torch.zeros(5, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        store_kvcache(kv, kv, q, q, torch.arange(5, dtype=torch.int32), k_block_scale=s, v_block_scale=s)
    with pytest.raises(RuntimeError, match="GPU"):
        gather_kvcache(q, q, bt, cu, 5, k_block_scale=s, v_block_scale=s)


def test_cache_checks():
    from xvllm.kv_ops import fp4_pages

    q = codes(np.zeros((4, 16, 2, 64), np.uint8))
    s = scales(np.zeros((4, 16, 2, 4), np.uint8))
    with pytest.raises(ValueError, match="needs k_block_scale"):
        fp4_pages(q, q, None, None)
    with pytest.raises(TypeError, match="scales"):
        fp4_pages(q, q, s.view(torch.uint8), s)
    with pytest.raises(TypeError, match="codes"):
        fp4_pages(q, q.view(torch.uint8), s, s)
    with pytest.raises(ValueError, match="layout"):
        fp4_pages(q, q[:3], s, s)
    with pytest.raises(ValueError, match="layout"):
        fp4_pages(q, q.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(q.dtype), s, s)
    for bad in (s[:, :, :, :3], s[:, :8]):
        with pytest.raises(ValueError, match="D/32"):
            fp4_pages(q, q, bad, bad)
    with pytest.raises(RuntimeError, match="GPU"):
        fp4_pages(q, q, s, s)


def _decode(lib, **kw):
    a = dict(q=A, qst=4096, qsh=128, kc=A, vc=A, ps=8192, ts=64, hs=1024, ks=A, vs=A, sps=512, sts=4, shs=64, bt=A, bts=256,
             sl=A, out=A, ost=4096, ws=A, wsb=1 << 30, B=64, Hq=32, Hkv=8, D=128, BS=16, maxb=256, scale=0.088)
    a.update(kw)
    return lib.xv_paged_decode_attention_fp4(*a.values(), None)


def test_decode_rejects_bad_arguments(lib):
    for kw in (dict(D=64), dict(BS=24), dict(BS=0), dict(Hq=24), dict(Hq=128), dict(Hq=12), dict(Hq=0), dict(Hkv=0), dict(q=A + 8),
               dict(kc=A + 8), dict(vc=A + 4), dict(qst=4100), dict(ts=72), dict(ts=48), dict(ts=0), dict(hs=1028), dict(ks=A + 2), dict(sts=6),
               dict(sts=0), dict(shs=66), dict(out=A + 2), dict(ost=4097), dict(ws=None), dict(ws=A + 8), dict(wsb=1024),
               dict(maxb=0), dict(maxb=1 << 25), dict(bts=255), dict(bts=1 << 24, maxb=256), dict(B=-1)):
        assert _decode(lib, **kw) == INVALID, kw
    assert _decode(lib, B=0) == 0


def test_decode_workspace_never_shrinks(lib):
    for hq, hkv in ((32, 8), (8, 8), (64, 8), (8, 1)):
        sizes = [lib.xv_paged_decode_fp4_workspace_size(b, hq, hkv) for b in range(0, 600)]
        assert sizes == sorted(sizes) and sizes[256] == sizes[-1]


def _gemm(lib, **kw):
    a = dict(x=A, xst=4096, w=A, wst=2048, s=A, sst=128, out=A, ost=1024, m=4, n=1024, k=4096, silu=0, ws=None, wsb=0)
    a.update(kw)
    return lib.xv_mxfp4_gemm(*a.values(), None)


def test_gemm_rejects_bad_arguments(lib):
    for kw in (dict(x=None), dict(x=A + 8), dict(xst=4092), dict(xst=4088), dict(w=A + 8), dict(w=None), dict(wst=2040),
               dict(wst=2032), dict(s=None), dict(sst=127), dict(out=None), dict(out=A + 1), dict(ost=1023), dict(m=-1),
               dict(n=0), dict(k=0), dict(k=4080), dict(n=1023, silu=1), dict(m=1 << 23), dict(n=(1 << 30) + 2), dict(m=200), dict(ws=A + 8)):
        assert _gemm(lib, **kw) == INVALID, kw
    assert _gemm(lib, m=0) == 0


def test_gemm_refuses_more_rows_than_a_launch_holds(lib):
    """A grid has fewer than 2^32 threads: at 96 weight rows to 512 threads no more than 805 million rows."""
    for m in (1, 16, 64, 100):
        for n in (1 << 30, 805306368, (1 << 29) + 2):
            for silu in (0, 1):
                ws = lib.xv_mxfp4_gemm_workspace_size(m, n, 32, silu)
                assert _gemm(lib, m=m, n=n, k=32, xst=32, wst=16, sst=1, ost=n, silu=silu, ws=A, wsb=ws) == INVALID, (m, n, silu)


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pool_of_4bit_pages(layout):
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool

    cfg = Qwen3Shape(256, 8, 2, 128, 512, 3)
    kv = KVPool(cfg, num_blocks=5, block_size=16, device="cpu", dtype=torch.float4_e2m1fn_x2, layout=layout)
    assert kv.kv_cache.shape == (2, 3, 5, 16, 2, 64) and kv.kv_cache.dtype == torch.float4_e2m1fn_x2
    assert kv.block_scale.shape == (2, 3, 5, 16, 2, 4) and kv.block_scale.dtype == torch.float8_e8m0fnu
    assert kv.block_bytes * 5 == kv.kv_cache.numel() + kv.block_scale.numel()
    assert kv.kv_cache.stride()[3:5] == ((2 * 64, 64) if layout == "nhd" else (64, 16 * 64))
    other = KVPool(cfg, num_blocks=2, block_size=16, device="cpu", dtype=torch.bfloat16)
    assert other.block_scale is None and other.block_bytes == 2 * 3 * 16 * 2 * 128 * 2


def test_pool_and_runner_refusals():
    from xvllm.config import Qwen3Shape
    from xvllm.kv_pool import KVPool
    from xvllm.model_runner import ModelRunner

    make = lambda d=128, **kw: KVPool(Qwen3Shape(256, 8, 2, d, 512, 1), num_blocks=2, block_size=16, device="cpu",
                                      dtype=torch.float4_e2m1fn_x2, **kw)
    with pytest.raises(ValueError, match="blocks of 32"):
        make(80)
    with pytest.raises(ValueError, match="k_scale"):
        make(k_scale=0.5)
    with pytest.raises(ValueError, match="cascade"):
        ModelRunner(None, make(), cascade_groups=2)


def test_attention_over_4bit_pages_refusals():
    from xvllm.layers.attention import (Attention, AttnInputs, AttnMetadata, CascadePlan, attention_context,
                                        cascade_decode_attention)

    pool, scale = codes(np.zeros((2, 1, 3, 16, 2, 64), np.uint8)), scales(np.zeros((2, 1, 3, 16, 2, 4), np.uint8))
    z = torch.zeros(1, dtype=torch.int32)
    plan = CascadePlan(z, z.view(1, 1), z, 1, 1)
    q, k = torch.zeros((1, 1024), dtype=torch.bfloat16), torch.zeros((1, 256), dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="cascade"):
        cascade_decode_attention(q, pool[0, 0], pool[1, 0], z.view(1, 1), z, plan, 8, 2, 128)
    attn = Attention(8, 128, 2)
    decode = AttnInputs(z, False, block_tables=z.view(1, 1), cache_seqlens=z)
    with attention_context(AttnMetadata(pool, block_scale=scale)), pytest.raises(TypeError, match="cascade"):
        attn(q, k, k, decode._replace(cascade=plan))
    with attention_context(AttnMetadata(pool)), pytest.raises(ValueError, match="block_scale"):
        attn(q, k, k, decode)


def _prefill_rows(monkeypatch, **kw):
    """The rows that a prefill over 4-bit pages (three sequences of 130, 1 and 20 keys) reads back, nothing launched."""
    from xvllm.layers import attention as A

    class Asked(Exception):
        pass

    def gather(k_cache, v_cache, block_tables, cu_seqlens_k, total_tokens, **scales):
        raise Asked(total_tokens)

    monkeypatch.setattr(A, "require_cuda", lambda *t: None)
    monkeypatch.setattr(A, "gather_kvcache", gather)
    pool, scale = codes(np.zeros((2, 1, 12, 16, 2, 64), np.uint8)), scales(np.zeros((2, 1, 12, 16, 2, 4), np.uint8))
    q, k = torch.zeros((6, 1024), dtype=torch.bfloat16), torch.zeros((6, 256), dtype=torch.bfloat16)
    cu_q, cu_k = torch.tensor([0, 3, 4, 6], dtype=torch.int32), torch.tensor([0, 130, 131, 151], dtype=torch.int32)
    attn = A.AttnInputs(None, True, cu_q, cu_k, 3, block_tables=torch.zeros((3, 9), dtype=torch.int32), **kw)
    with A.attention_context(A.AttnMetadata(pool, block_scale=scale)), pytest.raises(Asked) as asked:
        A.Attention(8, 128, 2)(q, k, k, attn)
    return asked.value.args[0]


def test_prefill_reads_back_the_keys_there_are(monkeypatch):
    assert _prefill_rows(monkeypatch, max_seqlen_k=130, total_seqlen_k=151) == 151
    assert _prefill_rows(monkeypatch, total_seqlen_k=151) == 151
    assert _prefill_rows(monkeypatch, max_seqlen_k=130) == 390  # only the longest is known: room for three of it
    for total in (129, 391, -1):
        with pytest.raises(ValueError, match="total_seqlen_k"):
            _prefill_rows(monkeypatch, max_seqlen_k=130, total_seqlen_k=total)
