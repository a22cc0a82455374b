"""Refusals of the windowed read back of 8-bit and 4-bit pages (no GPU)."""
import pytest
import torch

A, INVALID = 1 << 20, 1


@pytest.fixture(scope="module")
def lib():
    from xvllm import _C

    return _C.lib()


def _fp8(lib, **kw):
    a = dict(kc=A, vc=A, ps=16384, ts=1024, hs=128, bt=A, bts=64, BS=16, cuq=A, cuk=A, B=4, maxk=512, H=8, D=128, w=16, s=4, ks=1.0,
             vs=1.0, ko=A, vo=A, ost=1024)
    a.update(kw)
    return lib.xv_window_gather_kv_fp8(*a.values(), None)


def _fp4(lib, **kw):
    a = dict(kc=A, vc=A, ps=8192, ts=512, hs=64, ks=A, vs=A, sps=512, sts=32, shs=4, BS=16, bt=A, bts=8, maxb=8, cuq=A, cuk=A,
             B=4, T=100, H=8, D=128, w=16, s=4, ko=A, vo=A, ost=1024)
    a.update(kw)
    return lib.xv_window_gather_kv_fp4(*a.values(), None)


def test_entries_reject_bad_arguments(lib):
    for run, zero in ((_fp8, "maxk"), (_fp4, "T")):
        for kw in (dict(w=0), dict(w=-1), dict(s=-1), dict(cuq=None), dict(B=-1), dict(D=48), dict(ost=512), dict(ko=A + 8)):
            assert run(lib, **kw) == INVALID, kw
        assert run(lib, B=0) == 0 and run(lib, **{zero: 0}) == 0


def test_read_back_refuses(monkeypatch):
    from xvllm import kv_ops

    monkeypatch.setattr(kv_ops, "require_cuda", lambda *t: None)
    monkeypatch.setattr(kv_ops, "fp4_pages", lambda *a: ((0,) * 5, (0,) * 5, (4, 16, 2, 128)))
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.uint8).view(torch.float4_e2m1fn_x2)
    bt, cu = torch.zeros(1, 4, dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32)
    run = lambda **kw: kv_ops.gather_kvcache(pool, pool, bt, cu, 5, k_block_scale=bt, v_block_scale=bt, **kw)
    for kw in (dict(window=-1, cu_seqlens_q=cu), dict(window=1 << 31, cu_seqlens_q=cu), dict(sink_tokens=3), dict(cu_seqlens_q=cu),
               dict(window=4, sink_tokens=-1, cu_seqlens_q=cu), dict(window=4), dict(window=4, cu_seqlens_q=cu[:1])):
        with pytest.raises(ValueError, match="window"):
            run(**kw)


def test_windowed_prefill_hands_its_window_to_the_read_back(monkeypatch):
    from xvllm.layers import attention as At

    asked = {}

    class Asked(Exception):
        pass

    def gather(*a, **kw):
        asked.update(kw)
        raise Asked

    monkeypatch.setattr(At, "require_cuda", lambda *t: None)
    monkeypatch.setattr(At, "gather_kvcache", gather)
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.uint8).view(torch.float4_e2m1fn_x2)
    cu = torch.tensor([0, 5], dtype=torch.int32)
    q = torch.zeros(5, 256, dtype=torch.bfloat16)
    for kw in (dict(window=4, sink_tokens=2), {}):
        asked.clear()
        with pytest.raises(Asked):
            At.prefill_attention(q, None, None, cu, cu, 5, 2, 2, 128, k_cache=pool, v_cache=pool, block_tables=torch.zeros(1, 1),
                                 total_seqlen_k=5, k_block_scale=1, v_block_scale=1, **kw)
        got = {k: asked[k] for k in asked if k in ("cu_seqlens_q", "window", "sink_tokens")}
        if kw:
            assert torch.equal(got.pop("cu_seqlens_q"), cu)
        assert got == kw
