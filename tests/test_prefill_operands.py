"""What prefill_attention refuses before a kernel reads it: operands on other
devices, too few lengths or table rows, other heads, caches of two layouts."""
import pytest
import torch

BF16, I32, D = torch.bfloat16, torch.int32, 128


def _args(dev="cpu", **kw):
    """Four queries of two sequences; pages of 2 heads, dense keys of as many."""
    cu = torch.tensor([0, 1, 4], dtype=I32, device=dev)
    rows = torch.zeros(4, 2 * D, dtype=BF16, device=dev)
    cache = torch.zeros(6, 16, 2, D, dtype=BF16, device=dev)
    a = dict(q=torch.zeros(4, 4 * D, dtype=BF16, device=dev), k=rows, v=rows, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=3,
             num_qo_heads=4, num_kv_heads=2, head_dim=D, k_cache=None, v_cache=None, block_tables=None)
    if kw.pop("paged", False):
        a.update(k=None, v=None, k_cache=cache, v_cache=cache, block_tables=torch.zeros(2, 3, dtype=I32, device=dev))
    a.update(kw)
    return a


CU = torch.tensor([0, 1, 4], dtype=I32)
CACHE = torch.zeros(6, 16, 2, D, dtype=BF16)
BAD = [
    dict(q=torch.zeros(4, 2, D, dtype=BF16)), dict(q=torch.zeros(4, 4, 64, dtype=BF16)),
    dict(cu_seqlens_k=CU[:2]), dict(cu_seqlens_k=CU[:, None]), dict(cu_seqlens_q=CU[:0]),
    dict(k=None), dict(k=torch.zeros(3, 2 * D, dtype=BF16)), dict(k=torch.zeros(4, 3, D, dtype=BF16), v=torch.zeros(4, 3, D, dtype=BF16)),
    dict(paged=True, v_cache=None), dict(paged=True, block_tables=torch.zeros(1, 3, dtype=I32)),
    dict(paged=True, block_tables=torch.zeros(6, dtype=I32)), dict(paged=True, num_kv_heads=1),
    dict(paged=True, v_cache=torch.zeros(6, 2, 16, D, dtype=BF16).transpose(1, 2)),  # the same shape, head-major
    dict(paged=True, v_cache=CACHE[:5]), dict(paged=True, v_cache=CACHE.to(torch.float8_e4m3fn)),
    dict(paged=True, k_cache=CACHE.view(96, 2, D), v_cache=CACHE.view(96, 2, D)),
    dict(paged=True, k_cache=CACHE.transpose(2, 3), v_cache=CACHE.transpose(2, 3)),
]


@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("bad", BAD, ids=range(len(BAD)))
def test_refusals(monkeypatch, bad, window):
    from xvllm.layers import attention as A

    monkeypatch.setattr(A, "require_cuda", lambda *t: None)
    monkeypatch.setattr(A, "call", lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(A._C, "lib", lambda: pytest.fail("launched"))
    with pytest.raises(ValueError):
        A.prefill_attention(**_args(**bad), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 5])
def test_operands_on_the_host(dev, window):
    """They are refused, not read by the GPU."""
    from xvllm.layers.attention import prefill_attention

    for paged, name in ((False, "k"), (False, "v"), (True, "k_cache"), (True, "v_cache"), (True, "block_tables")):
        a = _args(dev, paged=paged)
        a[name] = a[name].cpu()
        with pytest.raises(RuntimeError, match="one device"):
            prefill_attention(**a, window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 2])
def test_unaligned_keys(dev, window):
    """Contiguous keys that start off a 16-byte boundary are copied."""
    from xvllm.layers.attention import prefill_attention

    a = _args(dev, window=window)
    for name in ("q", "k", "v"):
        a[name] = torch.randn(a[name].shape, device=dev).to(BF16)
    want = prefill_attention(**a)
    for name in ("k", "v"):
        flat = torch.empty(4 * 2 * D + 3, dtype=BF16, device=dev)[3:].view(4, 2 * D)
        assert flat.data_ptr() % 16 and flat.is_contiguous()
        a[name] = flat.copy_(a[name])
    assert torch.equal(prefill_attention(**a), want)


@pytest.mark.parametrize("window", [0, 5])
def test_the_entries_refuse_tokens_too_far_apart(window):
    """Offsets within 16 tokens are 32-bit ones."""
    from xvllm import _C

    lib, a, invalid = _C.lib(), 1 << 20, 1

    def run(paged, stride, batch=0):
        cache = (a, a, 16384, stride, 128, a, 64) if paged else (None, None, 0, 0, 0, None, 0)
        head = (a, 4096, 128, *((None, None, 0, 0) if paged else (a, a, stride, 128)), *cache, a, a, a, 4096, batch, 9)
        if window:
            return lib.xv_window_prefill_attention(*head, 64, 32, 8, D, 16, window, 0, 0.1, None)
        return lib.xv_prefill_attention(*head, 32, 8, D, 16, 0.1, None)

    for paged in (False, True):
        assert run(paged, 1 << 26) == 0 and run(paged, (1 << 26) + 8) == invalid and run(paged, -1024) == invalid
