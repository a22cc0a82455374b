"""4-bit (MXFP4) pages written by store_kvcache and read back by
gather_kvcache.  Every step of the format is exact (a power-of-two scale, a
rounding that is defined to the bit), so codes, scales and the bf16 rows read
back equal the 64-bit oracle's: no tolerance."""
import numpy as np
import pytest
import torch

import oracle.ops as O
from fp4_cases import as_codes, as_scales, on_device, random_pages, tables

pytestmark = pytest.mark.gpu


def _new_rows(rng, n, hkv, d):
    """bf16 rows of every size of block: ordinary, tiny and huge ones, zeros,
    exact ties, an infinity, a NaN, subnormals."""
    x = rng.standard_normal((n, hkv, d)).astype(np.float32)
    x *= np.exp2(rng.integers(-6, 7, (n, hkv, d // 32)).astype(np.float32)).repeat(32, axis=-1)
    flat = x.reshape(-1, 32)
    for i, row in enumerate((np.zeros(32), np.resize([6, .25, -.75, 1.25, -1.75, 2.5, -3.5, 5], 32), np.full(32, 7.0),
                             np.full(32, -6.96875), np.full(32, 3e38), np.full(32, 1e-40), np.resize([1e-38, -3e-39], 32),
                             np.resize([1.0, np.inf], 32), np.resize([np.nan, 2.0, 3.0], 32), np.full(32, -0.0))):
        if i < len(flat):
            flat[-1 - i] = row
    return torch.from_numpy(x).to(torch.bfloat16)


def _f64(t):
    return t.float().numpy().astype(np.float64)


@pytest.mark.parametrize("n,hkv,d,page,layout", [
    (1, 8, 128, 16, "hnd"), (37, 8, 128, 16, "nhd"), (300, 5, 128, 48, "wide"), (64, 1, 128, 256, "hnd"),
    (9, 3, 32, 16, "nhd"), (50, 2, 96, 16, "hnd"), (1100, 8, 128, 16, "hnd"),
])
def test_store_is_exact(dev, n, hkv, d, page, layout):
    from xvllm.kv_ops import store_kvcache

    rng = np.random.default_rng(n + d)
    nb = -(-n // page) + 3
    kc, ks = random_pages(rng, nb, page, hkv, d)
    vc, vs = random_pages(rng, nb, page, hkv, d)
    # k and v as views of one fused qkv row
    rows = torch.cat([_new_rows(rng, n, hkv, d), _new_rows(rng, n, hkv, d)], dim=1)
    slots = rng.permutation(nb * page)[:n].astype(np.int32)
    slots[::5] = -1
    dkc, dvc, dks, dvs = (on_device(a, dev, layout) for a in (kc, vc, ks, vs))
    fused = rows.to(dev)
    store_kvcache(fused[:, :hkv], fused[:, hkv:], as_codes(dkc), as_codes(dvc), torch.from_numpy(slots).to(dev),
                  k_block_scale=as_scales(dks), v_block_scale=as_scales(dvs))
    torch.cuda.synchronize()
    for want, wscale, got, gscale, x in ((kc, ks, dkc, dks, rows[:, :hkv]), (vc, vs, dvc, dvs, rows[:, hkv:])):
        q, s = O.quantize_fp4(_f64(x))
        for i, slot in enumerate(slots):
            if slot >= 0:
                want[slot // page, slot % page], wscale[slot // page, slot % page] = q[i], s[i]
        assert np.array_equal(gscale.cpu().numpy(), wscale)
        assert np.array_equal(got.cpu().numpy(), want)


def test_store_flat_cache_odd_layouts_and_other_stream(dev):
    """A flat [num_slots, Hkv, D/2] cache, int64 slots, rows that are not
    16-byte aligned, on a stream that is not the default one; no tokens at all."""
    from xvllm.kv_ops import store_kvcache

    rng = np.random.default_rng(5)
    n, hkv, d, slots_n = 21, 4, 128, 64
    x = _new_rows(rng, n, hkv, d + 32)
    key = x[:, :, 3 : d + 3]   # odd offset
    val = x.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :d]
    q = torch.zeros(slots_n, hkv, d // 2, dtype=torch.uint8, device=dev)
    s = torch.zeros(slots_n, hkv, d // 32, dtype=torch.uint8, device=dev)
    v, vs = q.clone(), s.clone()
    slots = torch.from_numpy(rng.permutation(slots_n)[:n])
    xd = x.to(dev)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        store_kvcache(xd[:, :, 3 : d + 3], xd.transpose(0, 1).contiguous().transpose(0, 1)[:, :, :d], as_codes(q), as_codes(v),
                      slots.to(dev), k_block_scale=as_scales(s), v_block_scale=as_scales(vs))
        store_kvcache(xd[:0, :, :d], xd[:0, :, :d], as_codes(q), as_codes(v), slots[:0].to(dev), k_block_scale=as_scales(s),
                      v_block_scale=as_scales(vs))
    stream.synchronize()
    wk, wks = O.quantize_fp4(_f64(key))
    wv, wvs = O.quantize_fp4(_f64(val))
    at = slots.numpy()
    assert np.array_equal(q.cpu().numpy()[at], wk) and np.array_equal(s.cpu().numpy()[at], wks)
    assert np.array_equal(v.cpu().numpy()[at], wv) and np.array_equal(vs.cpu().numpy()[at], wvs)
    rest = np.setdiff1d(np.arange(slots_n), at)
    assert not q.cpu().numpy()[rest].any() and not s.cpu().numpy()[rest].any()


@pytest.mark.parametrize("ctx,hkv,d,page,layout", [
    ([1], 8, 128, 16, "hnd"), ([0, 17, 0, 0, 300, 1, 16, 0], 8, 128, 16, "nhd"), ([700, 3], 5, 128, 256, "wide"),
    ([33, 95, 96, 97], 2, 96, 48, "hnd"), ([5, 0], 1, 32, 16, "nhd"),
])
def test_gather_is_exact(dev, ctx, hkv, d, page, layout):
    """Every code under every scale byte (0 and 255 among them), empty
    sequences, a table wider than any sequence; rows behind the last sequence
    keep what they held."""
    from xvllm.kv_ops import gather_kvcache

    rng = np.random.default_rng(sum(ctx) + d)
    bt, nb = tables(rng, ctx, page)
    bt = np.concatenate([bt, np.full((len(ctx), 3), -1, np.int32)], axis=1)
    kc, ks = random_pages(rng, nb, page, hkv, d, 0, 255)
    vc, vs = random_pages(rng, nb, page, hkv, d, 100, 150)
    cu = np.concatenate([[0], np.cumsum(ctx)]).astype(np.int32)
    total, behind = int(cu[-1]), 5
    out = tuple(torch.full((total + behind, hkv, d), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    args = [on_device(a, dev, layout) for a in (kc, vc, ks, vs)]
    k, v = gather_kvcache(as_codes(args[0]), as_codes(args[1]), torch.from_numpy(bt).to(dev), torch.from_numpy(cu).to(dev),
                          total + behind, k_block_scale=as_scales(args[2]), v_block_scale=as_scales(args[3]), out=out)
    torch.cuda.synchronize()
    assert k is out[0] and v is out[1]
    for c, s, got in ((kc, ks, k), (vc, vs, v)):
        deq = O.dequantize_fp4(c, s)
        want = np.concatenate([O.gather_paged(deq, bt[b], n) for b, n in enumerate(ctx) if n])
        want = torch.from_numpy(want).to(torch.bfloat16).float().numpy()  # exact but for overflow to infinity
        got = got.float().cpu().numpy()
        assert np.array_equal(got[:total], want, equal_nan=True)
        assert (got[total:] == 7).all()


def test_gather_of_more_than_the_last_level_cache(dev):
    """Outputs of more than 256 MB are written another way: every row of four
    long sequences over the same few blocks, the rows behind them untouched."""
    from xvllm.kv_ops import gather_kvcache

    rng = np.random.default_rng(6)
    ctx, page, nb = [16500, 16401, 17000, 16001], 16, 40
    kc, ks = random_pages(rng, nb, page, 8, 128)
    vc, vs = random_pages(rng, nb, page, 8, 128)
    bt = rng.integers(0, nb, (4, -(-max(ctx) // page))).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(ctx)])
    total = int(cu[-1]) + 5
    assert total * 8 * 128 * 4 > 256 << 20
    out = tuple(torch.full((total, 8, 128), 77.0, dtype=torch.bfloat16, device=dev) for _ in "kv")
    dkc, dvc, dks, dvs = (on_device(a, dev, "hnd") for a in (kc, vc, ks, vs))
    gather_kvcache(as_codes(dkc), as_codes(dvc), torch.from_numpy(bt).to(dev), torch.from_numpy(cu.astype(np.int32)).to(dev), total,
                   k_block_scale=as_scales(dks), v_block_scale=as_scales(dvs), out=out)
    torch.cuda.synchronize()
    rows = torch.from_numpy(np.concatenate([bt[b, np.arange(n) // page] * page + np.arange(n) % page for b, n in enumerate(ctx)]))
    for got, c, s in ((out[0], kc, ks), (out[1], vc, vs)):
        pool = torch.from_numpy(O.dequantize_fp4(c, s).reshape(nb * page, 8, 128)).to(torch.bfloat16).to(dev)
        assert torch.equal(got[:-5], pool[rows.to(dev)])
        assert (got[-5:] == 77).all()


def test_written_rows_read_back_in_a_graph(dev):
    """Store and read back recorded into one graph and replayed over new
    inputs: every replay equals the eager pair."""
    from xvllm.kv_ops import gather_kvcache, store_kvcache

    rng = np.random.default_rng(11)
    ctx, hkv, d, page = [40, 7, 130], 8, 128, 16
    bt, nb = tables(rng, ctx, page)
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(ctx)]).astype(np.int32)).to(dev)
    slots = torch.from_numpy(np.concatenate([bt[b, np.arange(n) // page] * page + np.arange(n) % page
                                             for b, n in enumerate(ctx)])).to(dev)
    btd = torch.from_numpy(bt).to(dev)
    q, s = (torch.zeros(2, nb, page, hkv, w, dtype=torch.uint8, device=dev) for w in (64, 4))
    x = torch.zeros(sum(ctx), 2, hkv, d, dtype=torch.bfloat16, device=dev)

    def both():
        store_kvcache(x[:, 0], x[:, 1], as_codes(q[0]), as_codes(q[1]), slots, k_block_scale=as_scales(s[0]),
                      v_block_scale=as_scales(s[1]))
        return gather_kvcache(as_codes(q[0]), as_codes(q[1]), btd, cu, sum(ctx), k_block_scale=as_scales(s[0]),
                              v_block_scale=as_scales(s[1]))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k, v = both()
    for i in range(4):
        x.normal_(generator=torch.Generator(device=dev).manual_seed(i))
        graph.replay()
        torch.cuda.synchronize()
        got = k.clone(), v.clone()
        want = both()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        ref = O.dequantize_fp4(*O.quantize_fp4(_f64(x[:, 0].cpu())))
        assert np.array_equal(got[0].float().cpu().numpy(), ref.astype(np.float32))


def test_python_refusals(dev):
    from xvllm.kv_ops import gather_kvcache, store_kvcache

    q = as_codes(torch.zeros(4, 16, 2, 64, dtype=torch.uint8, device=dev))
    s = as_scales(torch.zeros(4, 16, 2, 4, dtype=torch.uint8, device=dev))
    kv = torch.zeros(5, 2, 128, dtype=torch.bfloat16, device=dev)
    slots = torch.arange(5, dtype=torch.int32, device=dev)
    sc = dict(k_block_scale=s, v_block_scale=s)
    with pytest.raises(ValueError):
        store_kvcache(kv, kv, q, q, slots)                          # no scales
    with pytest.raises(ValueError):
        store_kvcache(kv, kv, q, q, slots[:4], **sc)                # a slot short
    with pytest.raises(ValueError):
        store_kvcache(kv[:, :1], kv[:, :1], q, q, slots, **sc)      # heads
    with pytest.raises(TypeError):
        store_kvcache(kv.float(), kv.float(), q, q, slots, **sc)
    bt, cu = torch.zeros(1, 4, dtype=torch.int32, device=dev), torch.tensor([0, 5], dtype=torch.int32, device=dev)
    with pytest.raises(TypeError):
        gather_kvcache(kv, kv, bt, cu, 5, **sc)                     # not 4-bit pages
    with pytest.raises(ValueError):
        gather_kvcache(q, q, bt, torch.zeros(3, dtype=torch.int32, device=dev), 5, **sc)  # two sequences, one table row
    with pytest.raises(ValueError):
        gather_kvcache(q, q, bt, cu, -1, **sc)
    with pytest.raises(ValueError):
        gather_kvcache(q, q, bt, cu, 5, out=(kv[:4], kv[:4]), **sc)
