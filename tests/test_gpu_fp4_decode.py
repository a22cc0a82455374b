"""Paged decode attention over 4-bit (MXFP4) pages against the oracle's 64-bit
attention over the same codes and scales.

Tolerance.  K, V and q are exact in the kernel's bf16 operands, products and
sums are fp32.  A rounding to bf16 is off by at most 2^-8 of the value (8
significant bits).  Two count: each weight p * scale (so at most 2^-8 of sum
p |v| / l, the weighted mean magnitude A of the column) and the output; partials
of a cut segment stay in fp32.  fp32 sums, exp2 and the score's 2^-24 roundings
add less than 2^-12 of A for the score sizes here (|s| < 64: an absolute 2^-16
in the exponent).  Together at most 2 * 2^-8 A + 2^-12 A < 2.1 * 2^-8 A.  A
single rounding is rarely at its bound; the kernel is held to 4 * 2^-9 A."""
import numpy as np
import pytest
import torch

import oracle.ops as O
from fp4_cases import as_codes, as_scales, on_device, random_pages, tables

pytestmark = pytest.mark.gpu

D = 128


def _reference(q, kc, ks, vc, vs, bt, ctx, scale=None):
    """(outputs, weighted mean magnitudes) [B, Hq, D] in 64 bits."""
    hq, hkv = q.shape[1], kc.shape[2]
    out, mag = np.zeros(q.shape), np.zeros(q.shape)
    page = kc.shape[1]
    scale = D ** -0.5 if scale is None else scale
    for b, n in enumerate(ctx):
        if n == 0:
            continue
        ids = bt[b, : -(-n // page)]
        k = O.dequantize_fp4(kc[ids], ks[ids]).reshape(-1, hkv, D)[:n]
        v = O.dequantize_fp4(vc[ids], vs[ids]).reshape(-1, hkv, D)[:n]
        for h in range(hq):
            s = k[:, h // (hq // hkv)] @ q[b, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[b, h] = w @ v[:, h // (hq // hkv)]
            mag[b, h] = w @ np.abs(v[:, h // (hq // hkv)])
    return out, mag


def _close(got, want, mag):
    got = got.float().cpu().numpy().astype(np.float64).reshape(want.shape)
    assert np.isfinite(got).all()
    excess = np.abs(got - want) - (4 * 2.0 ** -9 * mag + 1e-30)
    assert (excess <= 0).all(), f"max excess {excess.max():.4g} at {np.unravel_index(excess.argmax(), excess.shape)}"


def _inputs(rng, ctx, hq, hkv, page, qstd=1.0, **kw):
    bt, nb = tables(rng, ctx, page)
    kc, ks = random_pages(rng, nb, page, hkv, D, **{"low": 123, "high": 126, **kw})
    vc, vs = random_pages(rng, nb, page, hkv, D, 120, 130)
    q = torch.from_numpy(rng.standard_normal((len(ctx), hq, D)).astype(np.float32) * qstd).to(torch.bfloat16)
    return q, kc, ks, vc, vs, bt


def _call(dev, q, kc, ks, vc, vs, bt, ctx, hkv, layout="hnd", **kw):
    from xvllm.layers.attention import paged_decode_attention

    k, v, s1, s2 = (on_device(a, dev, layout) for a in (kc, vc, ks, vs))
    return paged_decode_attention(q.to(dev).flatten(1), as_codes(k), as_codes(v), torch.from_numpy(bt).to(dev),
                                  torch.tensor(ctx, dtype=torch.int32, device=dev), q.shape[1], hkv, D,
                                  k_block_scale=as_scales(s1), v_block_scale=as_scales(s2), **kw)


@pytest.mark.parametrize("hq,hkv,ctx,page,layout", [
    (32, 8, [1], 16, "hnd"), (32, 8, [1, 17, 300, 513, 16, 2048, 0, 77, 64, 65, 63], 16, "hnd"),
    (32, 8, [1, 17, 300, 513, 16, 2048, 0, 77], 16, "nhd"), (16, 8, [128, 511, 256, 300], 48, "wide"),
    (64, 8, [1000, 33, 4096, 15], 16, "hnd"), (8, 8, [5, 260, 100], 256, "nhd"), (2, 1, [9000], 16, "hnd"),
    (8, 1, [20001, 3], 256, "hnd"), (6, 3, [0, 0, 700], 32, "hnd"), (1, 1, [40], 16, "nhd"), (5, 5, [90, 91], 64, "wide"),
])
def test_decode_matches_oracle(dev, hq, hkv, ctx, page, layout):
    rng = np.random.default_rng(hq * 31 + len(ctx))
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv, page)
    out = _call(dev, q, kc, ks, vc, vs, bt, ctx, hkv, layout)
    torch.cuda.synchronize()
    _close(out, *_reference(q.double().numpy(), kc, ks, vc, vs, bt, ctx))
    for b, n in enumerate(ctx):
        if n == 0:
            assert not out[b].any()


@pytest.mark.parametrize("batch,lo,hi,page", [(300, 1, 90, 16), (64, 200, 900, 16), (257, 0, 3, 32)])
def test_decode_many_sequences(dev, batch, lo, hi, page):
    rng = np.random.default_rng(batch)
    ctx = rng.integers(lo, hi, batch).tolist()
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, 8, 2, page)
    out = _call(dev, q, kc, ks, vc, vs, bt, ctx, 2)
    torch.cuda.synchronize()
    _close(out, *_reference(q.double().numpy(), kc, ks, vc, vs, bt, ctx))


def test_decode_long_stream_per_wave(dev):
    """80 to 90 units per wave, past two windows of the block-id table: 80
    sequences over the same blocks (reads only), the reference in 64 bits on
    the device."""
    rng = np.random.default_rng(3)
    batch, hq, hkv, page, most = 80, 16, 8, 16, 9000
    q1, kc, ks, vc, vs, bt = _inputs(rng, [most], hq, hkv, page)
    ctx = rng.integers(8000, most + 1, batch).tolist()
    q = torch.from_numpy(rng.standard_normal((batch, hq, D)).astype(np.float32)).to(torch.bfloat16)
    out = _call(dev, q, kc, ks, vc, vs, np.repeat(bt, batch, axis=0), ctx, hkv)
    k, v = (torch.from_numpy(O.dequantize_fp4(c[bt[0]], s[bt[0]]).reshape(-1, hkv, D)).to(dev) for c, s in ((kc, ks), (vc, vs)))
    want, mag = np.zeros((batch, hq, D)), np.zeros((batch, hq, D))
    seen = torch.arange(k.shape[0], device=dev) < torch.tensor(ctx, device=dev)[:, None]
    for h in range(hq):
        s = q[:, h].to(dev).double() @ k[:, h // 2].t().contiguous() * D ** -0.5
        w = torch.softmax(s.masked_fill(~seen, -torch.inf), dim=-1)
        want[:, h], mag[:, h] = (w @ v[:, h // 2]).cpu().numpy(), (w @ v[:, h // 2].abs()).cpu().numpy()
    _close(out, want, mag)


@pytest.mark.parametrize("hq", [8, 4, 2, 1])
def test_decode_peaked_scores_scale_and_out(dev, hq):
    """Scores that climb along the sequence (every unit moves the maximum), an
    explicit scale, rows of a strided q and a strided out."""
    from xvllm.layers.attention import paged_decode_attention

    rng = np.random.default_rng(hq)
    ctx, hkv, page = [1500, 64, 1], 1, 16
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv, page)
    order = bt[0, : -(-ctx[0] // page)]
    for j, p in enumerate(order):
        ks[p] = np.clip(118 + j // 12, 1, 126)  # later keys are larger
    wide = torch.zeros(3, hq + 2, D, dtype=torch.bfloat16, device=dev)
    wide[:, 1 : hq + 1] = q.to(dev)
    room = torch.full((3, hq * D + 16), 9.0, dtype=torch.bfloat16, device=dev)
    k, v, s1, s2 = (on_device(a, dev, "hnd") for a in (kc, vc, ks, vs))
    out = paged_decode_attention(wide[:, 1 : hq + 1], as_codes(k), as_codes(v), torch.from_numpy(bt).to(dev).long(),
                                 torch.tensor(ctx, device=dev), hq, hkv, D, 0.25, room[:, : hq * D],
                                 k_block_scale=as_scales(s1), v_block_scale=as_scales(s2))
    torch.cuda.synchronize()
    _close(out, *_reference(q.double().numpy(), kc, ks, vc, vs, bt, ctx, 0.25))
    assert (room[:, hq * D :] == 9).all()


def test_decode_reads_no_unused_row(dev):
    """Scale 255 (NaN) in every row past a sequence's end and in every page no
    sequence holds; a NaN block inside a sequence shows in its columns only
    (V) or in the whole head (K)."""
    rng = np.random.default_rng(17)
    ctx, hq, hkv, page = [70, 16, 129, 1], 8, 2, 16
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv, page)
    used = np.zeros(ks.shape[:2], bool)
    for b, n in enumerate(ctx):
        t = np.arange(n)
        used[bt[b, t // page], t % page] = True
    ks[~used], vs[~used] = 255, 255
    want = _reference(q.double().numpy(), kc, ks, vc, vs, bt, ctx)
    out = _call(dev, q, kc, ks, vc, vs, bt, ctx, hkv)
    _close(out, *want)
    vs[bt[2, 3], 5, 1, 2] = 255          # V of token 53, head 1, values 64 .. 95
    ks[bt[0, 0], 0, 0, 1] = 255          # K of token 0, head 0
    got = _call(dev, q, kc, ks, vc, vs, bt, ctx, hkv).float().cpu().view(4, hq, D)
    nan = torch.zeros(4, hq, D, dtype=torch.bool)
    nan[2, 4:, 64:96] = True
    nan[0, :4] = True
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], out.float().cpu().view(4, hq, D)[~nan])


def test_decode_streams_and_graphs_share_nothing(dev):
    """Two graphs over the same cache, captured one after the other and replayed
    on two streams at once, and eager calls between: all equal the eager result."""
    rng = np.random.default_rng(23)
    hq, hkv, page = 32, 8, 16
    ctx = [3000, 10, 1200]
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv, page)
    from xvllm.layers.attention import paged_decode_attention

    k, v, s1, s2 = (on_device(a, dev, "hnd") for a in (kc, vc, ks, vs))
    btd, sl = torch.from_numpy(bt).to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev)
    qs = [q.to(dev).view(3, -1), (q * 2).to(dev).view(3, -1)]

    def f(x):
        return paged_decode_attention(x, as_codes(k), as_codes(v), btd, sl, hq, hkv, D, k_block_scale=as_scales(s1),
                                      v_block_scale=as_scales(s2))

    want = [f(x) for x in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f(x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for o in outs:
            o.fill_(0)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        eager = f(qs[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])


@pytest.mark.parametrize("batch", [1, 3])
def test_decode_through_a_wide_table(dev, batch):
    """A table of 2.2 million columns (35 million tokens): its rows, not those of 256 sequences, have to be within 2 GB."""
    rng = np.random.default_rng(batch)
    ctx = [90, 5, 33][:batch]
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, 8, 2, 16)
    wide = np.full((batch, 2_200_000), -1, np.int32)
    wide[:, : bt.shape[1]] = bt
    out = _call(dev, q, kc, ks, vc, vs, wide, ctx, 2)
    torch.cuda.synchronize()
    _close(out, *_reference(q.double().numpy(), kc, ks, vc, vs, bt, ctx))


def test_decode_of_unaligned_rows(dev):
    """q as whole rows that start 6 bytes into a buffer."""
    rng = np.random.default_rng(12)
    ctx, hq, hkv = [70, 1, 33], 8, 2
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv, 16)
    room = torch.zeros(q.numel() + 3, dtype=torch.bfloat16, device=dev)
    room[3:] = q.to(dev).flatten()
    out = _call(dev, room[3:].view(q.shape), kc, ks, vc, vs, bt, ctx, hkv)
    torch.cuda.synchronize()
    assert room[3:].view(q.shape).is_contiguous()
    _close(out, *_reference(q.double().numpy(), kc, ks, vc, vs, bt, ctx))


def test_decode_refusals(dev):
    rng = np.random.default_rng(1)
    q, kc, ks, vc, vs, bt = _inputs(rng, [20, 20], 4, 2, 16)
    good = dict(hkv=2)
    assert _call(dev, q, kc, ks, vc, vs, bt, [20, 20], **good).shape == (2, 4 * D)
    assert _call(dev, q[:0], kc, ks, vc, vs, bt, [], **good).shape == (0, 4 * D)
    with pytest.raises(ValueError):
        _call(dev, q, kc, ks, vc, vs, bt, [20, 20], hkv=4)
    with pytest.raises(ValueError):
        _call(dev, q, kc, ks, vc, vs, bt[:1], [20, 20], **good)
    with pytest.raises(ValueError):
        _call(dev, q, kc, ks, vc, vs, bt, [20], **good)
    with pytest.raises(TypeError):
        _call(dev, q.float(), kc, ks, vc, vs, bt, [20, 20], **good)
    with pytest.raises(RuntimeError):  # 6 query heads per kv head
        _call(dev, torch.zeros(2, 12, D, dtype=torch.bfloat16), kc, ks, vc, vs, bt, [20, 20], **good)
