"""Decode attention with a sliding window and sinks against 64-bit attention
over the keys each query sees."""
import pytest
import torch

from rows_cases import D, NAN, attend, check, paged, window_mask

pytestmark = pytest.mark.gpu

HEADS = [(8, 8), (6, 3), (32, 8), (8, 1)]


def _q(rows, hq, seed, dev):
    return torch.randn(rows, hq * D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(dev)


def _oracle(q, seqs, hq, window, sinks, scale=None):
    want = torch.zeros(len(seqs), hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(want)
    for b, x in enumerate(seqs):
        n = x.shape[1]
        if n:
            seen = window_mask([n - 1], n, window, sinks, q.device)
            want[b], tol[b] = (t[0] for t in attend(q[b].view(1, hq, D), x[0], x[1], seen, scale))
    return want, tol


def _run(dev, lens, hq, hkv, window, sinks, block=16, layout="hnd", seed=0, **kw):
    from xvllm.layers.attention import paged_decode_attention

    k, v, bt, seqs = paged(lens, block, hkv, seed, layout, dev)
    q = _q(len(lens), hq, seed + 1, dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = paged_decode_attention(q, k, v, bt, sl, hq, hkv, D, window=window, sink_tokens=sinks, **kw)
    want, tol = _oracle(q, seqs, hq, window, sinks, kw.get("softmax_scale"))
    check(got, want, tol, f"{lens} {hq}/{hkv} window {window} sinks {sinks} block {block}")
    return q, k, v, bt, sl, seqs, got


@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (33, 16), (100, 5), (128, 40), (5000, 4)])
def test_windows(dev, hq, hkv, window, sinks):
    lens = [1, 0, 2, 15, 16, 17, 31, 32, 33, 64, 100, 129, 300, 0, 517]
    _run(dev, lens, hq, hkv, window, sinks, block=48 if hq == 8 else 16, layout="nhd" if hkv == 8 else "hnd", seed=window + sinks)


@pytest.mark.parametrize("window,sinks,block", [(1000, 4, 16), (4096, 64, 256), (333, 700, 16), (2048, 0, 16)])
def test_long(dev, window, sinks, block):
    _run(dev, [9001, 4096, 12345], 32, 8, window, sinks, block=block, seed=7)


def test_one_long_sequence(dev):
    """A window that is cut into as many pieces as a segment may have."""
    _run(dev, [40000], 8, 1, 39000, 16, seed=3)


def test_more_rows_than_a_launch(dev):
    lens = [(37 * i) % 90 for i in range(300)]
    _run(dev, lens, 8, 8, 40, 3, seed=5)


@pytest.mark.parametrize("scale", [0.3, 0.0, -0.1])
def test_scales(dev, scale):
    _run(dev, [5, 70, 333], 16, 8, 50, 4, softmax_scale=scale, seed=9)


@pytest.mark.parametrize("block", [16, 48])
def test_values_no_query_sees(dev, block):
    """NaN and infinities before the window, whole pages of them included, stay out."""
    from xvllm.layers.attention import paged_decode_attention

    lens, hq, hkv, window, sinks = [300, 77, 16, 41], 32, 8, 37, 5
    k, v, bt, seqs = paged(lens, block, hkv, 1, dev=dev)
    q = _q(len(lens), hq, 2, dev)
    for b, n in enumerate(lens):
        hidden = torch.arange(sinks, max(sinks, n - window), device=dev)
        page = bt[b].long()[hidden // block]
        k[page, hidden % block] = NAN
        v[page, hidden % block] = float("inf")
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = paged_decode_attention(q, k, v, bt, sl, hq, hkv, D, window=window, sink_tokens=sinks)
    check(got, *_oracle(q, seqs, hq, window, sinks))


def test_nan_that_is_seen(dev):
    """A NaN value reaches its column only, a NaN key its head group's rows."""
    from xvllm.layers.attention import paged_decode_attention

    hq, hkv = 16, 8
    k, v, bt, _ = paged([50, 50], 16, hkv, 1, dev=dev)
    q = _q(2, hq, 2, dev)
    v[bt[0].long()[40 // 16], 40 % 16, 3, 17] = NAN
    k[bt[1].long()[40 // 16], 40 % 16, 2, 5] = NAN
    sl = torch.tensor([50, 50], dtype=torch.int32, device=dev)
    got = paged_decode_attention(q, k, v, bt, sl, hq, hkv, D, window=30, sink_tokens=2).view(2, hq, D).isnan()
    want = torch.zeros_like(got)
    want[0, 6:8, 17] = True
    want[1, 4:6] = True
    assert torch.equal(got, want)


def test_evicted_pages_are_not_read(dev):
    """Table entries before the window may name any page: here one of NaN."""
    from xvllm.layers.attention import paged_decode_attention

    lens, hq, hkv, window, sinks = [500, 200, 90], 32, 8, 64, 16
    k, v, bt, seqs = paged(lens, 16, hkv, 4, dev=dev)
    nan_page = bt[2, -1].clone()
    for b, n in enumerate(lens):
        bt[b, 1 : (n - window) // 16] = nan_page
    q = _q(3, hq, 2, dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = paged_decode_attention(q, k, v, bt, sl, hq, hkv, D, window=window, sink_tokens=sinks)
    check(got, *_oracle(q, seqs, hq, window, sinks))


def test_window_past_the_sequence_is_plain_decode(dev):
    from xvllm.layers.attention import paged_decode_attention

    lens = [200, 1, 77]
    q, k, v, bt, sl, seqs, got = _run(dev, lens, 32, 8, 1 << 20, 0, seed=11)
    plain = paged_decode_attention(q, k, v, bt, sl, 32, 8, D).view(3, 32, D).double()
    want, tol = _oracle(q, seqs, 32, 1 << 20, 0)
    assert ((plain - want).abs() <= tol + 2.0 ** -8 * want.abs() + 2.0 ** -7).all()


def test_layouts(dev):
    """Strided and unaligned q, a table that is a view, int64 indexes, out in a wider, 4-byte aligned buffer."""
    from xvllm.layers.attention import paged_decode_attention

    lens, hq, hkv, window, sinks = [70, 33, 200], 16, 8, 50, 4
    k, v, bt, seqs = paged(lens, 16, hkv, 6, dev=dev)
    wide = torch.randn(3, hq * D + 24, device=dev).to(torch.bfloat16)
    for q in (wide[:, 8 : 8 + hq * D], wide[:, 3 : 3 + hq * D], wide[:, 8 : 8 + hq * D].unflatten(1, (hq, D))):
        table = torch.stack([bt, bt], dim=2)[:, :, 0].long()
        buf = torch.full((3, hq * D + 6), 7.0, dtype=torch.bfloat16, device=dev)
        out = buf[:, 2 : 2 + hq * D]
        got = paged_decode_attention(q, k, v, table, torch.tensor(lens, device=dev), hq, hkv, D, out=out, window=window,
                                     sink_tokens=sinks)
        assert got.data_ptr() == out.data_ptr()
        check(got, *_oracle(q.reshape(3, -1), seqs, hq, window, sinks))
        assert (buf[:, :2] == 7).all() and (buf[:, -4:] == 7).all()


def test_lengths_past_the_table(dev):
    """Rows beyond the batch in the length and table buffers are not used; a length past the table reads the table's tokens."""
    from xvllm.layers.attention import paged_decode_attention

    k, v, bt, seqs = paged([64, 40, 16], 16, 8, 2, dev=dev)
    q = _q(2, 32, 3, dev)
    sl = torch.tensor([1000, 40, 16], dtype=torch.int32, device=dev)
    got = paged_decode_attention(q, k, v, bt, sl, 32, 8, D, window=20, sink_tokens=1)
    check(got, *_oracle(q, seqs[:2], 32, 20, 1))


def test_graph_replays(dev):
    """Two calls in one graph, replayed with other lengths and queries between eager calls."""
    from xvllm.layers.attention import paged_decode_attention

    hq, hkv, window, sinks = 32, 8, 48, 4
    k, v, bt, seqs = paged([200, 150, 60], 16, hkv, 8, dev=dev)
    q = _q(3, hq, 1, dev)
    sl = torch.tensor([200, 150, 60], dtype=torch.int32, device=dev)

    def body():
        a = paged_decode_attention(q, k, v, bt, sl, hq, hkv, D, window=window, sink_tokens=sinks)
        return a, paged_decode_attention(a, k, v, bt, sl, hq, hkv, D, window=window + 16, sink_tokens=0)

    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = body()
    for step, lens in enumerate(([200, 150, 60], [0, 149, 1], [123, 50, 48], [200, 0, 33])):
        q.copy_(_q(3, hq, 20 + step, dev))
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ea, eb = body()
        assert torch.equal(a, ea) and torch.equal(b, eb)
        check(a, *_oracle(q, [x[:, :n] for x, n in zip(seqs, lens)], hq, window, sinks))


def test_streams(dev):
    """Calls on two streams at once share nothing."""
    from xvllm.layers.attention import paged_decode_attention

    lens, hq, hkv = [3000, 1500, 777, 2048], 32, 8
    k, v, bt, seqs = paged(lens, 16, hkv, 8, dev=dev)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    qs = [_q(4, hq, s, dev) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_decode_attention(qs[i], k, v, bt, sl, hq, hkv, D, window=900 + 100 * i, sink_tokens=4))
    torch.cuda.synchronize()
    for i in range(2):
        want = _oracle(qs[i], seqs, hq, 900 + 100 * i, 4)
        for o in got[i]:
            check(o, *want)
            assert torch.equal(o, got[i][0])
