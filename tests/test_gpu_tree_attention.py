"""Attention of trees of drafted tokens against 64-bit attention over the keys
each node sees."""
import pytest
import torch

from rows_cases import D, NAN, attend, check, pack_mask, paged, random_tree, tree_seen

pytestmark = pytest.mark.gpu


def _inputs(dev, lens, nodes, hq, hkv, block=16, layout="hnd", seed=0, words=None, seen=None):
    """lens: tokens with the nodes among them."""
    k, v, bt, seqs = paged(lens, block, hkv, seed, layout, dev)
    words = words or max(1, -(-max(nodes) // 64))
    seen = seen or [tree_seen(random_tree(n, seed + i)) for i, n in enumerate(nodes)]
    mask = torch.cat([pack_mask(s, words) for s in seen]).to(dev)
    cu = torch.tensor([0] + nodes, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)
    q = torch.randn(sum(nodes), hq * D, generator=torch.Generator().manual_seed(seed + 1)).to(torch.bfloat16).to(dev)
    return q, k, v, bt, torch.tensor(lens, dtype=torch.int32, device=dev), cu, mask, seqs, seen


def _oracle(q, seqs, nodes, seen, hq, scale=None):
    want, tol, at = [], [], 0
    for x, n, s in zip(seqs, nodes, seen):
        if n == 0:
            continue
        ctx = x.shape[1]
        full = torch.ones(n, ctx, dtype=torch.bool, device=q.device)
        full[:, max(0, ctx - n) :] = s.to(q.device)[:, n - min(n, ctx) :]
        o, t = attend(q[at : at + n].view(n, hq, D), x[0], x[1], full, scale)
        want.append(o)
        tol.append(t)
        at += n
    return torch.cat(want), torch.cat(tol)


def _run(dev, lens, nodes, hq, hkv, scale=None, **kw):
    from xvllm.layers.attention import tree_attention

    q, k, v, bt, sl, cu, mask, seqs, seen = _inputs(dev, lens, nodes, hq, hkv, **kw)
    got = tree_attention(q, k, v, bt, sl, cu, mask, max(nodes), hq, hkv, D, softmax_scale=scale)
    check(got, *_oracle(q, seqs, nodes, seen, hq, scale), f"{lens} {nodes} {hq}/{hkv}")
    return q, k, v, bt, sl, cu, mask, seqs, seen, got


@pytest.mark.parametrize("hq,hkv", [(8, 8), (6, 3), (32, 8), (8, 1)])
@pytest.mark.parametrize("nodes", [[1], [1, 2, 3], [5, 0, 16, 7], [17, 1], [33, 8], [64, 40, 1]])
def test_small_trees(dev, hq, hkv, nodes):
    lens = [n + (0, 1, 40, 15, 333)[(i + sum(nodes)) % 5] if n else 0 for i, n in enumerate(nodes)]
    _run(dev, lens, nodes, hq, hkv, block=48 if hq == 8 else 16, layout="nhd" if hkv == 3 else "hnd", seed=sum(nodes))


@pytest.mark.parametrize("n", [65, 90, 128, 129, 200])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (8, 1)])
def test_large_trees(dev, n, hq, hkv):
    _run(dev, [n, n + 700, 20 + n // 2], [n, n - 1, n // 2], hq, hkv, seed=n)


@pytest.mark.parametrize("lens,nodes,hq", [([1024 + 900], [1024], 64), ([1003, 40, 900, 65], [1000, 3, 300, 65], 32), ([513] * 3, [513, 512, 257], 8)])
def test_trees_of_many_rows(dev, lens, nodes, hq):
    """More rows than a workgroup takes at once: each part of them has fewer ranges."""
    _run(dev, lens, nodes, hq, 8, seed=len(nodes))


@pytest.mark.parametrize("hq,hkv,nodes", [(32, 8, [20, 7]), (64, 8, [64]), (16, 8, [3, 30])])
def test_long_contexts(dev, hq, hkv, nodes):
    _run(dev, [5000 + 777 * i for i in range(len(nodes))], nodes, hq, hkv, block=256, seed=4)


def test_batches(dev):
    """More sequences than a launch takes, rows without a request among them."""
    nodes = [(5 * i) % 7 for i in range(290)]
    lens = [n + (11 * i) % 60 if n else 0 for i, n in enumerate(nodes)]
    _run(dev, lens, nodes, 8, 8, seed=2)


@pytest.mark.parametrize("scale", [0.25, 0.0, -0.1])
def test_scales(dev, scale):
    _run(dev, [60, 31], [9, 4], 16, 8, scale=scale, seed=6)


def test_rows_that_see_nothing(dev):
    """Empty masks with no context are zeros; with context they see it alone."""
    nodes = [6, 5]
    seen = [torch.eye(6, dtype=torch.bool), torch.zeros(5, 5, dtype=torch.bool)]
    seen[0][2] = False
    q, k, v, bt, sl, cu, mask, seqs, seen, got = _run(dev, [6, 45], nodes, 32, 8, seen=seen, seed=1)
    assert (got[2] == 0).all()


def test_masks_over_all_nodes(dev):
    """Masks need not be trees: any set of nodes, later ones too, and bit 63."""
    nodes = [64, 70]
    g = torch.Generator().manual_seed(3)
    seen = [torch.rand(n, n, generator=g) < 0.3 for n in nodes]
    seen[0][:, 63] = True
    _run(dev, [100, 81], nodes, 32, 8, seen=seen, seed=3)


def test_unused_nodes_hold_anything(dev):
    """Nodes that no row sees may not be in the cache: their slots hold NaN."""
    from xvllm.layers.attention import tree_attention

    nodes, hq, hkv = [20, 12], 32, 8
    seen = [tree_seen(random_tree(n, 5)) for n in nodes]
    for s in seen:
        s[7:9] = False
        s[:, 7:9] = False
    q, k, v, bt, sl, cu, mask, seqs, _ = _inputs(dev, [50, 33], nodes, hq, hkv, seen=seen)
    for b, (n, ctx) in enumerate(zip(nodes, (50, 33))):
        t = torch.tensor([ctx - n + 7, ctx - n + 8], device=dev)
        page = bt[b].long()[t // 16]
        k[page, t % 16] = NAN
        v[page, t % 16] = NAN
    got = tree_attention(q, k, v, bt, sl, cu, mask, 20, hq, hkv, D)
    check(got, *_oracle(q, seqs, nodes, seen, hq))


def test_chain_is_causal_attention(dev):
    """A tree of one branch is the last tokens' causal prefill."""
    from xvllm.layers.attention import prefill_attention

    nodes, hq, hkv = [9, 1, 30], 32, 8
    seen = [torch.tril(torch.ones(n, n)).bool() for n in nodes]
    q, k, v, bt, sl, cu, mask, seqs, seen, got = _run(dev, [200, 80, 31], nodes, hq, hkv, seen=seen, seed=8)
    cu_k = torch.tensor([0, 200, 280, 311], dtype=torch.int32, device=dev)
    chunk = prefill_attention(q, None, None, cu, cu_k, 30, hq, hkv, D, k_cache=k, v_cache=v, block_tables=bt)
    want, tol = _oracle(q, seqs, nodes, seen, hq)
    check(chunk, want, 2 * tol)


def test_layouts(dev):
    """Strided q and masks, spare mask words, int64 indexes, out wider than the rows; rows past the last node stay."""
    from xvllm.layers.attention import tree_attention

    nodes, hq, hkv = [10, 4], 16, 8
    q, k, v, bt, sl, cu, mask, seqs, seen = _inputs(dev, [40, 100], nodes, hq, hkv)
    rows = 20  # 14 nodes and 6 rows behind them
    wide = torch.randn(rows, hq * D + 16, device=dev).to(torch.bfloat16)
    wide[:14, 8 : 8 + hq * D] = q
    m = torch.full((rows, 3), -1, dtype=torch.int64, device=dev)
    m[:14, 0], m[:14, 1] = mask[:, 0], 0
    want = _oracle(q, seqs, nodes, seen, hq)
    for given in (m[:, :2], m[:, 0], m[:, :1]):
        buf = torch.full((rows, hq * D + 6), 7.0, dtype=torch.bfloat16, device=dev)
        tree_attention(wide[:, 8 : 8 + hq * D], k, v, bt.long(), sl.long(), cu.long(), given, 10, hq, hkv, D, out=buf[:, 2:-4])
        check(buf[:14, 2:-4], *want)
        assert (buf[14:] == 7).all() and (buf[:, :2] == 7).all() and (buf[:, -4:] == 7).all()


def test_same_result_every_time(dev):
    q, k, v, bt, sl, cu, mask, seqs, seen, got = _run(dev, [900, 40], [31, 12], 32, 8, seed=9)
    from xvllm.layers.attention import tree_attention

    for _ in range(4):
        assert torch.equal(tree_attention(q, k, v, bt, sl, cu, mask, 31, 32, 8, D), got)


def test_graph_replays(dev):
    """Replays with other lengths, trees and queries, with eager calls between them."""
    from xvllm.layers.attention import tree_attention

    hq, hkv = 32, 8
    q, k, v, bt, sl, cu, mask, seqs, seen = _inputs(dev, [90, 64, 33], [16, 16, 16], hq, hkv)

    def body():
        out = torch.zeros_like(q)
        return tree_attention(q, k, v, bt, sl, cu, mask, 16, hq, hkv, D, out=out)

    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body()
    for step, (lens, nodes) in enumerate((([90, 64, 33], [16, 16, 16]), ([50, 0, 30], [3, 0, 16]), ([16, 16, 1], [16, 15, 1]))):
        trees = [tree_seen(random_tree(n, step + i)) for i, n in enumerate(nodes)]
        t = sum(nodes)
        mask[:t] = torch.cat([pack_mask(s, 1) for s in trees]).to(dev)
        cu.copy_(torch.tensor([0] + nodes).cumsum(0))
        sl.copy_(torch.tensor(lens))
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, body())
        check(got[:t], *_oracle(q[:t], [x[:, :n] for x, n in zip(seqs, lens)], nodes, trees, hq))
        assert (got[t:] == 0).all()
