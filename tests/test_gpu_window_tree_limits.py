"""Windowed and tree attention where sizes are large or calls overlap: pages past
2^32 elements, batches of several launches, trees of several passes in graphs and
on two streams."""
import pytest
import torch

from rows_cases import D, check, pack_mask, paged, random_tree, tree_seen
from test_gpu_tree_attention import _inputs, _oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", ["decode", "prefill", "tree", "large_tree"])
def test_far_pages(dev, call):
    """A page's offset takes more than 32 bits, in elements: as with the same pages at the pool's start."""
    from xvllm.layers.attention import paged_decode_attention, prefill_attention, tree_attention

    hq, hkv, lens, block = 32, 8, [700, 300], 256
    k, v, bt, _ = paged(lens, block, hkv, 3, dev=dev)
    far = (1 << 32) // (block * hkv * D)
    if torch.cuda.mem_get_info()[0] < 3 * far * block * hkv * D * 2:
        pytest.skip("needs 26 GB of free memory")
    big = [torch.empty(far + len(x), hkv, block, D, dtype=torch.bfloat16, device=dev).transpose(1, 2) for x in (k, v)]
    for b, x in zip(big, (k, v)):
        b[far:] = x
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    n = {"decode": 1, "prefill": 40, "tree": 5, "large_tree": 40}[call]
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=dev)
    q = torch.randn(2 * n, hq * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    mask = pack_mask(tree_seen(random_tree(n, 2)), 1).repeat(2, 1).to(dev)

    def run(kc, vc, table):
        if call == "decode":
            return paged_decode_attention(q, kc, vc, table, sl, hq, hkv, D, window=260, sink_tokens=3)
        if call == "prefill":
            cu_k = torch.tensor([0, 700, 1000], dtype=torch.int32, device=dev)
            return prefill_attention(q, None, None, cu, cu_k, n, hq, hkv, D, k_cache=kc, v_cache=vc, block_tables=table,
                                     window=260, sink_tokens=3)
        return tree_attention(q, kc, vc, table, sl, cu, mask, n, hq, hkv, D)

    want = run(k, v, bt)
    assert torch.isfinite(want).all() and torch.equal(run(*big, bt + far), want)


def test_large_trees_of_many_sequences(dev):
    """More sequences than a launch takes, of no node up to two passes."""
    from xvllm.layers.attention import tree_attention

    nodes = [300 if i in (17, 270) else (7 * i) % 45 for i in range(290)]
    lens = [n + (13 * i) % 90 if n else 0 for i, n in enumerate(nodes)]
    q, k, v, bt, sl, cu, mask, seqs, seen = _inputs(dev, lens, nodes, 2, 2, seed=5)
    got = tree_attention(q, k, v, bt, sl, cu, mask, 300, 2, 2, D)
    check(got, *_oracle(q, seqs, nodes, seen, 2))


def test_large_trees_in_a_graph(dev):
    """Replays with trees of other sizes, some without rows in a later pass, with eager calls between them."""
    from xvllm.layers.attention import tree_attention

    hq, hkv, room = 32, 8, [100, 70, 130]
    q, k, v, bt, sl, cu, mask, seqs, _ = _inputs(dev, [500, 300, 140], room, hq, hkv)

    def body():
        return tree_attention(q, k, v, bt, sl, cu, mask, 130, hq, hkv, D, out=torch.zeros_like(q))

    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body()
    for step, (lens, nodes) in enumerate((([500, 300, 140], room), ([130, 0, 140], [130, 0, 3]), ([65, 299, 1], [65, 64, 1]))):
        trees = [tree_seen(random_tree(n, step + i)) for i, n in enumerate(nodes)]
        t = sum(nodes)
        mask[:t] = torch.cat([pack_mask(s, mask.shape[1]) for s in trees]).to(dev)
        cu.copy_(torch.tensor([0] + nodes).cumsum(0))
        sl.copy_(torch.tensor(lens))
        q.normal_()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, body())
        check(got[:t], *_oracle(q[:t], [x[:, :n] for x, n in zip(seqs, lens)], nodes, trees, hq))
        assert (got[t:] == 0).all()


def test_large_trees_on_two_streams(dev):
    from xvllm.layers.attention import tree_attention

    nodes, hq, hkv = [90, 40, 64], 32, 8
    q, k, v, bt, sl, cu, mask, seqs, seen = _inputs(dev, [3000, 900, 64], nodes, hq, hkv)
    qs = [q, q.flip(0)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tree_attention(qs[i], k, v, bt, sl, cu, mask, 90, hq, hkv, D))
    torch.cuda.synchronize()
    for i in range(2):
        check(got[i][0], *_oracle(qs[i], seqs, nodes, seen, hq))
        assert all(torch.equal(o, got[i][0]) for o in got[i])
