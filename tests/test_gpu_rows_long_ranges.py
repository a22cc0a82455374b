"""Windowed decode and small trees over so many pages that a wave's range takes
its table of page ids, 32 units of two pages at a time, several times over."""
import pytest
import torch

from rows_cases import D, attend, check, pack_mask, random_tree, tree_seen, window_mask

pytestmark = pytest.mark.gpu

ROWS, HQ, HKV, PAGES = 64, 32, 8, 700
WAVES = 1024  # ranges of a launch that fills the GPU
# sum |q k| scale stays at 20 (the oracle's tolerance), and a few dozen tokens carry a row: a wrong page shows
SCALE = 0.2


def _pool(dev, block, seed):
    """Sequences of 7800 to 9000 tokens whose tables name the pages of a small pool again and again."""
    g = torch.Generator(device=dev).manual_seed(seed)
    k, v = torch.randn(2, PAGES, HKV, block, D, generator=g, device=dev).to(torch.bfloat16).transpose(2, 3)
    lens = [7800 + (619 * i) % 1201 for i in range(ROWS)]
    bt = torch.randint(0, PAGES, (ROWS, -(-max(lens) // block)), generator=g, device=dev, dtype=torch.int32)
    return g, k, v, bt, lens


def _keys(k, v, bt, n):
    page = bt[: -(-n // k.shape[1])].long()
    return [x[page].reshape(-1, HKV, D)[:n] for x in (k, v)]


@pytest.mark.parametrize("window,sinks,block", [(8192, 0, 16), (7700, 40, 48)])
def test_decode(dev, window, sinks, block):
    from xvllm.layers.attention import paged_decode_attention

    g, k, v, bt, lens = _pool(dev, block, 1)
    assert HKV * sum(min(n, window) // 32 for n in lens) > 96 * WAVES
    q = torch.randn(ROWS, HQ * D, generator=g, device=dev).to(torch.bfloat16)
    got = paged_decode_attention(q, k, v, bt, torch.tensor(lens, dtype=torch.int32, device=dev), HQ, HKV, D, SCALE, window=window,
                                 sink_tokens=sinks)
    for b, n in enumerate(lens):
        want, tol = attend(q[b].view(1, HQ, D), *_keys(k, v, bt[b], n), window_mask([n - 1], n, window, sinks, dev), SCALE)
        check(got[b : b + 1], want, tol, f"sequence {b} of {n}, window {window}, sinks {sinks}, block {block}")


@pytest.mark.parametrize("nodes,block", [(4, 16), (8, 48)])  # 16 and 32 rows
def test_trees(dev, nodes, block):
    from xvllm.layers.attention import tree_attention

    g, k, v, bt, lens = _pool(dev, block, 2)
    assert HKV * sum(n // 32 for n in lens) > 96 * WAVES
    q = torch.randn(ROWS * nodes, HQ * D, generator=g, device=dev).to(torch.bfloat16)
    trees = [tree_seen(random_tree(nodes, i)) for i in range(ROWS)]
    cu = torch.arange(0, ROWS * nodes + 1, nodes, dtype=torch.int32, device=dev)
    mask = torch.cat([pack_mask(t, 1) for t in trees]).to(dev)
    got = tree_attention(q, k, v, bt, torch.tensor(lens, dtype=torch.int32, device=dev), cu, mask, nodes, HQ, HKV, D, SCALE)
    for b, n in enumerate(lens):
        seen = torch.ones(nodes, n, dtype=torch.bool, device=dev)
        seen[:, n - nodes :] = trees[b].to(dev)
        rows = slice(b * nodes, (b + 1) * nodes)
        want, tol = attend(q[rows].view(nodes, HQ, D), *_keys(k, v, bt[b], n), seen, SCALE)
        check(got[rows], want, tol, f"sequence {b} of {n}, {nodes} nodes, block {block}")
