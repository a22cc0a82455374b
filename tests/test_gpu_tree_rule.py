"""Trees of 17 to 32 rows on both sides of the number of (sequence, kv head)
segments at which the kernels change."""
import pytest
import torch

from rows_cases import D, check
from test_gpu_tree_attention import _inputs, _oracle


@pytest.mark.gpu
@pytest.mark.parametrize("hkv", [1, 8])
@pytest.mark.parametrize("rows", [17, 32])
def test_trees_of_up_to_32_rows(dev, rows, hkv):
    from xvllm.layers.attention import tree_attention

    for batch in (256 // hkv, 256 // hkv + 1):
        nodes = [rows if i % 3 == 0 else (5 * i) % (rows + 1) for i in range(batch)]
        lens = [n + (37 * i) % 200 if n else 0 for i, n in enumerate(nodes)]
        q, k, v, bt, sl, cu, mask, seqs, seen = _inputs(dev, lens, nodes, hkv, hkv, seed=rows)
        run = lambda: tree_attention(q, k, v, bt, sl, cu, mask, rows, hkv, hkv, D)
        got = run()
        check(got, *_oracle(q, seqs, nodes, seen, hkv), f"{batch} sequences of up to {rows} rows")
        assert torch.equal(run(), got)


def test_a_workspace_for_the_largest_batch_does_for_all():
    from xvllm import _C

    size = _C.lib().xv_tree_attention_workspace_size
    for nodes in (1, 4, 5, 8, 9, 64, 300):
        for hkv in (1, 2, 8):
            sizes = [size(b, nodes, 4 * hkv, hkv) for b in (*range(1, 40), 128, 129, 255, 256, 257, 600)]
            assert sizes == sorted(sizes)
