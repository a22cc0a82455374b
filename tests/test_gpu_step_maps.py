"""Block tables, slots and positions built on the GPU against the same built
request by request on the host."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _host(old, new, bt, free, head, block, total, depths=None, owned=None):
    bt = [list(r) for r in bt]
    width = len(bt[0]) if bt else 0
    pos, slots, cu_q, cu_k, own = [], [], [0], [0], []
    for b, (o, n) in enumerate(zip(old, new)):
        have = max(-(-o // block), owned[b] if owned else 0)
        own.append(max(have, -(-(o + n) // block)))
        for blk in range(have, -(-(o + n) // block)):
            if blk < width:
                bt[b][blk] = free[head] if head < len(free) else -1
            head += 1
        for p in range(o, o + n):
            page = bt[b][p // block] if p // block < width else -1
            slots.append(page * block + p % block if page >= 0 else -1)
            pos.append(o + depths[len(pos)] if depths is not None and len(pos) < total else p)
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + o + n)
    pos, slots = (pos + [0] * total)[:total], (slots + [-1] * total)[:total]
    return cu_q, cu_k, [o + n for o, n in zip(old, new)], pos, slots, [head], own, bt


def _run(dev, old, new, block, total=None, head=None, short=0, width=None, depths=None, seed=0,
         owned=None):
    from xvllm.kv_ops import step_maps

    r = np.random.RandomState(seed)
    need = [-(-(o + n) // block) for o, n in zip(old, new)]
    width = max(1, width or max(need, default=1) + 1)
    have = [max(-(-o // block), owned[b] if owned else 0) for b, o in enumerate(old)]
    width = max([width] + have)
    pages = r.permutation(sum(need) + sum(have) + 5 + (head or 0)).tolist()
    bt = [[-7] * width for _ in old]
    for b, k in enumerate(have):
        bt[b][: min(k, width)] = [pages.pop() for _ in range(k)][:width]
    free = pages[: len(pages) - short] if short else pages
    total = sum(new) if total is None else total
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    tables = i32(bt).view(len(old), width)
    m = step_maps(i32(old), i32(new), tables, i32(free), block, total, free_head=None if head is None else i32([head]),
                  depths=None if depths is None else i32(depths), row_blocks=None if owned is None else i32(owned))
    want = _host(old, new, bt, free, head or 0, block, total, depths, owned)
    for name, got, w in zip(("cu_q", "cu_k", "ends", "positions", "slots", "free_head", "row_blocks", "tables"), (*m, tables), want):
        assert got.cpu().reshape(-1).tolist() == np.asarray(w, dtype=np.int64).reshape(-1).tolist(), name
    assert m.positions.dtype == torch.int64 and m.slot_mapping.dtype == torch.int32


@pytest.mark.parametrize("block", [1, 16, 48, 256])
@pytest.mark.parametrize("old,new", [([0], [1]), ([15], [1]), ([16], [1]), ([5, 0, 31, 32], [1, 40, 1, 0]), ([0, 0, 0], [0, 0, 0]),
                                     ([1000, 3, 0, 77], [3, 500, 1, 99])])
def test_maps(dev, block, old, new):
    _run(dev, old, new, block)


@pytest.mark.parametrize("rows", [63, 64, 65, 256, 257, 1000, 4096])
def test_rows(dev, rows):
    r = np.random.RandomState(rows)
    _run(dev, r.randint(0, 200, rows).tolist(), (r.randint(0, 9, rows) * r.randint(0, 2, rows)).tolist(), 16, seed=rows)


def test_long(dev):
    _run(dev, [100000, 0, 5], [3, 70001, 20000], 16)


@pytest.mark.parametrize("total", [0, 3, 40, 61, 100])
def test_row_counts(dev, total):
    """More rows than tokens: the rest have no slot; fewer: the rest are left out."""
    _run(dev, [3, 50, 0], [30, 1, 30], 16, total=total)


def test_free_head(dev):
    _run(dev, [3, 50, 0], [30, 1, 30], 16, head=4)


@pytest.mark.parametrize("short", [1, 5, 8])
def test_free_list_runs_out(dev, short):
    _run(dev, [3, 50, 0], [30, 1, 90], 16, short=short)


def test_table_is_full(dev):
    from xvllm.kv_ops import step_maps

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    bt = i32([[5, -1, -1], [6, 7, 8], [9, -1, -1]])
    m = step_maps(i32([3, 40, 16]), i32([100, 1, 4]), bt, i32(list(range(20, 40))), 16, 105)
    assert bt.tolist() == [[5, 20, 21], [6, 7, 8], [9, 26, -1]] and m.free_head.tolist() == [7]
    slots = m.slot_mapping.tolist()
    assert slots[:45] == [5 * 16 + i for i in range(3, 16)] + [20 * 16 + i for i in range(16)] + [21 * 16 + i for i in range(16)]
    assert slots[45:100] == [-1] * 55 and slots[100:] == [8 * 16 + 8] + [26 * 16 + i for i in range(4)]


def test_rows_keep_blocks_past_their_tokens(dev):
    """Blocks of rejected tokens are used before the list is."""
    _run(dev, [3, 50, 0, 16, 40], [30, 1, 30, 1, 0], 16, owned=[2, 3, 5, 0, 9])
    _run(dev, [100, 7, 0], [3, 90, 20], 48, owned=[4, 1, 0], head=2)


def test_depths(dev):
    _run(dev, [7, 0, 30], [5, 0, 6], 16, depths=[0, 0, 1, 1, 2, 0, 1, 1, 2, 2, 3])
    _run(dev, [7, 0, 30], [2, 0, 2], 16, total=6, depths=[0, 1, 0, 0, 9, 9])


def test_negative_lengths_count_as_none(dev):
    from xvllm.kv_ops import step_maps

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    m = step_maps(i32([-3, 4]), i32([2, -5]), torch.full((2, 3), -1, dtype=torch.int32, device=dev), i32([9, 8]), 16, 2)
    assert m.cache_seqlens.tolist() == [2, 4] and m.cu_seqlens_q.tolist() == [0, 2, 2] and m.slot_mapping.tolist() == [144, 145]


def test_no_rows(dev):
    from xvllm.kv_ops import step_maps

    e = torch.zeros(0, dtype=torch.int32, device=dev)
    m = step_maps(e, e, torch.zeros((0, 4), dtype=torch.int32, device=dev), e, 16, 3)
    assert m.cu_seqlens_q.tolist() == [0] and m.slot_mapping.tolist() == [-1] * 3 and m.free_head.tolist() == [0]


def test_table_rows_of_a_wider_buffer(dev):
    from xvllm.kv_ops import step_maps

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    buf = torch.full((5, 9), -3, dtype=torch.int32, device=dev)
    step_maps(i32([0, 0]), i32([40, 10]), buf[1:4, 2:6], i32([5, 6, 7, 8]), 16, 50)
    want = torch.full((5, 9), -3, dtype=torch.int32)
    want[1, 2:5], want[2, 2] = torch.tensor([5, 6, 7], dtype=torch.int32), 8
    assert torch.equal(buf.cpu(), want)


def test_steps_in_a_graph(dev):
    """A decode step's maps, replayed: the lengths and the free list's head move on the device."""
    from xvllm.kv_ops import step_maps

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    start = [15, 3, 31, 0]
    lens, new, head = i32(start), i32([1, 1, 0, 1]), i32([0])
    bt, free = torch.full((4, 6), -1, dtype=torch.int32, device=dev), i32(list(range(50, 90)))
    bt[0, 0], bt[1, 0], bt[2, :2] = 1, 2, i32([3, 4])

    def body():
        m = step_maps(lens, new, bt, free, 16, 4, free_head=head)
        lens.copy_(m.cache_seqlens)
        head.copy_(m.free_head)
        return m

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        body()
    torch.cuda.synchronize()
    lens.copy_(i32(start))
    head.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m = body()
    host_bt = [[1] + [-1] * 5, [2] + [-1] * 5, [3, 4] + [-1] * 4, [-1] * 6]
    bt.copy_(i32(host_bt))
    old, at = list(start), 0
    for _ in range(40):
        graph.replay()
        torch.cuda.synchronize()
        cu_q, cu_k, ends, pos, slots, h, own, host_bt = _host(old, [1, 1, 0, 1], host_bt, list(range(50, 90)), at, 16, 4)
        assert m.slot_mapping.tolist() == slots and m.positions.tolist() == pos and bt.tolist() == host_bt
        assert lens.tolist() == ends and head.tolist() == h
        old, at = ends, h[0]
