"""Moving the pages of a cache of states on the GPU, bit for bit against moves on lists."""
import types

import pytest
import torch

import viby_model_b200 as V
from oracle import linear_oracle as O
from viby_model_b200 import _cabi, canon_cache as CC

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pools(N, seed=0, big=False):
    """States of many types and page sizes: Canon states, write positions, linear attention states, odd ones."""
    g = torch.Generator().manual_seed(seed)
    out = [torch.randn(N, 960, 4, generator=g).bfloat16(), torch.randn(N, 640, 3, generator=g).half(),
           torch.randint(0, 99, (N,), generator=g, dtype=torch.int32), torch.randint(0, 255, (N, 7), generator=g).to(torch.uint8),
           torch.randn(N, 2, 33, 17, generator=g), torch.randn(N, 5, generator=g).double(), torch.randn(N, 3, generator=g).half(),
           torch.zeros(N, 0)]
    if big:
        out.append(torch.randn(N, 4, 64, 64, generator=g))
    return [t.to(DEV) for t in out]


def same(got, want):
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), f"tensor {i}"


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("N", [1, 2, 5, 64, 300])
def test_reorder(N, index):
    for seed in range(3):
        states = pools(N, seed)
        g = torch.Generator().manual_seed(seed)
        source = torch.randint(0, N, (N,), generator=g) if seed else torch.roll(torch.arange(N), 1)
        want = O.move_pages(states, source.to(DEV))
        V.reorder_pages(states, source.to(index).to(DEV))
        same(states, want)


@pytest.mark.parametrize("N", [3, 17, 256])
def test_copy_fork_chains_and_equal_destinations(N):
    for src, dst in (([0, 0], [1, 2]), ([0, 1, 2], [1, 2, 0]), ([1, 2, 0], [0, 0, 0]), ([2, 2], [2, 1]), ([0], [0])):
        states = pools(N)
        source = list(range(N))
        for s, d in reversed(list(zip(src, dst))):  # of equal destinations the first counts
            source[d] = s
        want = O.move_pages(states, source)
        V.copy_pages(states, torch.tensor(src, device=DEV), torch.tensor(dst, device=DEV))
        same(states, want)


@pytest.mark.parametrize("N", [1, 40, 700])
def test_free(N):
    states = pools(N)
    pages = torch.randperm(N, generator=torch.Generator().manual_seed(1))[: (N + 1) // 2]
    want = O.move_pages(states, range(N), pages.tolist())
    V.free_pages(states, torch.cat([pages, pages[:1]]).int().to(DEV))
    same(states, want)


@pytest.mark.parametrize("N", [1, 2, 31, 256, 257, 1000])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.9, 1.0])
def test_compact(N, share):
    states = pools(N, 2)
    live = torch.rand(N, generator=torch.Generator().manual_seed(N)) < share
    source, new, n = O.compact_plan(live.tolist())
    want = O.move_pages(states, source)
    for mask in (live, live.to(torch.uint8) * 3):
        again = [t.clone() for t in states]
        new_index, count = V.compact_pages(again, mask.to(DEV))
        same(again, want)
        assert new_index.dtype == count.dtype == torch.int32
        assert new_index.tolist() == new and count.tolist() == [n]


def test_indexes_outside_move_nothing():
    N = 9
    states = pools(N)
    want = O.move_pages(states, [0, 1, 2, 3, 4, 5, 0, 7, 8])
    V.reorder_pages(states, torch.tensor([0, -1, N, 3, 2 ** 40, 5, 0, -2 ** 50, 8], device=DEV))
    same(states, want)
    want = O.move_pages(want, [3, 1, 2, 3, 4, 5, 6, 7, 8])
    V.copy_pages(states, torch.tensor([-1, 3, N, 1], device=DEV), torch.tensor([0, 0, 1, -1], device=DEV))
    same(states, want)
    want = O.move_pages(want, range(N), [4])
    V.free_pages(states, torch.tensor([-1, 4, N + 3], device=DEV))
    same(states, want)


def test_layers_interleaved_in_one_pool_and_rows_behind():
    N, L = 12, 3
    pool = torch.randn(N + 2, L, 5, 7, device=DEV)
    before = pool.clone()
    source = torch.randint(0, N, (N,), generator=torch.Generator().manual_seed(4))
    V.reorder_pages([pool[:N, i] for i in range(L)], source.to(DEV))
    assert torch.equal(pool[:N], before[source.to(DEV)])
    assert torch.equal(pool[N:], before[N:])
    V.reorder_pages([pool[:N, 1]], torch.roll(torch.arange(N), 2).to(DEV))  # the other layers stay
    assert torch.equal(pool[:N, 0], before[source.to(DEV), 0]) and torch.equal(pool[:N, 2], before[source.to(DEV), 2])


def test_many_tensors_many_pages():
    states = [torch.randn(6, 11, device=DEV) for _ in range(300)]  # more than one launch's table
    want = O.move_pages(states, [5, 4, 3, 2, 1, 0])
    V.reorder_pages(states, torch.tensor([5, 4, 3, 2, 1, 0], device=DEV))
    same(states, want)
    N = _cabi.PAGES_MAX_PAGES
    states = [torch.randn(N, 100, device=DEV), torch.arange(N, device=DEV), torch.randn(N, 3, device=DEV).half()]
    source = torch.randperm(N, generator=torch.Generator().manual_seed(0)).to(DEV)
    want = O.move_pages(states, source.cpu())
    V.reorder_pages(states, source)
    same(states, want)


def test_large_pages():
    states = [torch.randn(9, 4, 160, 160, device=DEV) for _ in range(4)] + [torch.randn(9, 1_000_003, device=DEV)]
    want = O.move_pages(states, [1, 1, 1, 3, 8, 5, 4, 7, 0])
    V.reorder_pages(states, torch.tensor([1, 1, 1, 3, 8, 5, 4, 7, 0], device=DEV))
    same(states, want)


def test_table_is_reusable_and_captured():
    N = 33
    states = pools(N, 5, big=True)
    table = V.PageTable(states)
    source = torch.arange(N, device=DEV)
    live = torch.ones(N, dtype=torch.bool, device=DEV)
    table.reorder(source)
    table.compact(live)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        table.reorder(source)
        new_index, count = table.compact(live)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        source.copy_(torch.randint(0, N, (N,), generator=g))
        live.copy_(torch.rand(N, generator=g) < 0.5)
        plan, new, n = O.compact_plan(live.tolist())
        want = O.move_pages(O.move_pages(states, source.cpu()), plan)
        graph.replay()
        torch.cuda.synchronize()
        same(states, want)
        assert new_index.tolist() == new and count.tolist() == [n]


def test_another_stream():
    states = pools(20)
    want = O.move_pages(states, list(range(19, -1, -1)))
    idx = torch.arange(19, -1, -1, device=DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        V.reorder_pages(states, idx)
    s.synchronize()
    same(states, want)


def test_pages_far_apart():
    far = (1 << 32) + 48  # bytes from page to page
    buf = torch.zeros(3 * far, dtype=torch.uint8, device=DEV)
    t = buf.as_strided((3, 4096), (far, 1))
    t.copy_(torch.randint(0, 255, (3, 4096)).to(torch.uint8))
    want = O.move_pages([t], [2, 0, 1])
    V.reorder_pages([t], torch.tensor([2, 0, 1], device=DEV))
    same([t], want)


def test_large_tables_refuse_before_anything_moves():
    """More tensors than one launch takes: what one launch refuses is refused across launches too, and nothing has moved."""
    states = [torch.full((4, 8), float(n), device=DEV) + torch.arange(4, device=DEV)[:, None] for n in range(_cabi.PAGES_MAX_TENSORS + 3)]
    idx = torch.tensor([1, 0, 3, 2], device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        V.reorder_pages(states + [states[0]], idx)
    own = torch.tensor([1, 0, 3, 2], dtype=torch.int64, device=DEV)
    table = V.PageTable(states + [own.view(4, 1)])
    before = [t.clone() for t in states]
    with pytest.raises(ValueError, match="among the pages"):
        table.reorder(own)
    with pytest.raises(ValueError, match="among the pages"):
        table.copy(own[:2], own[2:])
    torch.cuda.synchronize()
    same(states, before)
    want = O.move_pages(states + [own.view(4, 1)], idx.cpu())
    table.reorder(idx)
    same(states + [own.view(4, 1)], want)
