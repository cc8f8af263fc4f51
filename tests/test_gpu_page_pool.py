"""Pages of a pool over steps that go wrong or are replayed: no page is lost, none is held twice, no request sees another's."""
import pytest
import torch

import plain_ops
from libortho_b200 import PagePool, _C_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def held(pool):
    """Pages in the table, and the free ones."""
    return [p for row in pool.block_table.tolist() for p in row if p >= 0], pool.free_pages.tolist()[:int(pool.available)]


@pytest.mark.parametrize("tokens_a_step", [1, 3, 40])
def test_a_request_past_the_table_loses_no_page(tokens_a_step):
    """Two columns of four tokens: the request's tokens from the ninth on have no place, and what is free stays so."""
    pool = PagePool(2, 12, 4, max_pages=2, device=DEV)
    pool.step(i32([8, 1]), 9)
    n = 8
    while n < 48:
        f = min(tokens_a_step, 48 - n)
        step = pool.step(i32([f, 0]), f)
        n += f
        assert step.slots.tolist() == [-1] * f and step.positions.tolist() == list(range(n - f, n))
        assert step.counts.tolist() == [f, 0, 9] and pool.lengths.tolist() == [n, 1]
    used, free = held(pool)
    assert len(used) == 3 and sorted(used + free) == list(range(12))
    # the other request still gets a page
    step = pool.step(i32([0, 7]), 7)
    assert (step.slots >= 0).all()
    pool.release(torch.tensor([True, True], device=DEV))
    used, free = held(pool)
    assert not used and sorted(free) == list(range(12)) and pool.lengths.tolist() == [0, 0]


def test_a_step_that_ends_behind_the_table_takes_what_the_table_holds():
    """Eight tokens cached, eight more, a table of three columns of four: one page, not two."""
    table = i32([[3, 5, -1], [-1, -1, -1]])
    step = _C_ops.page_step(i32([8, 0]), i32([8, 1]), table, i32([0, 1, 2, 4]), i32([4]), 4, 9)
    assert step.counts.tolist() == [9, 2, 2] and table.tolist() == [[3, 5, 4], [2, -1, -1]]
    assert step.slots.tolist() == [16, 17, 18, 19, -1, -1, -1, -1, 8]


@pytest.mark.parametrize("available", [0, 1])
def test_a_column_without_a_page_names_no_page(available):
    """The table's rows held other requests' pages; those of columns that get none may not be taken for this request's."""
    P, D = 4, 64
    table = i32([[0, 7, 6], [1, 7, 6]])
    free = i32([5, 4])
    step = _C_ops.page_step(i32([4, 3]), i32([5, 2]), table, free, i32([available]), P, 7)
    granted = 5 if available else -1
    assert table.tolist() == [[0, granted, -1], [1, -1, 6]]
    want = plain_ops.page_step([4, 3], [5, 2], [[0, 7, 6], [1, 7, 6]], [5, 4], available, P, 7)
    assert step.slots.tolist() == want[2] and step.counts.tolist() == want[5] and table.tolist() == want[6]
    # the step after: nothing is written to page 7 or 6, and nothing is read from there
    step = _C_ops.page_step(step.lengths, i32([1, 1]), table, free, step.counts[2:], P, 2)
    assert step.slots.tolist() == [-1, -1]
    k, v = (torch.randn(8, P, 1, D, device=DEV).half() for _ in range(2))
    q = torch.randn(2, 1, D, device=DEV).half()
    before = _C_ops.paged_attention(q, k, v, table, step.lengths)
    k[6:], v[6:] = 9.0, 9.0
    assert torch.equal(_C_ops.paged_attention(q, k, v, table, step.lengths), before)


def test_a_captured_step_goes_on_at_every_replay():
    B, pages, P, T = 3, 20, 4, 6
    eager, pool = (PagePool(B, pages, P, max_pages=6, device=DEV) for _ in range(2))
    fresh = i32([0, 0, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = pool.step(fresh, T)
    for f, gone in (([3, 1, 2], None), ([1, 4, 1], [False, True, False]), ([1, 2, 3], None), ([0, 1, 1], [True, False, True]), ([2, 2, 2], None)):
        want = eager.step(i32(f), T)
        fresh.copy_(i32(f))
        graph.replay()
        for name, g, w in zip(want._fields, step, want):
            assert torch.equal(g, w), name
        for p in (eager, pool):
            if gone:
                p.release(torch.tensor(gone, device=DEV))
        for a, b in ((pool.lengths, eager.lengths), (pool.block_table, eager.block_table), (pool.available, eager.available), (pool.free_pages, eager.free_pages)):
            assert torch.equal(a, b)
        used, free = held(pool)
        assert sorted(used + free) == list(range(pages))


def test_an_earlier_step_keeps_what_it_said():
    pool = PagePool(2, 20, 4, device=DEV)
    first = pool.step(i32([5, 1]), 6)
    was = [t.tolist() for t in first]
    pool.step(i32([1, 1]), 2)
    pool.release(torch.tensor([True, False], device=DEV))
    assert [t.tolist() for t in first] == was


def test_requests_that_lack_pages_are_named():
    """Five pages of four tokens: the third request's second page is not there, the first one's table ends."""
    pool = PagePool(4, 5, 4, max_pages=3, device=DEV)
    assert pool.incomplete().tolist() == [False] * 4
    pool.step(i32([9, 4, 3, 0]), 16)                         # 3 + 1 + 1 pages: just enough
    assert pool.incomplete().tolist() == [False] * 4
    step = pool.step(i32([0, 0, 2, 0]), 2)
    assert (step.slots >= 0).tolist() == [True, False] and pool.incomplete().tolist() == [False, False, True, False]
    pool.release(torch.tensor([False, True, False, False], device=DEV))
    step = pool.step(i32([0, 0, 1, 0]), 1)                   # a page is free again, but it is not the one that the fifth token lacks
    assert step.slots.tolist() == [-1] and pool.incomplete().tolist() == [False, False, True, False]
    pool.release(torch.tensor([False, False, True, False], device=DEV))
    pool.step(i32([3, 0, 6, 0]), 9)
    assert pool.incomplete().tolist() == [False] * 4
    pool.step(i32([1, 0, 0, 0]), 1)
    assert pool.incomplete().tolist() == [True, False, False, False]
    pool.release(torch.tensor([True, False, False, False], device=DEV))
    assert pool.incomplete().tolist() == [False] * 4
