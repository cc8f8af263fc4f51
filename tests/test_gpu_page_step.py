"""Pages, slots and positions of a step against whole numbers in Python."""
import random

import pytest
import torch

import plain_ops
from libortho_b200 import PagePool, PageStep, _C_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check(cached, fresh, table, free, available, P, T, out=None):
    W = len(table[0]) if table else 0
    dev_table = i32(table).view(len(cached), W)
    want = plain_ops.page_step(cached, fresh, table, free, available, P, T)
    got = _C_ops.page_step(i32(cached), i32(fresh), dev_table, i32(free), i32([available]), P, T, out=out)
    assert isinstance(got, PageStep) and (out is None or got is out)
    for name, g, w in zip(("lengths", "starts", "slots", "positions", "requests", "counts", "table"), (*got, dev_table), want):
        assert g.flatten().tolist() == (sum(w, []) if name == "table" else w), name
    assert got.slots.dtype == torch.int64 and all(t.dtype == torch.int32 for i, t in enumerate(got) if i != 2)
    return got


def case(rng, B, L, F, P, short=0, narrow=0, none=0.1):
    cached = [rng.choice([0, rng.randint(0, L), rng.randint(0, L // P) * P]) for _ in range(B)]
    fresh = [0 if rng.random() < none else rng.randint(0, F) for _ in range(B)]
    pages = list(range(sum(-(-c // P) for c in cached) + sum(-(-f // P) + 1 for f in fresh) + 3))
    rng.shuffle(pages)
    W = max(1, max(-(-(c + f) // P) for c, f in zip(cached, fresh)) - narrow) if B else 1
    table = [[pages.pop() if j < -(-c // P) else -1 for j in range(W)] for c in cached]
    return cached, fresh, table, pages, max(0, len(pages) - short)


@pytest.mark.parametrize("B,L,F,P", [(1, 0, 1, 16), (1, 100, 1, 1), (3, 40, 7, 5), (64, 300, 1, 16), (256, 90, 40, 24), (511, 64, 3, 8),
                                     (513, 64, 3, 8), (1500, 50, 9, 64), (7, 5, 3000, 128), (600, 0, 0, 16)])
def test_steps(B, L, F, P):
    rng = random.Random(B * 7 + L)
    c = case(rng, B, L, F, P)
    total = sum(c[1])
    for T in {total, total + 3, 0, max(0, total - 2)}:
        check(*c, P, T)


@pytest.mark.parametrize("short,narrow", [(5, 0), (1000, 0), (0, 2), (9, 1)])
def test_a_pool_or_table_without_room(short, narrow):
    rng = random.Random(short + narrow)
    c = case(rng, 40, 60, 30, 8, short=short, narrow=narrow)
    check(*c, 8, sum(c[1]))


def test_what_cannot_be():
    """Negative lengths count as nothing, more available than there are pages as all of them, fewer than none as none; an old page that is
    missing gives no slot."""
    check([-3, 5, 2], [4, -2, 1], [[-1, -1], [3, 4], [0, 1]], [7, 8, 9], 50, 4, 6)
    check([-3, 5, 2], [4, -2, 1], [[-1, -1], [3, 4], [-1, 1]], [7, 8, 9], -1, 4, 6)
    check([2 ** 31 - 1], [2 ** 31 - 1], [[1, 2]], [3], 1, 2 ** 31 - 1, 5)
    check([], [], [], [1, 2], 2, 4, 3)
    check([3], [1], [[5]], [], 0, 4, 1)


def test_strided_tables_reused_outputs_streams_and_capture():
    rng = random.Random(5)
    cached, fresh, table, free, available = case(rng, 30, 50, 4, 8)
    T, W = sum(fresh), len(table[0])
    want = check(cached, fresh, table, free, available, 8, T)
    check(cached, fresh, table, free, available, 8, T, out=PageStep(*(torch.full_like(t, 77) for t in want)))
    wide = torch.full((30, W + 5), 99, dtype=torch.int32, device=DEV)
    part = wide[:, 2:2 + W]
    part.copy_(i32(table))
    args = [i32(cached), i32(fresh).repeat_interleave(2)[::2], part, i32(free), i32([available])]
    got = _C_ops.page_step(*args, 8, T)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (wide[:, :2] == 99).all() and (wide[:, 2 + W:] == 99).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        part.copy_(i32(table))
        got = _C_ops.page_step(*args, 8, T)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _C_ops.page_step(*args, 8, T)
    part.copy_(i32(table))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_steps_in_place():
    """Lengths and counts that are the next step's inputs, more tokens than one CTA has threads and more requests than one chunk."""
    P, B, T, pages = 8, 700, 3000, 9000
    rng = random.Random(11)
    free = list(range(pages))
    rng.shuffle(free)
    table, lengths, available = [[-1] * 12 for _ in range(B)], [0] * B, pages
    dev_table, dev_free = i32(table), i32(free)
    step = _C_ops.page_step(i32(lengths), i32([0] * B), dev_table, dev_free, i32([available]), P, T)
    for _ in range(8):
        fresh = [rng.randint(0, 8) for _ in range(B)]
        want = plain_ops.page_step(lengths, fresh, table, free, available, P, T)
        got = _C_ops.page_step(step.lengths, i32(fresh), dev_table, dev_free, step.counts[2:], P, T, out=step)
        for g, w in zip((*got, dev_table), want):
            assert g.flatten().tolist() == (sum(w, []) if isinstance(w[0], list) else w)
        lengths, table, available = want[0], want[6], want[5][2]
        assert got is step


def test_a_pool_over_steps():
    """Prompts, decoding and requests that leave: no page is held twice, and all come back."""
    rng = random.Random(3)
    B, pages, P = 9, 60, 4
    pool = PagePool(B, pages, P, max_pages=12, device=DEV)
    lengths = [0] * B
    for step in range(30):
        fresh = [rng.choice([0, 1, 1, rng.randint(0, 9)]) if n < 30 else 0 for n in lengths]
        s = pool.step(i32(fresh), sum(fresh) + 2)
        lengths = [n + f for n, f in zip(lengths, fresh)]
        assert pool.lengths.tolist() == lengths and int(s.counts[0]) == sum(fresh)
        table, used = pool.block_table.tolist(), []
        for b, n in enumerate(lengths):
            used += table[b][:-(-n // P)]
            assert all(p == -1 for p in table[b][-(-n // P):])
        left = int(pool.available)
        assert -1 not in used and sorted(used + pool.free_pages.tolist()[:left]) == list(range(pages))
        gone = [n > 20 and rng.random() < 0.5 for n in lengths]
        pool.release(torch.tensor(gone, device=DEV))
        lengths = [0 if g else n for n, g in zip(lengths, gone)]


def test_refusals():
    a = [i32([1, 2]), i32([1, 1]), i32([[0, 1], [2, 3]]), i32([4, 5]), i32([2])]
    _C_ops.page_step(*a, 4, 2)

    def refused(error, match, at=None, value=None, P=4, T=2, out=None):
        b = list(a)
        if at is not None:
            b[at] = value
        with pytest.raises(error, match=match):
            _C_ops.page_step(*b, P, T, out=out)
    refused(TypeError, "cached", 0, a[0].long())
    refused(RuntimeError, "CPU", 0, a[0].cpu())
    refused(RuntimeError, "CPU", 2, a[2].cpu())
    refused(ValueError, "fresh", 1, i32([1]))
    refused(ValueError, "block_table", 2, i32([[0, 1]]))
    refused(ValueError, "block_table", 2, i32([[0, 1], [2, 3]]).T)
    refused(ValueError, "available", 4, i32([1, 2]))
    refused(ValueError, "page_size", P=0)
    refused(ValueError, "tokens", T=-1)
    refused(TypeError, "block_table", 2, None)
    refused(TypeError, "out", out=(1, 2))
    step = _C_ops.page_step(*a, 4, 3)
    refused(ValueError, "slots", out=step)
