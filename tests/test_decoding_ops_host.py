"""The operators around the projections without a GPU: what the C entries and the Python surface refuse before any launch."""
import ctypes
from pathlib import Path

import pytest
import torch

import plain_ops
from libortho_b200 import LowRankAdapters, OrthoLinear, PagedAttentionBlock, PagePool, _C_ops, _lib, rotary_table

OK, NULL, SHAPE, ALIGN, WORKSPACE = 0, 1, 2, 3, 5


def status(name, desc, **change):
    """Status of a call with one field of a record changed."""
    for k, v in change.items():
        setattr(desc, k, v)
    fn = getattr(_lib.lib(), "ortho_b200_" + name)
    return fn(ctypes.byref(desc), None) if name in ("page_step", "rotary_append") else fn(ctypes.byref(desc), None, 0, None)


def page_step():
    d = _lib.PageStepDesc()
    for k in "cached fresh block_table free_pages available lengths starts slots positions request_of counts".split():
        setattr(d, k, 256)
    d.requests, d.width, d.table_stride, d.free_count, d.tokens, d.page_size = 2, 3, 3, 4, 5, 16
    return d


def rotary():
    d = _lib.RotaryAppendDesc()
    for k in "q k v q_out k_cache v_cache slots positions table".split():
        setattr(d, k, 256)
    d.tokens, d.q_heads, d.kv_heads, d.head_dim, d.rotary, d.table_rows, d.pages, d.page_size = 2, 4, 2, 64, 64, 10, 3, 16
    d.axes, d.section_ends = 1, (ctypes.c_int32 * 4)(32)
    return d


def attention():
    d = _lib.PagedAttentionDesc()
    for k in "q k_cache v_cache out block_table lengths".split():
        setattr(d, k, 256)
    d.batch, d.q_heads, d.kv_heads, d.head_dim, d.rows, d.width, d.table_stride, d.pages, d.page_size = 2, 4, 2, 64, 2, 3, 3, 9, 16
    d.q_token_stride, d.q_head_stride, d.out_token_stride, d.out_head_stride = 256, 64, 256, 64
    d.k_page_stride = d.v_page_stride = 2048
    d.k_slot_stride = d.v_slot_stride = 128
    d.k_head_stride = d.v_head_stride = 64
    return d


def low_rank():
    d = _lib.LowRankDesc()
    for k in "x y out down up ids".split():
        setattr(d, k, 256)
    d.tokens, d.K, d.N, d.adapters, d.rank, d.x_stride, d.y_stride, d.out_stride = 2, 64, 32, 3, 16, 64, 32, 32
    return d


def test_records_match_the_header():
    """Sizes of the records as the C compiler lays them out (8-byte fields first, then 4-byte ones)."""
    sizes = {_lib.PageStepDesc: 17 * 8, _lib.RotaryAppendDesc: 9 * 8 + 23 * 8 + 7 * 4 + 4, _lib.PagedAttentionDesc: 8 * 8 + 20 * 8 + 8,
             _lib.LowRankDesc: 8 * 8 + 8 * 8 + 8}
    for desc, size in sizes.items():
        assert ctypes.sizeof(desc) == size, desc


@pytest.mark.parametrize("change,want", [
    ({"requests": -1}, SHAPE), ({"page_size": 0}, SHAPE), ({"tokens": 1 << 31}, SHAPE), ({"free_count": -1}, SHAPE),
    ({"counts": None}, NULL), ({"cached": None}, NULL), ({"block_table": None}, NULL), ({"free_pages": None}, NULL), ({"slots": None}, NULL)])
def test_page_step_refuses(change, want):
    assert status("page_step", page_step(), **change) == want
    assert _lib.lib().ortho_b200_page_step(None, None) == NULL


@pytest.mark.parametrize("change,want", [
    ({"type": 2}, SHAPE), ({"tokens": -1}, SHAPE), ({"kv_heads": 0}, SHAPE), ({"head_dim": 0}, SHAPE), ({"rotary": 3}, SHAPE), ({"rotary": 66}, SHAPE),
    ({"axes": 0}, SHAPE), ({"axes": 5}, SHAPE), ({"axes": 2}, SHAPE), ({"page_size": 0}, SHAPE), ({"k": None}, NULL), ({"q_out": None}, NULL),
    ({"positions": None}, NULL), ({"table": None}, NULL), ({"slots": None}, NULL), ({"tokens": 0, "k": None}, OK)])
def test_rotary_append_refuses(change, want):
    assert status("rotary_append", rotary(), **change) == want
    assert _lib.lib().ortho_b200_rotary_append(None, None) == NULL


@pytest.mark.parametrize("change,want", [
    ({"type": 2}, SHAPE), ({"batch": -1}, SHAPE), ({"q_heads": 5}, SHAPE), ({"kv_heads": 0}, SHAPE), ({"head_dim": 60}, SHAPE), ({"head_dim": 264}, SHAPE),
    ({"window": -1}, SHAPE), ({"page_size": 0}, SHAPE), ({"width": 1 << 30}, SHAPE), ({"q": None}, NULL), ({"lengths": None}, NULL),
    ({"block_table": None}, NULL), ({"q": 264}, ALIGN), ({"v_cache": 258}, ALIGN), ({"k_slot_stride": 100}, ALIGN), ({"out_head_stride": 65}, ALIGN),
    ({"batch": 0, "q": None}, OK)])
def test_paged_attention_refuses(change, want):
    assert status("paged_attention", attention(), **change) == want
    assert _lib.lib().ortho_b200_paged_attention(None, None, 0, None) == NULL
    assert _lib.lib().ortho_b200_paged_attention_workspace_bytes(None) == -1


@pytest.mark.parametrize("change,want", [
    ({"type": 2}, SHAPE), ({"tokens": -1}, SHAPE), ({"K": 60}, SHAPE), ({"N": 0}, SHAPE), ({"adapters": 0}, SHAPE), ({"rank": 12}, SHAPE),
    ({"rank": 264}, SHAPE), ({"x": None}, NULL), ({"ids": None}, NULL), ({"x": 258}, ALIGN), ({"up": 264}, ALIGN), ({"x_stride": 60}, ALIGN),
    ({"tokens": 200}, WORKSPACE), ({"tokens": 0, "x": None}, OK)])
def test_low_rank_add_refuses(change, want):
    assert status("low_rank_add", low_rank(), **change) == want
    assert _lib.lib().ortho_b200_low_rank_add(None, None, 0, None) == NULL
    assert _lib.lib().ortho_b200_low_rank_add_workspace_bytes(None) == -1


def test_cpu_tensors_raise():
    i = torch.zeros(2, dtype=torch.int32)
    h = torch.zeros(2, 2, 8, dtype=torch.float16)
    cache = torch.zeros(1, 4, 2, 8, dtype=torch.float16)
    for call in (lambda: _C_ops.page_step(i, i, i.view(2, 1), i, i[:1], 4, 2),
                 lambda: _C_ops.rotary_append(h, h, h, cache, cache, i.long(), i, torch.zeros(4, 8)),
                 lambda: _C_ops.paged_attention(h, cache, cache, i.view(2, 1), i),
                 lambda: _C_ops.low_rank_add(h[0], h[0], h.view(1, 8, 4), h.view(1, 4, 8), i)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_adapters_are_placed_and_checked_on_the_host():
    m = LowRankAdapters(2, 16, 12, 5)
    assert m.down.shape == (2, 8, 16) and m.up.shape == (2, 12, 8) and m.ranks.tolist() == [0, 0]
    a, b = torch.randn(3, 16), torch.randn(12, 3)
    m.load(1, a, b, 0.5)
    assert torch.equal(m.down[1, :3], a.half()) and torch.equal(m.up[1, :, :3], b.half()) and not m.down[1, 3:].any() and not m.up[1, :, 3:].any()
    m.load(1, a[:1], b[:, :1])
    assert not m.down[1, 1:].any() and m.ranks.tolist() == [0, 1] and m.scales.tolist() == [0.0, 1.0]
    for bad in ((2, a, b), (-1, a, b)):
        with pytest.raises(IndexError):
            m.load(*bad)
    for bad in ((0, a, b.T), (0, torch.randn(6, 16), torch.randn(12, 6)), (0, a[:0], b[:, :0])):
        with pytest.raises(ValueError):
            m.load(*bad)
    with pytest.raises(ValueError):
        LowRankAdapters(1, 12, 8, 4)
    with pytest.raises(TypeError):
        LowRankAdapters(1, 16, 8, 4, dtype=torch.float32)


def test_rotary_table():
    t = rotary_table(5000, 8)
    assert t.shape == (5000, 8) and t.dtype == torch.float32
    angle = 4999 * 10000.0 ** -0.25
    assert abs(float(t[4999, 1]) - torch.tensor(angle, dtype=torch.float64).cos()) < 1e-7
    assert abs(float(t[4999, 5]) - torch.tensor(angle, dtype=torch.float64).sin()) < 1e-7
    with pytest.raises(ValueError):
        rotary_table(4, 3)


def test_the_plain_forms_by_hand():
    """The oracle itself on cases small enough to write down."""
    got = plain_ops.page_step([3, 0], [2, 1], [[7, -1], [-1, -1]], [4, 5, 6], 3, 4, 4)
    assert got == ([5, 1], [0, 2, 3], [31, 24, 20, -1], [3, 4, 0, -1], [0, 0, 1, -1], [3, 2, 1], [[7, 6], [5, -1]])
    x, _ = plain_ops.rotate(torch.tensor([[[1.0, 2.0, 3.0, 4.0]]]), torch.tensor([[1]]), torch.tensor([[1.0, 1, 0, 0], [0, 1, 1, 0]]), [2], False)
    assert x.flatten().tolist() == [-3.0, 2.0, 1.0, 4.0]
    x, _ = plain_ops.rotate(torch.tensor([[[1.0, 2.0, 3.0, 4.0]]]), torch.tensor([[1]]), torch.tensor([[1.0, 1, 0, 0], [0, 1, 1, 0]]), [2], True)
    assert x.flatten().tolist() == [-2.0, 1.0, 3.0, 4.0]
    k = torch.zeros(2, 2, 1, 8)
    v = torch.arange(32.0).view(2, 2, 1, 8)
    out, lse, _, _ = plain_ops.attention(torch.ones(1, 1, 8), k, v, torch.tensor([[1, 0]]), torch.tensor([3]), 1.0)
    assert torch.allclose(out[0, 0], (v[1, 0, 0] + v[1, 1, 0] + v[0, 0, 0]).double() / 3) and abs(float(lse[0, 0]) - 1.0986122886681098) < 1e-12
    out, _ = plain_ops.low_rank(torch.ones(1, 8), torch.ones(1, 2), torch.ones(1, 8, 8), torch.ones(1, 2, 8), torch.tensor([0]))
    assert out.tolist() == [[65.0, 65.0]]


def test_every_arrival_at_a_cluster_barrier_is_waited_for():
    """A second arrival before the wait for the first one is undefined, and what is sent between them may meet a CTA that has not started."""
    sources = Path(_lib.__file__).parent / "csrc"
    for path in sorted(sources.glob("*.cu*")):
        if path.name == "tma.cuh":                           # (their definitions)
            continue
        text = path.read_text()
        assert text.count("cluster_arrive()") == text.count("cluster_wait()"), path.name


def test_the_plain_page_step_takes_only_pages_that_the_table_holds():
    """The oracle by hand: a table of two columns of four tokens, then one of three."""
    got = plain_ops.page_step([8, 0], [8, 1], [[0, 1], [-1, -1]], [2, 3, 4, 5], 4, 4, 9)
    assert got == ([16, 1], [0, 8, 9], [-1] * 8 + [20], [8, 9, 10, 11, 12, 13, 14, 15, 0], [0] * 8 + [1], [9, 1, 3], [[0, 1], [5, -1]])
    got = plain_ops.page_step([8], [8], [[0, 1, -1]], [2, 3], 2, 4, 8)
    assert got[2] == [12, 13, 14, 15, -1, -1, -1, -1] and got[5] == [8, 1, 1] and got[6] == [[0, 1, 3]]
    assert plain_ops.page_step([2 ** 31 - 1], [5], [[0, 1]], [2, 3], 2, 4, 1)[5] == [5, 0, 2]


def test_the_plain_page_step_names_no_page_where_none_is_left():
    got = plain_ops.page_step([4, 3], [5, 2], [[0, 7, 6], [1, 7, 6]], [5, 4], 1, 4, 7)
    assert got[6] == [[0, 5, -1], [1, -1, 6]] and got[2] == [20, 21, 22, 23, -1, 7, -1] and got[5] == [7, 3, 0]


def test_a_pool_names_requests_that_lack_pages():
    pool = PagePool(5, 9, 4, max_pages=2, device="cpu")
    pool.block_table.copy_(torch.tensor([[3, 1], [-1, 2], [4, -1], [5, -1], [6, 7]]))
    pool.lengths.copy_(torch.tensor([8, 5, 4, 5, 2 ** 31 - 1]))
    assert pool.incomplete().tolist() == [False, True, False, True, True]


def test_rotary_append_needs_caches_only_where_there_are_pages():
    for k_cache, v_cache in ((None, 256), (256, None), (None, None)):
        assert status("rotary_append", rotary(), k_cache=k_cache, v_cache=v_cache) == NULL
        assert status("rotary_append", rotary(), k_cache=k_cache, v_cache=v_cache, pages=0, tokens=0) == OK


def test_a_block_keeps_its_angles_in_32_bits():
    table = rotary_table(5000, 16)
    for convert in (lambda m: m.half(), lambda m: m.bfloat16().float(), lambda m: m.to(torch.float64), lambda m: m.half().float()):
        block = convert(PagedAttentionBlock(OrthoLinear(64, 64), OrthoLinear(32, 64), 2, 1, table))
        assert block.table.dtype == torch.float32 and torch.equal(block.table, table)
