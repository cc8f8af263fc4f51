"""The attention part of a decoder block over several steps: prompts and decoding requests together, against 64 bits."""
import pytest
import torch

import plain_ops
import workloads as wl
from libortho_b200 import LowRankAdapters, PagedAttentionBlock, PagedCache, PagePool, _C_ops, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dense(m):
    """The module's weight in 64 bits."""
    w = _C_ops.dequant_dump(m.base_weight, m.base_scales)[1].double()
    row = torch.repeat_interleave(torch.arange(m.out_features, device=DEV), (m.ortho_row_ptr[1:] - m.ortho_row_ptr[:-1]).long())
    w.index_put_((row, m.ortho_col_indices.long()), m.ortho_values.double() * m.alpha, accumulate=True)
    return w


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_against_dense_attention(dtype):
    width, Hq, Hkv, D, P = 256, 4, 2, 64, 8
    qkv = wl.make_layer(width, (Hq + 2 * Hkv) * D, 0.01, seed=1, device=DEV).to_module()
    proj = wl.make_layer(Hq * D, width, 0.01, seed=2, device=DEV).to_module()
    g = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)                   # noqa: E731
    sets = [LowRankAdapters(3, m.in_features, m.out_features, 16, device=DEV, dtype=dtype) for m in (qkv, proj)]
    for s in sets:
        for i, rank in enumerate((16, 5, 8)):
            s.load(i, r(rank, s.in_features) * s.in_features ** -0.5, r(s.out_features, rank) * 0.1, 0.5 + i)
    table = rotary_table(128, D, device=DEV)
    block = PagedAttentionBlock(qkv, proj, Hq, Hkv, table, qkv_adapters=sets[0], proj_adapters=sets[1])
    B = 5
    pool, cache = PagePool(B, 60, P, max_pages=10, device=DEV), PagedCache(60, P, Hkv, D, device=DEV, dtype=dtype)
    adapter = torch.tensor([0, -1, 2, 1, 0], dtype=torch.int32, device=DEV)
    seen = [[] for _ in range(B)]                             # every request's inputs so far
    for fresh in ([7, 0, 19, 1, 0], [1, 12, 1, 1, 0], [1, 1, 1, 1, 30], [1, 1, 1, 1, 1]):
        step = pool.step(torch.tensor(fresh, dtype=torch.int32, device=DEV), sum(fresh) + 2)
        x = r(sum(fresh) + 2, width).to(dtype)
        ids = torch.where(step.requests >= 0, adapter[step.requests.clamp(min=0).long()], -1)
        got = block(x, cache, pool, step, ids=ids)
        assert got.shape == x.shape and got.dtype == dtype and torch.isfinite(got).all()
        at = 0
        for b, n in enumerate(fresh):
            seen[b] += [x[at + i] for i in range(n)]
            at += n
        want = torch.zeros(sum(fresh), width, dtype=torch.float64, device=DEV)
        at = 0
        for b, n in enumerate(fresh):
            if not n:
                continue
            xs, e = torch.stack(seen[b]), int(adapter[b])

            def through(m, s, v):
                y = v.double() @ dense(m).T
                return y if e < 0 else y + float(s.scales[e]) * (v.double() @ s.down[e].double().T @ s.up[e].double().T)
            heads = through(qkv, sets[0], xs).view(-1, Hq + 2 * Hkv, D)
            pos = torch.arange(len(xs), dtype=torch.int32, device=DEV).view(1, -1)
            q, k = (plain_ops.rotate(heads[:, a:z], pos, table, [D // 2], False)[0] for a, z in ((0, Hq), (Hq, Hq + Hkv)))
            v = heads[:, Hq + Hkv:]
            k, v = (t.repeat_interleave(Hq // Hkv, dim=1) for t in (k, v))
            score = torch.einsum("thd,shd->hts", q, k) * D ** -0.5
            score = score.masked_fill(torch.ones_like(score[0], dtype=torch.bool).triu(1), -torch.inf)
            o = torch.einsum("hts,shd->thd", torch.softmax(score, -1), v).flatten(1)
            want[at:at + n] = through(proj, sets[1], o)[-n:]
            at += n
        # six roundings to 16 bits on the way (activations of the projections to FP16 as well), each relative to values of the outputs' size
        off = (got[:sum(fresh)].double() - want).norm() / want.norm()
        assert off <= 6 * plain_ops.U[dtype], float(off)


def test_a_block_that_is_converted_turns_by_the_same_angles():
    """``half()`` and the like are for weights; angles of late positions do not fit 16 bits."""
    width, Hq, Hkv, D, P = 256, 4, 2, 64, 8
    qkv = wl.make_layer(width, (Hq + 2 * Hkv) * D, 0.01, seed=1, device=DEV).to_module()
    proj = wl.make_layer(Hq * D, width, 0.01, seed=2, device=DEV).to_module()
    table = rotary_table(4096, D, device=DEV)
    x = torch.randn(9, width, device=DEV).half()

    def step(block):
        pool, cache = PagePool(2, 40, P, device=DEV), PagedCache(40, P, Hkv, D, device=DEV)
        s = pool.step(torch.tensor([7, 2], dtype=torch.int32, device=DEV), 9)
        return block(x, cache, pool, s, positions=s.positions + 4000)
    want = step(PagedAttentionBlock(qkv, proj, Hq, Hkv, table))
    got = step(PagedAttentionBlock(qkv, proj, Hq, Hkv, table).half())
    assert torch.equal(got, want)


def test_a_captured_step_through_the_block():
    """Step and block in one graph, replayed for token after token: what the same steps give one by one."""
    width, Hq, Hkv, D, P, B = 256, 4, 2, 64, 8, 3
    qkv = wl.make_layer(width, (Hq + 2 * Hkv) * D, 0.01, seed=1, device=DEV).to_module()
    proj = wl.make_layer(Hq * D, width, 0.01, seed=2, device=DEV).to_module()
    block = PagedAttentionBlock(qkv, proj, Hq, Hkv, rotary_table(128, D, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(5)
    tokens = torch.randn(12, B, width, generator=g, device=DEV).half()
    fresh = torch.ones(B, dtype=torch.int32, device=DEV)
    pools, caches = zip(*((PagePool(B, 20, P, max_pages=4, device=DEV), PagedCache(20, P, Hkv, D, device=DEV)) for _ in range(2)))
    want = [block(x, caches[0], pools[0], pools[0].step(fresh, B)) for x in tokens]
    first = [block(x, caches[1], pools[1], pools[1].step(fresh, B)) for x in tokens[:2]]
    x, graph = tokens[2].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block(x, caches[1], pools[1], pools[1].step(fresh, B))
    for i, one in enumerate(want):
        if i >= 2:
            x.copy_(tokens[i])
            graph.replay()
        assert torch.equal(first[i] if i < 2 else got, one)
    assert torch.equal(caches[1].k, caches[0].k) and torch.equal(caches[1].v, caches[0].v) and pools[1].lengths.tolist() == [12] * B
