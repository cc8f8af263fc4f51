"""The attention part of a decoder block on a cache held in 4 bits: prompts and decoding requests together, against 64 bits."""
import pytest
import torch

import plain_ops
import quantised_ops
import workloads as wl
from libortho_b200 import PagedAttentionBlock, PagePool, QuantisedCache, rotary_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def block_of(width, Hq, Hkv, D, **kw):
    qkv = wl.make_layer(width, (Hq + 2 * Hkv) * D, 0.01, seed=1, device=DEV).to_module()
    proj = wl.make_layer(Hq * D, width, 0.01, seed=2, device=DEV).to_module()
    return PagedAttentionBlock(qkv, proj, Hq, Hkv, rotary_table(128, D, device=DEV), **kw)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group,window", [(None, 0), (64, 9)])
def test_steps(dtype, group, window):
    """Every step's tokens through the block, and through the projections with quantisation and attention in 64 bits between them."""
    width, Hq, Hkv, D, P, B = 256, 4, 2, 128, 8, 5
    block = block_of(width, Hq, Hkv, D, window=window)
    g = torch.Generator(device=DEV).manual_seed(3)
    pool, cache = PagePool(B, 60, P, max_pages=10, device=DEV), QuantisedCache(60, P, Hkv, D, group, device=DEV, dtype=dtype)
    mine = QuantisedCache(60, P, Hkv, D, group, device=DEV, dtype=dtype)
    for fresh in ([7, 0, 19, 1, 0], [1, 12, 1, 1, 0], [1, 1, 1, 1, 30], [1, 1, 1, 1, 1]):
        T = sum(fresh)
        step = pool.step(torch.tensor(fresh, dtype=torch.int32, device=DEV), T + 2)
        x = torch.randn(T + 2, width, generator=g, device=DEV).to(dtype)
        got = block(x, cache, pool, step)
        assert got.shape == x.shape and got.dtype == dtype and torch.isfinite(got).all()
        q, k, v = block.qkv(x).view(T + 2, Hq + 2 * Hkv, D)[:T].split((Hq, Hkv, Hkv), dim=1)
        pos = step.positions[:T].view(1, -1)
        q = plain_ops.rotate(q, pos, block.table, [D // 2], False)[0].to(dtype)
        k = plain_ops.rotate(k, pos, block.table, [D // 2], False)[0]
        at = step.slots[:T] // P, step.slots[:T] % P
        for codes, held, y in ((mine.k, mine.k_scales, k), (mine.v, mine.v_scales, v.double())):
            c, s, z = quantised_ops.quantise(y, held.shape[3], dtype)
            codes[at], held[at] = (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8), torch.stack((s, z), -1).to(dtype)
        for a, b in ((cache.k, mine.k), (cache.v, mine.v), (cache.k_scales, mine.k_scales), (cache.v_scales, mine.v_scales)):
            assert torch.equal(a, b)
        o, _, bound, _ = quantised_ops.attention(q, mine.k, mine.v, mine.k_scales, mine.v_scales, pool.block_table, step.positions[:T] + 1, D ** -0.5, window=window, rows=step.requests[:T])
        # both sides round the attention's outputs and the projection's, at most U each
        want = block.proj(o.flatten(1).to(dtype))
        off = (got[:T].double() - want.double()).norm() / want.double().norm()
        assert off <= 4 * plain_ops.U[dtype], float(off)
    back = cache.read(torch.arange(60 * P, device=DEV))
    for x, codes, held in zip(back, (mine.k, mine.v), (mine.k_scales, mine.v_scales)):
        assert torch.equal(x.double(), quantised_ops.nearest(quantised_ops.held(codes, held), dtype).flatten(0, 1))


def test_a_captured_step():
    """Step and block in one graph, replayed for token after token: what the same steps give one by one."""
    width, Hq, Hkv, D, P, B = 256, 4, 2, 64, 8, 3
    block = block_of(width, Hq, Hkv, D)
    g = torch.Generator(device=DEV).manual_seed(5)
    tokens = torch.randn(12, B, width, generator=g, device=DEV).half()
    fresh = torch.ones(B, dtype=torch.int32, device=DEV)
    pools, caches = zip(*((PagePool(B, 20, P, max_pages=4, device=DEV), QuantisedCache(20, P, Hkv, D, device=DEV)) for _ in range(2)))
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
    assert torch.equal(caches[1].k, caches[0].k) and torch.equal(caches[1].v_scales, caches[0].v_scales) and pools[1].lengths.tolist() == [12] * B


def test_two_graphs_that_run_at_once():
    """Two captured steps on streams of their own share no scratch: each gives what it gives alone."""
    Hq, Hkv, D, P = 8, 1, 64, 16
    g = torch.Generator(device=DEV).manual_seed(7)
    made = []
    for n in (20000, 30000):
        pages = n // P + 1
        cache = QuantisedCache(pages, P, Hkv, D, device=DEV)
        k = torch.randn(n, Hkv, D, generator=g, device=DEV).half()
        cache.append(None, k, k.flip(0), torch.arange(n, device=DEV))
        table, n = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, -1), torch.tensor([n], dtype=torch.int32, device=DEV)
        q = torch.randn(1, Hq, D, generator=g, device=DEV).half()
        want = cache.attention(q, table, n)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            got = [cache.attention(q, table, n) for _ in range(20)]
        made.append((graph, stream, got, want, (cache, table, n, q)))
    for _ in range(3):
        for graph, stream, *_ in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for _, _, got, want, _ in made for x in got)
