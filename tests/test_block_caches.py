"""PagedAttentionBlock on caches of a user's own: an object with tensors ``k`` and ``v`` alone, and one with methods."""
import types

import pytest
import torch

import workloads as wl
from libortho_b200 import PagedAttentionBlock, PagedCache, PagePool, PageStep, paged, rotary_table


def fake_block(monkeypatch, calls):
    def rotary_append(q, k, v, k_cache, v_cache, slots, positions, table, **kw):
        calls.append(("append", k_cache, v_cache, kw))
        return q

    def paged_attention(q, k_cache, v_cache, block_table, lengths, **kw):
        calls.append(("attention", k_cache, v_cache, kw))
        return q
    monkeypatch.setattr(paged._C, "rotary_append", rotary_append)
    monkeypatch.setattr(paged._C, "paged_attention", paged_attention)
    qkv, proj = torch.nn.Linear(16, 32), torch.nn.Linear(16, 16)
    return PagedAttentionBlock(qkv, proj, 2, 1, rotary_table(8, 8), window=5)


def test_tensors_alone_and_methods(monkeypatch):
    calls = []
    block = fake_block(monkeypatch, calls)
    one = torch.zeros(3, dtype=torch.int32)
    step, pool = PageStep(*[one] * 6), types.SimpleNamespace(block_table=one.view(1, 3))
    k, v = torch.zeros(1), torch.zeros(2)
    block(torch.zeros(3, 16), types.SimpleNamespace(k=k, v=v), pool, step)
    assert [(c[0], c[1] is k, c[2] is v) for c in calls] == [("append", True, True), ("attention", True, True)]
    assert calls[1][3]["window"] == 5 and calls[1][3]["rows"] is one

    class Own:
        def append(self, q, k, v, *rest, **kw):
            calls.append("own append")
            return q

        def attention(self, q, *rest, **kw):
            calls.append("own attention")
            return q
    block(torch.zeros(3, 16), Own(), pool, step)
    assert calls[2:] == ["own append", "own attention"]


@pytest.mark.gpu
def test_tensors_alone_give_what_a_paged_cache_gives():
    dev, width, Hq, Hkv, D = "cuda:0", 256, 4, 2, 64
    block = PagedAttentionBlock(wl.make_layer(width, (Hq + 2 * Hkv) * D, 0.01, seed=1, device=dev).to_module(), wl.make_layer(Hq * D, width, 0.01, seed=2, device=dev).to_module(),
                                Hq, Hkv, rotary_table(64, D, device=dev))
    pool, a, b = PagePool(2, 8, 8, device=dev), PagedCache(8, 8, Hkv, D, device=dev), PagedCache(8, 8, Hkv, D, device=dev)
    x = torch.randn(9, width, device=dev).half()
    step = pool.step(torch.tensor([5, 4], dtype=torch.int32, device=dev), 9)
    assert torch.equal(block(x, a, pool, step), block(x, types.SimpleNamespace(k=b.k, v=b.v), pool, step)) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and a.k.any()
