"""The operators of a cache held in 4 bits without a GPU: what the C entries and the Python surface refuse before any launch, and the oracle by hand."""
import ctypes

import pytest
import torch

import quantised_ops
from libortho_b200 import QuantisedCache, _C_ops, _lib
from test_decoding_ops_host import ALIGN, NULL, OK, SHAPE, WORKSPACE, attention, rotary

F16, BF16 = torch.float16, torch.bfloat16


def cache():
    c = _lib.QuantisedCacheDesc()
    c.k = c.v = c.k_scales = c.v_scales = 256
    c.pages, c.page_size, c.kv_heads, c.head_dim, c.groups = 9, 16, 2, 64, 1
    for n in "kv":
        setattr(c, n + "_page_stride", 1024), setattr(c, n + "_slot_stride", 32), setattr(c, n + "_head_stride", 512)
        setattr(c, n + "s_page_stride", 32), setattr(c, n + "s_slot_stride", 1), setattr(c, n + "s_head_stride", 16)
    return c


def read():
    d = _lib.ReadQuantisedDesc()
    d.slots = d.k_out = d.v_out = 256
    d.count, d.k_token_stride, d.k_head_stride, d.v_token_stride, d.v_head_stride = 2, 128, 64, 128, 64
    return d


def change(record, changes):
    for k, v in changes.items():
        setattr(record, k, v)
    return ctypes.byref(record)


def statuses(d_append=None, d_read=None, d_attention=None, c=None):
    l, n = _lib.lib(), (lambda x, make: ctypes.byref(x or make()))
    return (l.ortho_b200_rotary_append_quantised(n(d_append, rotary), n(c, cache), None), l.ortho_b200_read_quantised(n(d_read, read), n(c, cache), None),
            l.ortho_b200_paged_attention_quantised(n(d_attention, attention), n(c, cache), None, 0, None))


def test_records_match_the_header():
    assert ctypes.sizeof(_lib.QuantisedCacheDesc) == 4 * 8 + 17 * 8 and ctypes.sizeof(_lib.ReadQuantisedDesc) == 3 * 8 + 5 * 8 + 8


@pytest.mark.parametrize("changes,want", [
    ({"pages": -1}, SHAPE), ({"page_size": 0}, SHAPE), ({"kv_heads": 0}, SHAPE), ({"head_dim": 60}, SHAPE), ({"head_dim": 264}, SHAPE), ({"groups": 0}, SHAPE),
    ({"groups": 2}, SHAPE), ({"k": None}, NULL), ({"v_scales": None}, NULL), ({"v": 258}, ALIGN), ({"k_scales": 258}, ALIGN), ({"k_slot_stride": 30}, ALIGN), ({"v_head_stride": 2}, ALIGN)])
def test_a_cache_is_refused_by_all(changes, want):
    c = cache()
    change(c, changes)
    assert statuses(c=c) == (want, want, want)
    l = _lib.lib()
    assert l.ortho_b200_paged_attention_quantised_workspace_bytes(ctypes.byref(attention()), ctypes.byref(c)) == -1


@pytest.mark.parametrize("changes,want", [
    ({"type": 2}, SHAPE), ({"tokens": -1}, SHAPE), ({"kv_heads": 1}, SHAPE), ({"head_dim": 32}, SHAPE), ({"rotary": 12}, SHAPE), ({"rotary": 72}, SHAPE), ({"axes": 0}, SHAPE),
    ({"axes": 2}, SHAPE), ({"k": None}, NULL), ({"q_out": None}, NULL), ({"positions": None}, NULL), ({"table": None}, NULL), ({"slots": None}, NULL),
    ({"q": 260}, ALIGN), ({"v_head_stride": 66}, ALIGN), ({"out_token_stride": 2}, ALIGN), ({"tokens": 0, "k": None}, OK)])
def test_append_refuses(changes, want):
    assert _lib.lib().ortho_b200_rotary_append_quantised(change(rotary(), changes), ctypes.byref(cache()), None) == want
    assert _lib.lib().ortho_b200_rotary_append_quantised(None, ctypes.byref(cache()), None) == NULL
    assert _lib.lib().ortho_b200_rotary_append_quantised(ctypes.byref(rotary()), None, None) == NULL


@pytest.mark.parametrize("changes,want", [
    ({"type": 2}, SHAPE), ({"count": -1}, SHAPE), ({"count": 1 << 31}, SHAPE), ({"slots": None}, NULL), ({"k_out": None}, NULL), ({"v_out": 264}, ALIGN), ({"k_head_stride": 60}, ALIGN),
    ({"count": 0, "k_out": None}, OK)])
def test_read_refuses(changes, want):
    assert _lib.lib().ortho_b200_read_quantised(change(read(), changes), ctypes.byref(cache()), None) == want
    assert _lib.lib().ortho_b200_read_quantised(None, ctypes.byref(cache()), None) == NULL
    assert _lib.lib().ortho_b200_read_quantised(ctypes.byref(read()), None, None) == NULL


@pytest.mark.parametrize("changes,want", [
    ({"type": 2}, SHAPE), ({"batch": -1}, SHAPE), ({"q_heads": 5}, SHAPE), ({"kv_heads": 1}, SHAPE), ({"head_dim": 128}, SHAPE), ({"window": -1}, SHAPE), ({"width": 1 << 30}, SHAPE),
    ({"q": None}, NULL), ({"lengths": None}, NULL), ({"block_table": None}, NULL), ({"q": 264}, ALIGN), ({"out_head_stride": 65}, ALIGN),
    ({"batch": 10 ** 6, "width": 500}, WORKSPACE), ({"batch": 0, "q": None}, OK)])
def test_attention_refuses(changes, want):
    l = _lib.lib()
    assert l.ortho_b200_paged_attention_quantised(change(attention(), changes), ctypes.byref(cache()), None, 0, None) == want
    assert l.ortho_b200_paged_attention_quantised(None, ctypes.byref(cache()), None, 0, None) == NULL
    assert l.ortho_b200_paged_attention_quantised(ctypes.byref(attention()), None, None, 0, None) == NULL
    assert l.ortho_b200_paged_attention_quantised_workspace_bytes(None, ctypes.byref(cache())) == -1


def test_cpu_tensors_raise():
    i = torch.zeros(2, dtype=torch.int32)
    h = torch.zeros(2, 2, 8, dtype=F16)
    c = [torch.zeros(1, 4, 2, 4, dtype=torch.uint8)] * 2 + [torch.zeros(1, 4, 2, 1, 2, dtype=F16)] * 2
    for call in (lambda: _C_ops.rotary_append_quantised(h, h, h, *c, i.long(), i, torch.zeros(4, 8)), lambda: _C_ops.read_quantised(*c, i.long()),
                 lambda: _C_ops.paged_attention_quantised(h, *c, i.view(2, 1), i)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_a_cache_is_made_and_checked_on_the_host():
    c = QuantisedCache(3, 16, 2, 128, 64, device="cpu", dtype=BF16)
    assert c.k.shape == c.v.shape == (3, 16, 2, 64) and c.k_scales.shape == (3, 16, 2, 2, 2) and c.v_scales.dtype == BF16 and not c.k.any()
    assert c.k.stride() == (2048, 64, 1024, 1) and c.k_scales.stride() == (128, 4, 64, 2, 1)
    assert QuantisedCache(3, 16, 2, 72, device="cpu").k_scales.shape == QuantisedCache(3, 16, 2, 72, 72, device="cpu").k_scales.shape == (3, 16, 2, 1, 2)
    for bad in ((3, 16, 2, 60), (3, 16, 2, 264), (3, 16, 2, 96, 64), (3, 16, 2, 128, 32), (3, 16, 2, 0)):
        with pytest.raises(ValueError):
            QuantisedCache(*bad, device="cpu")
    with pytest.raises(TypeError):
        QuantisedCache(3, 16, 2, 64, device="cpu", dtype=torch.float32)


def test_the_plain_forms_by_hand():
    x = torch.tensor([[0.0, 15.0, 0.5, 1.5, 2.5, 7.25, 14.5, 13.5]], dtype=torch.float64)
    codes, scale, zero = quantised_ops.quantise(x, 1, F16)
    assert codes.tolist() == [[0, 15, 0, 2, 2, 7, 14, 14]] and scale.tolist() == [[1.0]] and zero.tolist() == [[0.0]]
    codes, scale, zero = quantised_ops.quantise(torch.full((1, 8), -3.5, dtype=torch.float64), 1, BF16)
    assert codes.tolist() == [[0] * 8] and scale.tolist() == [[0.0]] and zero.tolist() == [[-3.5]]
    _, scale, _ = quantised_ops.quantise(torch.tensor([[1.0, torch.inf]], dtype=torch.float64), 1, F16)
    assert torch.isnan(scale).all()
    # the whole range of the type: a 15th of it, 8733.87, would round to 8736, and the last code to 65536
    codes, scale, zero = quantised_ops.quantise(torch.tensor([[-65504.0, 65504.0]], dtype=torch.float64), 1, F16)
    assert scale.tolist() == [[8728.0]] and codes.tolist() == [[0, 15]]
    v = torch.tensor([1.0 + 2 ** -11, 1.0 + 3 * 2 ** -11, 65519.0, 65520.0, 2.0 ** -25, 3 * 2.0 ** -26, -2.0 ** -24], dtype=torch.float64)
    assert quantised_ops.nearest(v, F16).tolist() == [1.0, 1.0 + 2 ** -9, 65504.0, float("inf"), 0.0, 2.0 ** -24, -2.0 ** -24]
    assert torch.equal(quantised_ops.nearest(v.float().double(), BF16), v.float().to(BF16).double())
    cache = torch.tensor([[0x21, 0x43, 0xFF, 0x00]], dtype=torch.uint8)
    assert quantised_ops.held(cache, torch.tensor([[[2.0, -1.0]]])).tolist() == [[1.0, 3.0, 5.0, 7.0, 29.0, 29.0, -1.0, -1.0]]
