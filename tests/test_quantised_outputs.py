"""Where the operators of a cache held in 4 bits write: memory that several of their threads would write at once is refused, strides that do not count are not looked at."""
import ctypes

import pytest
import torch

from libortho_b200 import QuantisedCache, _C_ops, _lib, rotary_table
from test_decoding_ops_host import ALIGN, SHAPE, attention, rotary
from test_quantised_host import cache, change, read

DEV = "cuda:0"
F16 = torch.float16


def apart():
    c = cache()
    c.k, c.v, c.k_scales, c.v_scales = 256, 1 << 20, 2 << 20, 3 << 20
    return c


@pytest.mark.parametrize("changes", [{"k": 1 << 20}, {"k_scales": 3 << 20}, {"k_page_stride": 0}, {"v_slot_stride": 0}, {"k_head_stride": 0}, {"vs_page_stride": 0}, {"ks_slot_stride": 0},
                                     {"vs_head_stride": 0}])
def test_a_written_cache_without_room_is_refused(changes):
    c = apart()
    change(c, changes)
    assert _lib.lib().ortho_b200_rotary_append_quantised(ctypes.byref(rotary()), ctypes.byref(c), None) == SHAPE


@pytest.mark.parametrize("changes", [{"out_token_stride": 0}, {"out_head_stride": 0}])
def test_expanded_outputs_are_refused(changes):
    l = _lib.lib()
    assert l.ortho_b200_rotary_append_quantised(change(rotary(), changes), ctypes.byref(apart()), None) == SHAPE
    assert l.ortho_b200_paged_attention_quantised(change(attention(), changes), ctypes.byref(cache()), None, 0, None) == SHAPE
    assert l.ortho_b200_paged_attention_quantised_workspace_bytes(change(attention(), changes), ctypes.byref(cache())) == -1


@pytest.mark.parametrize("changes,want", [({"k_out": 512, "v_out": 512}, SHAPE), ({"k_token_stride": 0}, SHAPE), ({"v_token_stride": 0}, SHAPE), ({"k_head_stride": 0}, SHAPE), ({"v_head_stride": 0}, SHAPE),
                                          ({"k_token_stride": 4}, ALIGN)])
def test_outputs_read_back_need_room(changes, want):
    d = read()
    d.v_out = 1 << 20
    assert _lib.lib().ortho_b200_read_quantised(change(d, changes), ctypes.byref(apart()), None) == want


def rows(T, H, D, token=None, head=None, at=0, room=1 << 16):
    """A [T, H, D] view with these strides."""
    head = D if head is None else head
    return torch.zeros(room, dtype=F16, device=DEV).as_strided((T, H, D), (H * head if token is None else token, head, 1), at)


@pytest.fixture
def filled():
    c = QuantisedCache(3, 8, 2, 64, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(20, h, 64, generator=g, device=DEV).half() for h in (4, 2, 2))
    slots = torch.randperm(24, generator=g, device=DEV)[:20]
    c.append(None, k, v, slots)
    return c, q, k, v, slots


def tensors(c):
    return c.k, c.v, c.k_scales, c.v_scales


@pytest.mark.gpu
def test_read_refuses_outputs_that_meet(filled):
    c, _, _, _, slots = filled
    one = torch.zeros(1 << 16, dtype=F16, device=DEV)
    view = lambda token, head, at=0: one.as_strided((20, 2, 64), (token, head, 1), at)                  # noqa: E731
    other = torch.zeros(20, 2, 64, dtype=F16, device=DEV)
    for bad in (view(0, 64), view(128, 0), view(64, 64), view(8, 64), view(128, 56), view(120, 64), view(64, 24)):
        for out in ((bad, other), (other, bad)):
            with pytest.raises(ValueError, match="expanded or overlap"):
                _C_ops.read_quantised(*tensors(c), slots, out=out)
    for a, b in ((view(128, 64), view(128, 64)), (view(128, 64), view(128, 64, 64)), (view(128, 64), view(128, 64, 19 * 128)), (view(256, 64), view(256, 64, 56)), (view(256, 128), view(512, 64, 256)),
                 (view(256, 64), view(256, 64, 256 * 10))):
        with pytest.raises(ValueError, match="two tensors"):
            _C_ops.read_quantised(*tensors(c), slots, out=(a, b))
    assert not one.any() and not other.any()


@pytest.mark.gpu
def test_read_writes_into_views(filled):
    c, _, _, _, slots = filled
    want = c.read(slots)
    one = torch.zeros(1 << 16, dtype=F16, device=DEV)
    view = lambda token, head, at=0: one.as_strided((20, 2, 64), (token, head, 1), at)                  # noqa: E731
    for a, b in ((view(256, 64), view(256, 64, 128)), (view(256, 128), view(256, 128, 64)), (view(64, 2048), view(64, 2048, 4096)), (view(128, 64), view(128, 64, 20 * 128)), (view(72, 2048), view(144, 64, 8192))):
        one.zero_()
        got = _C_ops.read_quantised(*tensors(c), slots, out=(a, b))
        assert got[0] is a and got[1] is b and torch.equal(a, want[0]) and torch.equal(b, want[1])
        assert int((one != 0).sum()) == int((want[0] != 0).sum() + (want[1] != 0).sum())
    # a single token: its stride does not count
    a, b = (rows(1, 2, 64, 133) for _ in range(2))
    _C_ops.read_quantised(*tensors(c), slots[:1], out=(a, b))
    assert torch.equal(a, want[0][:1]) and torch.equal(b, want[1][:1])


@pytest.mark.gpu
def test_append_and_attention_outputs(filled):
    c, q, k, v, slots = filled
    table, positions = rotary_table(64, 64, device=DEV), torch.arange(20, dtype=torch.int32, device=DEV)
    append = lambda out, q=q, n=20: _C_ops.rotary_append_quantised(q[:n], k[:n], v[:n], *tensors(c), slots[:n], positions[:n], table, out=out)       # noqa: E731
    want = append(None)
    pages, rows_of, lengths = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV), torch.zeros(20, dtype=torch.int32, device=DEV), positions + 1
    attend = lambda out, q=q, n=20: _C_ops.paged_attention_quantised(q[:n], *tensors(c), pages, lengths[:n], rows=rows_of[:n], out=out)              # noqa: E731
    answer = attend(None)
    for call, right in ((append, want), (attend, answer)):
        for bad in (rows(20, 4, 64, 0), rows(20, 4, 64, 256, 0), rows(20, 4, 64, 64), rows(20, 4, 64, 248), rows(20, 4, 64, 256, 56)):
            with pytest.raises(ValueError, match="expanded or overlap"):
                call(bad)
        fused = torch.zeros(1 << 14, dtype=F16, device=DEV)
        mine = fused.as_strided((20, 4, 64), (256, 64, 1), 0)
        mine.copy_(q)
        for at in (64, 256, 8):
            with pytest.raises(ValueError, match="q's memory"):
                call(fused.as_strided((20, 4, 64), (256, 64, 1), at), mine)
        assert torch.equal(call(mine, mine), right)                            # in place
        single = rows(1, 4, 64, 131)
        assert torch.equal(call(single, n=1), right[:1])
        heads = rows(20, 1, 64, 72, 51)
        if call is append:
            assert torch.equal(append(heads, q[:, :1]), want[:, :1])
    with pytest.raises(ValueError, match="two tensors"):
        _C_ops.rotary_append_quantised(None, k, v, c.k, c.k, c.k_scales, c.v_scales, slots)
    with pytest.raises(ValueError, match="two tensors"):
        _C_ops.rotary_append_quantised(None, k, v, c.k, c.v, c.v_scales, c.v_scales, slots)
