"""Low-rank adapters of many requests against 64 bits."""
import math

import pytest
import torch

import plain_ops
from libortho_b200 import LowRankAdapters, _C_ops, _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def make(T, K, N, E, R, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=DEV) * std).to(dtype)          # noqa: E731
    ids = torch.randint(-1, E, (T,), generator=g, device=DEV, dtype=torch.int32)
    return r(T, K), r(T, N), r(E, R, K, std=K ** -0.5), r(E, N, R, std=R ** -0.5), ids, torch.rand(E, generator=g, device=DEV) + 0.5


def check(x, y, down, up, ids, scales=None, ranks=None):
    want, bound = plain_ops.low_rank(x, y, down, up, ids, scales, ranks)
    before = y.clone()
    got = _C_ops.low_rank_add(x, y, down, up, ids, scales=scales, ranks=ranks)
    assert got.shape == y.shape and got.dtype == y.dtype and torch.equal(y, before)
    plain_ops.within(got, want, plain_ops.rounded(want, bound, y.dtype))
    none = (ids < 0) | (ids >= down.shape[0])
    assert torch.equal(got[none], y[none])
    again = y.clone()
    assert _C_ops.low_rank_add(x, again, down, up, ids, scales=scales, ranks=ranks, out=again) is again
    assert torch.equal(again, got)                           # in place, and the same bits again
    assert _lib.lib().ortho_b200_query_kernel_status() == 0
    return got


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T", [1, 2, 8, 9, 31, 64, 100, 129, 300])
@pytest.mark.parametrize("K,N,E,R", [(512, 384, 3, 16), (8, 1, 1, 8), (2912, 1003, 12, 8), (264, 130, 5, 64)])
def test_tokens(T, K, N, E, R, dtype):
    check(*make(T, K, N, E, R, dtype, seed=T))


@pytest.mark.parametrize("R", [8, 16, 24, 32, 40, 64, 72, 96, 128, 200, 256])
def test_ranks(R):
    for T, dtype in ((5, F16), (140, BF16)):
        x, y, down, up, ids, scales = make(T, 320, 203, 4, R, dtype, seed=R)
        check(x, y, down, up, ids, scales)
        ranks = torch.tensor([R, 0, 3, R - 7], dtype=torch.int32, device=DEV)
        check(x, y, down, up, ids, scales, ranks)
        # what lies behind a rank is not read
        down[1], up[1] = math.nan, math.nan
        down[2, 8:], up[2, :, 8:] = math.nan, math.inf
        check(x, y, down, up, ids, scales, ranks)
        check(x, y, down, up, ids, scales, torch.tensor([R + 100, -5, 8, 1], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("K", [8, 16, 24, 32, 40, 248, 256, 264, 1000, 4096, 14336])
@pytest.mark.parametrize("N", [1, 2, 7, 8, 31, 32, 33, 64, 129, 1000])
def test_widths(K, N):
    check(*make(6, K, N, 2, 16, F16, seed=K + N))


def test_widths_of_prompts():
    for K, N in ((40, 33), (1000, 129), (4096, 1030)):
        check(*make(200, K, N, 3, 24, BF16, seed=K))


@pytest.mark.parametrize("T,E,K,N,R", [(40, 40, 264, 2100, 24), (128, 3, 64, 12000, 8), (90, 60, 520, 3001, 72), (100, 100, 96, 1500, 256), (3, 3, 1024, 26000, 16),
                                       (17, 17, 4096, 5000, 64)])
def test_few_tokens_with_much_to_do(T, E, K, N, R):
    """More tiles and columns than clusters find room for: two kernels instead of one."""
    for dtype in (F16, BF16):
        x, y, down, up, ids, scales = make(T, K, N, E, R, dtype, seed=T)
        check(x, y, down, up, ids, scales, torch.arange(E, device=DEV, dtype=torch.int32) % (R + 3))
        ids[:] = torch.arange(T, device=DEV) % E
        check(x, y, down, up, ids)


def test_more_adapters_than_tokens_and_the_reverse():
    check(*make(20, 256, 128, 300, 8, F16))
    check(*make(600, 256, 128, 1, 8, F16))
    check(*make(1030, 64, 72, 500, 8, BF16))
    x, y, down, up, _, scales = make(257, 128, 96, 2, 16, F16)
    for ids in ([0] * 257, [-1] * 257, [5] * 257, [i % 2 for i in range(257)], [-1] * 256 + [1], [2 ** 31 - 1] * 200 + [0] * 57):
        check(x, y, down, up, torch.tensor(ids, dtype=torch.int32, device=DEV), scales)


def test_large_and_small_inner_values():
    """Inner sums beyond FP16's range, and so small that FP16 would lose them, with an outer matrix that brings them back."""
    for factor in (2.0 ** 9, 2.0 ** -12):
        x, y, down, up, ids, scales = make(40, 512, 200, 3, 16, F16)
        check((x * factor).to(F16), y, (down * (32 if factor > 1 else 0.25)).to(F16), (up * 2.0 ** (-13 if factor > 1 else 12)).to(F16), ids, scales)
    x, y, down, up, ids, scales = make(40, 512, 200, 3, 16, BF16)
    check((x * 1e15).to(BF16), y, (down * 1e10).to(BF16), (up * 1e-25).to(BF16), ids, scales)


def test_infinite_and_nan_activations_stay_with_their_token():
    for T in (12, 150):
        x, y, down, up, ids, scales = make(T, 128, 100, 2, 16, F16)
        ids[:] = torch.arange(T, device=DEV) % 2
        clean = _C_ops.low_rank_add(x, y, down, up, ids, scales=scales)
        x[3, 5], x[6, 0], y[8, 4] = math.inf, math.nan, math.inf
        got = _C_ops.low_rank_add(x, y, down, up, ids, scales=scales)
        assert not torch.isfinite(got[3]).any() and torch.isnan(got[6]).all() and got[8, 4] == math.inf
        rest = [t for t in range(T) if t not in (3, 6, 8)]
        assert torch.equal(got[rest], clean[rest])
        # an infinite weight acts on the tokens of its adapter alone
        down[1, 2, 3] = math.inf
        got = _C_ops.low_rank_add(x, y, down, up, ids, scales=scales)
        even = [t for t in rest if t % 2 == 0]
        assert torch.equal(got[even], clean[even]) and not torch.isfinite(got[1]).any()


def test_inner_values_that_overflow_are_infinite():
    """1e30 * 1e30 is infinite in FP32 and so is what it is added to, with the sign of `up`."""
    for T in (12, 150):
        x, y, down, up, ids, scales = make(T, 128, 100, 2, 16, BF16)
        ids[:] = torch.arange(T, device=DEV) % 2
        clean = _C_ops.low_rank_add(x, y, down, up, ids)
        x[3] = 1e30
        down[1] = 0
        down[1, 2] = 1e30
        up[1, :, 2] = torch.where(torch.arange(100, device=DEV) % 3 == 0, -0.5, 2.0)
        got = _C_ops.low_rank_add(x, y, down, up, ids)
        assert torch.equal(got[3].float(), torch.where(torch.arange(100, device=DEV) % 3 == 0, -math.inf, math.inf))
        even = [t for t in range(T) if t % 2 == 0]
        assert torch.equal(got[even], clean[even])


def test_strides_shapes_streams_and_capture():
    x, y, down, up, ids, scales = make(24, 256, 120, 3, 16, F16)
    want = check(x, y, down, up, ids, scales)
    wx, wy = torch.zeros(24, 300, dtype=F16, device=DEV), torch.full((24, 200), 3.0, dtype=F16, device=DEV)
    for ax, ay in ((8, 8), (1, 3)):
        sx, sy = wx[:, ax:ax + 256], wy[:, ay:ay + 120]
        sx.copy_(x)
        sy.copy_(y)
        assert torch.equal(_C_ops.low_rank_add(sx, sy, down, up, ids, scales=scales), want)
        assert torch.equal(_C_ops.low_rank_add(sx, sy, down, up, ids, scales=scales, out=sy), want)
        assert (wy[:, :ay] == 3).all() and (wy[:, ay + 120:] == 3).all()
        wy.fill_(3.0)
    assert torch.equal(_C_ops.low_rank_add(x.view(2, 3, 4, 256), y.view(2, 3, 4, 120), down, up, ids, scales=scales), want.view(2, 3, 4, 120))
    assert torch.equal(_C_ops.low_rank_add(x.T.contiguous().T, y.T.contiguous().T, down, up, ids.repeat_interleave(3)[::3], scales=scales), want)
    assert torch.equal(_C_ops.low_rank_add(x[0], y[0], down, up, ids[:1], scales=scales), want[0])
    assert _C_ops.low_rank_add(x[:0], y[:0], down, up, ids[:0]).shape == (0, 120)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_C_ops.low_rank_add(x, y, down, up, ids, scales=scales) for _ in range(4)]
    mine = [_C_ops.low_rank_add(x, y, down, up, ids, scales=scales) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got + mine)
    graph, i = torch.cuda.CUDAGraph(), ids.clone()
    with torch.cuda.graph(graph):
        got = _C_ops.low_rank_add(x, y, down, up, i, scales=scales)
    i.copy_(ids.flip(0))
    graph.replay()
    assert torch.equal(got, _C_ops.low_rank_add(x, y, down, up, ids.flip(0), scales=scales))


@pytest.mark.parametrize("T", [1, 5, 64, 128, 200])
def test_one_tensor_as_input_base_and_output(T):
    """x + up (down x), written over x."""
    x, _, down, up, ids, scales = make(T, 512, 512, 4, 16, F16, seed=T)
    for _ in range(5):
        mine = x.clone()
        want = _C_ops.low_rank_add(x, x, down, up, ids, scales=scales)
        assert _C_ops.low_rank_add(mine, mine, down, up, ids, scales=scales, out=mine) is mine and torch.equal(mine, want)
    # and where the output begins inside x
    wide = torch.zeros(T, 1200, dtype=F16, device=DEV)
    wide[:, :512] = x
    y = torch.randn(T, 512, device=DEV).to(F16)
    want = _C_ops.low_rank_add(x, y, down, up, ids, scales=scales)
    assert torch.equal(_C_ops.low_rank_add(wide[:, :512], y, down, up, ids, scales=scales, out=wide[:, 264:776]), want)


def test_the_module():
    g = torch.Generator(device=DEV).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV) * 0.1             # noqa: E731
    m = LowRankAdapters(4, 128, 96, 20, device=DEV, dtype=BF16)
    pairs = {i: (r(rank, 128), r(96, rank), scale) for i, rank, scale in ((0, 20, 1.0), (1, 3, 0.5), (3, 8, 2.0))}
    m.load(1, r(20, 128), r(96, 20), 9.0)                                    # replaced below by a smaller one
    for i, (a, b, s) in pairs.items():
        m.load(i, a, b, s)
    x, y = r(30, 128).to(BF16), r(30, 96).to(BF16)
    ids = (torch.arange(30, device=DEV) % 5 - 1).int()
    got = m(x, y, ids)
    down, up = torch.zeros(4, 24, 128, dtype=BF16, device=DEV), torch.zeros(4, 96, 24, dtype=BF16, device=DEV)
    for i, (a, b, _) in pairs.items():
        down[i, :len(a)], up[i, :, :len(a)] = a.to(BF16), b.to(BF16)
    want, bound = plain_ops.low_rank(x, y, down, up, ids, torch.tensor([1.0, 0.5, 0.0, 2.0]))
    plain_ops.within(got, want, plain_ops.rounded(want, bound, BF16))
    assert torch.equal(got[ids == 2], y[ids == 2])
    m.remove(3)
    assert torch.equal(m(x, y, ids)[ids == 3], y[ids == 3])
    m.scales[0] = 1.0 + 2.0 ** -20
    half = m.half()
    assert half.scales.dtype == torch.float32 and float(half.scales[0]) == 1.0 + 2.0 ** -20 and half.down.dtype == F16
    other = LowRankAdapters(4, 128, 96, 20, device=DEV)
    other.load_state_dict(half.state_dict())
    assert torch.equal(other(x.half(), y.half(), ids), half(x.half(), y.half(), ids))


def test_refusals():
    x, y, down, up, ids, scales = make(5, 64, 40, 3, 16, F16)
    base = dict(x=x, y=y, down=down, up=up, ids=ids)

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            _C_ops.low_rank_add(**{**base, **change})
    refused(RuntimeError, "CPU", x=x.cpu())
    refused(RuntimeError, "CPU", ids=ids.cpu())
    refused(TypeError, "x must be", x=x.float())
    refused(TypeError, "y must be", y=y.to(BF16))
    refused(TypeError, "ids", ids=ids.long())
    refused(ValueError, "ids", ids=ids[:4])
    refused(ValueError, "tokens", y=y[:4])
    refused(ValueError, "in_features", x=x[:, :32])
    refused(ValueError, "adapters", up=up[:2])
    refused(ValueError, "rank", down=down[:, :12].contiguous(), up=up[:, :, :12].contiguous())
    refused(ValueError, "contiguous", down=down[:, ::2], up=up[:, :, :8].contiguous())
    refused(ValueError, "scales", scales=scales[:2])
    refused(TypeError, "scales", scales=scales.half())
    refused(TypeError, "ranks", ranks=scales)
    refused(ValueError, "out", out=y[:4])
    refused(ValueError, "out", out=torch.zeros(40, 5, dtype=F16, device=DEV).T)
    refused(TypeError, "up must be a tensor", up=None)


@pytest.mark.parametrize("T,K,N,E,R,kernels", [
    (1, 4096, 12288, 8, 16, 1), (1, 4096, 12288, 8, 32, 1), (1, 4096, 12288, 8, 40, 2), (1, 4096, 1000, 8, 48, 2), (1, 512, 1000, 8, 256, 2),
    (4, 4096, 4096, 32, 16, 1), (4, 4096, 4096, 32, 24, 2), (4, 4096, 12288, 32, 16, 2), (16, 1024, 2048, 16, 8, 2), (16, 1024, 1000, 16, 32, 1),
    (77, 2912, 1003, 12, 8, 1), (28, 264, 1000, 28, 48, 1), (32, 264, 900, 40, 64, 1), (28, 264, 1000, 28, 72, 2), (36, 264, 1000, 36, 16, 2), (128, 264, 1000, 30, 24, 1)])
def test_one_kernel_where_two_are_not_faster(T, K, N, E, R, kernels):
    """Several rounds of 32 ranks, columns over several clusters, more tiles than clusters find room for: measured beside the rule."""
    x, y, down, up, ids, scales = make(T, K, N, E, R, BF16 if R % 16 else F16, seed=T + R)
    check(x, y, down, up, ids, scales, torch.arange(E, device=DEV, dtype=torch.int32) % (R + 3))
    ids[:] = torch.arange(T, device=DEV) % E
    check(x, y, down, up, ids)
    before = _lib.lib().ortho_b200_launch_count()
    _C_ops.low_rank_add(x, y, down, up, ids)
    assert _lib.lib().ortho_b200_launch_count() - before == kernels
