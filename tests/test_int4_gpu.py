"""Products with 4-bit weights against the same sums in 64 bits.

Tolerance, against M = sum |x| s (q + z), as the sums of x q and of x are taken apart.  Codes and both parts of x are exact in fp16; x is off by
2^-24 |x|, or by 2^-39 of the largest of its 64.  The 16 products of a step are added by the tensor core, taken as 17 truncations of 2^-24 M
(what it keeps is not documented): 2^-20 M a step, and no step has more than its share of M.  A tile's sum of x: 19 rounded
additions, 2^-20 M.  The difference, its scale and the addition round: 2^-22 M a tile, for at most the tiles of a slice, and
seven pairwise sums.  Then the bias and what is added, half a step each.
"""
import math

import pytest
import torch

from mx230_b200 import _lib
from mx230_b200 import llm_attention as la

pytestmark = pytest.mark.gpu


def weights(n_in, n_out, group, zeros, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-n_in // group)
    codes = torch.randint(0, 16, (n_in, n_out), device="cuda", generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(groups, n_out, device="cuda", generator=g)) * 0.01).half()
    z = torch.randint(0, 16, (groups, n_out), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z


class Dense:
    """s (q - z) and s (q + z) in 64 bits."""

    def __init__(self, codes, scales, z, group):
        at = torch.arange(codes.shape[0], device="cuda") // group
        zero, s = 8.0 if z is None else z.double()[at], scales.double()[at]
        self.w, self.mag = (codes.double() - zero) * s, (codes.double() + zero) * s

    def limit(self, x, want, *more):
        tiles, x = -(-self.w.shape[0] // 64), x.double().abs()
        out = x @ self.mag * (2.0 ** -19 + (tiles + 8) * 2.0 ** -22) + want.abs() * 2.0 ** -23 + 1e-30
        for t in more:
            out = out + t.double().abs() * 2.0 ** -23
        return out + x.amax(1, keepdim=True) * self.mag.amax(0) * self.w.shape[0] * 2.0 ** -35


def check(got, want, lim, what):
    err = (got.double() - want).abs()
    assert (err <= lim).all(), (what, float((err / lim).max()))


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128, 192])
@pytest.mark.parametrize("n_in,n_out,rows", [(1, 1, 1), (33, 17, 3), (64, 16, 1), (896, 1152, 1), (896, 1152, 5), (1000, 77, 2), (4864, 896, 8),
                                             (2047, 130, 4), (4160, 513, 11), (130, 40001, 7), (9000, 24, 16), (64, 5000, 33)])
def test_matches_the_sums(handle, n_in, n_out, rows, group, zeros):
    codes, scales, z = weights(n_in, n_out, group, zeros, n_in + n_out)
    w = la.pack_int4(handle, codes, scales, z, group=group)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, b, old = (torch.randn(*s, device="cuda", generator=g) for s in ((rows, n_in), (n_out,), (rows, n_out)))
    d = Dense(codes, scales, z, group)
    want = x.double() @ d.w
    y = torch.full((rows, n_out), math.nan, device="cuda")
    la.gemv_int4(handle, y, x, w)
    check(y, want, d.limit(x, want), "plain")
    la.gemv_int4(handle, y, x, w, b, add=old)
    want = want + b.double() + old.double()
    check(y, want, d.limit(x, want, b, old), "bias and add")
    acc = old.clone()
    la.gemv_int4(handle, acc, x, w, b, add=acc)
    assert torch.equal(acc, y), "added in place"


@pytest.mark.parametrize("n_in,n_out,group", [(896, 1152, 32), (4864, 896, 64), (14336, 96, 128), (300, 3000, 64), (4096, 6000, 128)])
def test_a_row_does_not_depend_on_the_others(handle, n_in, n_out, group):
    codes, scales, z = weights(n_in, n_out, group, True, 5)
    w = la.pack_int4(handle, codes, scales, z, group=group)
    x = torch.randn(37, n_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    alone = torch.empty(37, n_out, device="cuda")
    for r in range(37):
        la.gemv_int4(handle, alone[r], x[r], w)
    for n in (2, 3, 4, 5, 7, 8, 9, 12, 16, 17, 37):
        y = torch.empty(n, n_out, device="cuda")
        la.gemv_int4(handle, y, x[:n], w)
        assert torch.equal(y, alone[:n]), n


@pytest.mark.parametrize("n_in,n_out,rows,group", [(65536, 40, 5, 128), (32769, 100, 2, 32), (40000, 33, 9, 192), (4096, 2400, 3, 1 << 20), (700, 300, 4, 704)])
def test_long_rows_and_wide_groups(handle, n_in, n_out, rows, group):
    """Up to eight CTAs along the inputs, more rows than fit beside them, groups that end inside a stage or never."""
    codes, scales, z = weights(n_in, n_out, group, True, n_in)
    w = la.pack_int4(handle, codes, scales, z, group=group)
    x = torch.randn(rows, n_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    y, d = torch.empty(rows, n_out, device="cuda"), Dense(codes, scales, z, group)
    la.gemv_int4(handle, y, x, w)
    want = x.double() @ d.w
    check(y, want, d.limit(x, want), (n_in, group))
    handle.check_status()


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e20])
def test_ranges_of_x(handle, scale):
    """Very small, very large and mixed rows: x is split relative to the largest of 64 values."""
    n_in, n_out = 640, 200
    codes, scales, z = weights(n_in, n_out, 64, True, 9)
    w = la.pack_int4(handle, codes, scales, z)
    d = Dense(codes, scales, z, 64)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, n_in, device="cuda", generator=g) * scale
    x[1] = 0.0
    x[2, ::64] *= 1e6
    x[3, 64:128] = 0.0
    x[4] *= torch.exp2(torch.randint(-12, 12, (n_in,), device="cuda", generator=g).float())
    x[5, 1:] = 0.0
    y = torch.empty(6, n_out, device="cuda")
    la.gemv_int4(handle, y, x, w)
    want = x.double() @ d.w
    check(y, want, d.limit(x, want), scale)
    assert (y[1] == 0).all()


def test_infinities_and_nan_stay_in_their_row(handle):
    codes, scales, _ = weights(256, 64, 64, False, 2)
    w = la.pack_int4(handle, codes, scales)
    d = Dense(codes, scales, None, 64)
    x = torch.randn(7, 256, device="cuda")
    clean = torch.empty(7, 64, device="cuda")
    la.gemv_int4(handle, clean, x, w)
    x[2, 70], x[4, 3], x[5, 255] = math.nan, math.inf, -math.inf
    y = torch.empty(7, 64, device="cuda")
    la.gemv_int4(handle, y, x, w)
    assert torch.equal(y[[0, 1, 3, 6]], clean[[0, 1, 3, 6]])
    assert torch.isnan(y[2]).all()
    for r, k, v in ((4, 3, math.inf), (5, 255, -math.inf)):
        want = v * d.w[k]   # NaN where the weight is 0
        assert torch.equal(torch.isnan(want), torch.isnan(y[r])) and torch.equal(want[~torch.isnan(want)], y[r].double()[~torch.isnan(want)])


@pytest.mark.parametrize("n_in,group", [(256, 32), (250, 32), (97, 32), (160, 32), (64, 32), (256, 128), (130, 64)])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_one_infinity_gives_its_weight_the_sign(handle, n_in, group, value):
    """In either half of a tile, in the last one too, whose other half may be nothing: inf s (q - z), NaN where that is 0."""
    codes, scales, z = weights(n_in, 48, group, True, 4)
    w = la.pack_int4(handle, codes, scales, z, group=group)
    d = Dense(codes, scales, z, group)
    for rows in (1, 6):
        x = torch.randn(rows, n_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
        for k in (0, 33, n_in // 2, n_in - 1):
            if k >= n_in:
                continue
            at = x.clone()
            at[rows - 1, k] = value
            y = torch.empty(rows, 48, device="cuda")
            la.gemv_int4(handle, y, at, w)
            want = value * d.w[k]
            nan = torch.isnan(want)
            assert torch.equal(nan, torch.isnan(y[-1])) and torch.equal(want[~nan], y[-1].double()[~nan]), (rows, k)
            assert torch.isfinite(y[:-1]).all()


def test_strides_and_what_lies_beside(handle):
    n_in, n_out, rows = 200, 50, 6
    codes, scales, z = weights(n_in, n_out, 64, True, 3)
    w = la.pack_int4(handle, codes, scales, z)
    d = Dense(codes, scales, z, 64)
    for off, wide in ((0, 208), (1, 203), (3, 211)):
        store = torch.randn(rows * wide + 8, device="cuda")
        x = store[off:off + rows * wide].view(rows, wide)[:, :n_in]
        whole = torch.full((rows + 2, n_out + 7), 5.0, device="cuda")
        y = whole[1:rows + 1, 3:3 + n_out]
        add = torch.randn(rows, n_out + 1, device="cuda")[:, 1:]
        la.gemv_int4(handle, y, x, w, add=add)
        want = x.double() @ d.w + add.double()
        check(y, want, d.limit(x, want, add), off)
        inside = torch.zeros_like(whole, dtype=torch.bool)
        inside[1:rows + 1, 3:3 + n_out] = True
        assert (whole[~inside] == 5).all()
    one = torch.randn(1, n_in, device="cuda")
    y = torch.empty(4, n_out, device="cuda")
    la.gemv_int4(handle, y, one.expand(4, n_in), w)
    single = torch.empty(n_out, device="cuda")
    la.gemv_int4(handle, single, one[0], w)
    assert torch.equal(y, single.expand(4, n_out))


def test_high_bits_of_codes_and_large_zeros(handle):
    codes, scales, _ = weights(128, 32, 64, False, 4)
    z = torch.full((2, 32), 255, dtype=torch.uint8, device="cuda")
    x = torch.randn(2, 128, device="cuda")
    a, b = torch.empty(2, 32, device="cuda"), torch.empty(2, 32, device="cuda")
    la.gemv_int4(handle, a, x, la.pack_int4(handle, codes, scales, z))
    la.gemv_int4(handle, b, x, la.pack_int4(handle, codes + 240, scales, z))
    assert torch.equal(a, b)
    d = Dense(codes, scales, z, 64)
    want = x.double() @ d.w
    check(a, want, d.limit(x, want), "zeros of 255")


@pytest.mark.parametrize("n_in,n_out,rows,stage", [(896, 20000, 2, 0), (896, 20000, 6, 2), (14336, 4096, 8, 3), (4096, 40000, 1, 1), (4096, 40000, 1, 2)])
def test_weights_that_never_arrive(handle, n_in, n_out, rows, stage):
    """The wait for them ends, the outputs without them are NaN and the others right; the next call is right again."""
    codes, scales, z = weights(n_in, n_out, 64, True, 12)
    w = la.pack_int4(handle, codes, scales, z)
    x = torch.randn(rows, n_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    y, again = torch.empty(rows, n_out, device="cuda"), torch.zeros(rows, n_out, device="cuda")
    la.gemv_int4(handle, y, x, w)
    handle.check_status()
    try:
        handle.set_option(_lib.OPT_WAIT_LIMIT, 2000)   # 2e6 SM cycles, about 1 ms
        handle.set_option(_lib.OPT_TEST_DROP_TILE, stage)
        la.gemv_int4(handle, again, x, w)
        with pytest.raises(_lib.Mx230Error) as e:
            handle.check_status()
        assert e.value.code == _lib.ERR_DEVICE_STATUS
    finally:
        handle.set_option(_lib.OPT_TEST_DROP_TILE, -1)
        handle.set_option(_lib.OPT_WAIT_LIMIT, 4000000)
    lost = torch.isnan(again)
    assert lost.any() and not lost.all() and torch.equal(again[~lost], y[~lost])
    la.gemv_int4(handle, again, x, w)
    handle.check_status()
    assert torch.equal(again, y)


def test_captured_replayed_and_on_another_stream(handle):
    n_in, n_out = 4864, 896
    codes, scales, z = weights(n_in, n_out, 64, True, 7)
    w = la.pack_int4(handle, codes, scales, z)
    x, y = torch.randn(3, n_in, device="cuda"), torch.zeros(3, n_out, device="cuda")
    side = torch.cuda.Stream()
    la.gemv_int4(handle, y, x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        la.gemv_int4(handle, y, x, w)
        la.gemv_int4(handle, y, x, w, add=y)
    for seed in (1, 2):
        x.copy_(torch.randn(3, n_in, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(y)
        la.gemv_int4(handle, want, x, w)
        la.gemv_int4(handle, want, x, w, add=want)
        assert torch.equal(want, y)
    got = torch.zeros_like(y)
    torch.cuda.synchronize()
    la.gemv_int4(handle, got, x, w, stream=side)   # two at once
    la.gemv_int4(handle, want, x, w)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_refusals(handle):
    codes, scales, z = weights(256, 48, 64, True, 1)
    w = la.pack_int4(handle, codes, scales, z)
    x, y = torch.zeros(2, 256, device="cuda"), torch.zeros(2, 48, device="cuda")
    la.gemv_int4(handle, y[:0], x[:0], w)
    bad = [lambda: la.gemv_int4(handle, y, x[:, :255], w), lambda: la.gemv_int4(handle, y[:1], x, w), lambda: la.gemv_int4(handle, y, x.half(), w),
           lambda: la.gemv_int4(handle, y.cpu(), x, w), lambda: la.gemv_int4(handle, y, x, w, torch.zeros(47, device="cuda")),
           lambda: la.gemv_int4(handle, y, x, w, add=y[:1]), lambda: la.gemv_int4(handle, y[:1].expand(2, 48), x, w),
           lambda: la.gemv_int4(handle, torch.zeros(48, 2, device="cuda").t(), x, w),
           lambda: la.pack_int4(handle, codes, scales.float(), z), lambda: la.pack_int4(handle, codes, scales, z[:2]),
           lambda: la.pack_int4(handle, codes, scales, z, group=128), lambda: la.pack_int4(handle, codes.t(), scales, z),
           lambda: la.pack_int4(handle, codes[:60].contiguous(), scales[:1].contiguous())]   # 64 or 128 or more
    for call in bad:
        with pytest.raises(_lib.Mx230Error) as e:
            call()
        assert e.value.code == _lib.ERR_INVALID_ARG
    long = la.pack_int4(handle, torch.zeros(65537, 4, dtype=torch.uint8, device="cuda"), torch.zeros(513, 4, dtype=torch.float16, device="cuda"), group=128)
    with pytest.raises(_lib.Mx230Error) as e:
        la.gemv_int4(handle, torch.zeros(1, 4, device="cuda"), torch.zeros(1, 65537, device="cuda"), long)
    assert e.value.code == _lib.ERR_UNSUPPORTED
    with pytest.raises(_lib.Mx230Error) as e:
        la.pack_int4(handle, codes, torch.zeros(6, 48, dtype=torch.float16, device="cuda"), group=48)
    assert e.value.code == _lib.ERR_UNSUPPORTED
