"""Products with 4-bit weights where sums could lose what a 64-bit sum does not: inputs that are far larger than the others, or infinite;
and groups of 32 with outputs wide enough for two and four output tiles a warp.

Tolerance, against M = sum |x| |w|.  Weights are exact, x is off by 2^-23 |x| or by 2^-39 of the largest of its 64.  The 16 products of a
step are added by the tensor core, taken as 17 truncations of 2^-24 M (what it keeps is not documented): 2^-19 M for all steps with
the first term.  Scale and addition round: 2^-22 M a tile, for at most the tiles of a slice, and seven pairwise sums.
"""
import math

import pytest
import torch

from mx230_b200 import llm_attention as la

pytestmark = pytest.mark.gpu


def weights(n_in, n_out, group, zeros, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-n_in // group)
    codes = torch.randint(0, 16, (n_in, n_out), device="cuda", generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(groups, n_out, device="cuda", generator=g)) * 0.01).half()
    z = torch.randint(0, 16, (groups, n_out), device="cuda", generator=g, dtype=torch.uint8) if zeros else torch.full((groups, n_out), 8, device="cuda", dtype=torch.uint8)
    return codes, scales, z


def dense(codes, scales, z, group):
    at = torch.arange(codes.shape[0], device="cuda") // group
    return (codes.double() - z.double()[at]) * scales.double()[at]


def limit(x, w):
    x, w, n_in = x.double().abs(), w.abs(), w.shape[0]
    tiles = -(-n_in // 64)
    out = x @ w * (2.0 ** -19 + (tiles + 8) * 2.0 ** -22) + 1e-30
    for t in range(0, n_in, 64):
        out = out + x[:, t:t + 64].amax(1, keepdim=True) * w[t:t + 64].sum(0) * 2.0 ** -39
    return out


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n_in,n_out,rows", [(500, 96, 1), (500, 5000, 2), (500, 20000, 1), (900, 3000, 4), (4096, 500, 3), (900, 700, 8), (500, 9000, 6)])
def test_what_has_weight_zero_does_not_count(handle, n_in, n_out, rows, group, zeros):
    """A few inputs a million times as large as the others, with codes that are their zero points."""
    codes, scales, z = weights(n_in, n_out, group, zeros, n_in + rows)
    x = torch.randn(rows, n_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows))
    for k in (3, 70, n_in // 2, n_in - 1):
        codes[k] = z[k // group]
        x[:, k] *= 1e6
    w = la.pack_int4(handle, codes, scales, z if zeros else None, group=group)
    d = dense(codes, scales, z, group)
    y = torch.empty(rows, n_out, device="cuda")
    la.gemv_int4(handle, y, x, w)
    err, lim = (y.double() - x.double() @ d).abs(), limit(x, d)
    assert (err <= lim).all(), float((err / lim).max())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 3, 7])
@pytest.mark.parametrize("first,second", [(5, 9), (5, 40), (5, 70), (130, 249), (64, 127)])
@pytest.mark.parametrize("signs", [(1, 1), (1, -1), (-1, -1)])
def test_several_infinities(handle, first, second, signs, rows, group):
    """Of one sign or of both, in one step, tile or group or not: infinite of the sum's sign, NaN where both meet or a weight is 0."""
    codes, scales, z = weights(250, 500, group, True, 6)
    w, d = la.pack_int4(handle, codes, scales, z, group=group), dense(codes, scales, z, group)
    x = torch.randn(rows, 250, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8))
    clean, y = torch.empty(rows, 500, device="cuda"), torch.empty(rows, 500, device="cuda")
    la.gemv_int4(handle, clean, x, w)
    x[-1, first], x[-1, second] = signs[0] * math.inf, signs[1] * math.inf
    la.gemv_int4(handle, y, x, w)
    want = x[-1, first].double() * d[first] + x[-1, second].double() * d[second]
    nan = torch.isnan(want)
    assert nan.any() and not nan.all()
    assert torch.equal(torch.isnan(y[-1]), nan) and torch.equal(y[-1].double()[~nan], want[~nan])
    assert torch.equal(y[:-1], clean[:-1])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n_in,n_out,rows", [(896, 5001, 1), (4096, 6000, 2), (97, 40001, 1), (2047, 4000, 4), (33, 9007, 2), (700, 30000, 3), (4160, 14336, 1), (31, 20001, 2)])
def test_wide_products_in_groups_of_32(handle, n_in, n_out, rows, zeros):
    """An odd number of groups, inputs that end inside one, outputs that end inside a tile or a warp's tiles; a row's bits are those of the row alone."""
    codes, scales, z = weights(n_in, n_out, 32, zeros, n_in)
    w, d = la.pack_int4(handle, codes, scales, z if zeros else None, group=32), dense(codes, scales, z, 32)
    x = torch.randn(8, n_in, device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows))
    y, other, all8 = (torch.full((n, n_out), math.nan, device="cuda") for n in (rows, 1, 8))
    la.gemv_int4(handle, y, x[:rows], w)
    err, lim = (y.double() - x[:rows].double() @ d).abs(), limit(x[:rows], d)
    assert (err <= lim).all(), float((err / lim).max())
    la.gemv_int4(handle, other[0], x[rows - 1], w)
    la.gemv_int4(handle, all8, x, w)
    assert torch.equal(other[0], y[-1]) and torch.equal(all8[:rows], y)


def test_packed_on_another_stream(handle):
    """Its memory is not what was freed on the current stream, where work may still use it."""
    codes, scales, z = weights(4096, 2048, 64, True, 3)
    side = torch.cuda.Stream()
    x, y, want = torch.randn(2, 4096, device="cuda"), torch.empty(2, 2048, device="cuda"), torch.empty(2, 2048, device="cuda")
    w = la.pack_int4(handle, codes, scales, z)
    la.gemv_int4(handle, want, x, w)
    size, freed = w.nbytes(), w.packed.data_ptr()
    del w
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        w = la.pack_int4(handle, codes, scales, z, stream=stream)
        assert w.nbytes() == size and w.packed.data_ptr() != freed
        side.synchronize()
        y.zero_()
        la.gemv_int4(handle, y, x, w)
        assert torch.equal(y, want)
        torch.cuda.synchronize()
    again = la.pack_int4(handle, codes, scales, z)
    assert again.packed.data_ptr() == freed   # (the allocator does give that memory to the stream it was freed on)
