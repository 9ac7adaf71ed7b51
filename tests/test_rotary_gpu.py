"""Rotary positions in the forms beyond the reference's against the formula in 64 bits.

Tolerance.  cos and sin: the remainder of the angle is rounded to 2^-28 turns (2.4e-8 rad), the function is good to an ulp (6e-8), the
factor rounds once more (6e-8): below 1.5e-7.  Two products with it, one of them rounded, and the rounded sum: below
(|a| + |b|) factor 3e-7; then half a step of the output's type.
"""
import math

import numpy as np
import pytest
import torch

from mx230_b200 import _lib
from mx230_b200 import llm_attention as la

pytestmark = pytest.mark.gpu

SCALINGS = [None, {"kind": "linear", "factor": 4.0}, {"kind": "ntk", "factor": 8.0},
            {"kind": "wavelength", "factor": 8.0, "low": 1.0, "high": 4.0, "length": 8192},
            {"kind": "yarn", "factor": 16.0, "slow": 1.0, "fast": 32.0, "length": 4096}]


def frequencies(rot, theta, s):
    """Written from the formulas, in 64 bits: (radians per position, factor)."""
    i = np.arange(rot // 2)
    f = theta ** (-2.0 * i / rot)
    if s is None:
        return f, 1.0
    if s["kind"] == "linear":
        return f / s["factor"], 1.0
    if s["kind"] == "ntk":
        return (theta * s["factor"] ** (rot / (rot - 2.0))) ** (-2.0 * i / rot) if rot > 2 else f, 1.0
    if s["kind"] == "wavelength":
        smooth = np.clip((s["length"] * f / (2 * np.pi) - s["low"]) / (s["high"] - s["low"]), 0, 1)
        return smooth * f + (1 - smooth) * f / s["factor"], 1.0
    pair = lambda turns: rot * math.log(s["length"] / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = max(math.floor(pair(s["fast"])), 0), min(math.ceil(pair(s["slow"])), rot - 1)
    ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
    return ramp * f / s["factor"] + (1 - ramp) * f, 0.1 * math.log(s["factor"]) + 1


def plain(x, pos, freq, factor, interleaved, inverse):
    """(result, bound on the error before the last rounding) in 64 bits; x [n][heads][dim] on the host."""
    x, half = x.double(), len(freq)
    ang = torch.from_numpy(np.asarray(pos, np.float64)[:, None] * freq)[:, None]
    c, s = torch.cos(ang) * factor, torch.sin(ang) * factor * (-1 if inverse else 1)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, tol = x.clone(), torch.zeros_like(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    tol[..., a] = tol[..., b] = (x[..., a].abs() + x[..., b].abs()) * factor * 3e-7
    return y, tol


def close(got, want, tol, what):
    err = (got.double().cpu() - want).abs()
    t = got.dtype
    limit = tol + want.abs() * (torch.finfo(t).eps / 2 if t != torch.float32 else 0.0) + (2.0 ** -25 if t == torch.float16 else 1e-37)
    assert (err <= limit).all(), (what, float((err - limit).max()), float(err.max()))


def run(handle, x, pos, plan, inverse=False, out=None, **kw):
    out = torch.full_like(x, 7.0, memory_format=torch.contiguous_format) if out is None else out
    la.rotary(handle, out, x, pos, plan, inverse, **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,heads,dim,rot", [(1, 1, 2, 2), (1, 16, 64, 64), (5, 3, 64, 32), (37, 12, 80, 20), (130, 7, 65, 64), (33, 2, 96, 24),
                                             (700, 1, 128, 128), (3, 300, 64, 64), (2, 5, 1024, 1024), (9, 4, 7, 6), (2, 2, 4100, 4096)])
def test_matches_the_formula(handle, n, heads, dim, rot, dtype, interleaved):
    g = torch.Generator().manual_seed(n * 1000 + dim)
    x = torch.randn(n, heads, dim, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (n,), generator=g, dtype=torch.int32)
    s = SCALINGS[(n + heads + rot) % len(SCALINGS)]
    plan = la.Rotary(rot, 5e5, s, interleaved)
    freq, factor = frequencies(rot, 5e5, s)
    for inverse in (False, True):
        got = run(handle, x.cuda(), pos.cuda(), plan, inverse)
        want, tol = plain(x, pos.numpy(), freq, factor, interleaved, inverse)
        close(got, want, tol, (n, heads, dim, rot, inverse))
        assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
        again = x.cuda()
        run(handle, again, pos.cuda(), plan, inverse, out=again)
        assert torch.equal(again, got), "in place"


@pytest.mark.parametrize("s", SCALINGS)
@pytest.mark.parametrize("rot", [2, 8, 64, 128])
def test_scaled_frequencies(handle, s, rot):
    """One pair at a time, at positions where a frequency's error would show: 1e6 positions of 2^-53 relative error are 1e-10 rad."""
    plan = la.Rotary(rot, 1e4, s)
    freq, factor = frequencies(rot, 1e4, s)
    assert abs(plan.factor - factor) <= 2 ** -24 * factor
    x = torch.ones(4, 1, rot)
    pos = torch.tensor([0, 1, 999_983, 16_777_259], dtype=torch.int32)
    want, tol = plain(x, pos.numpy(), freq, factor, False, False)
    close(run(handle, x.cuda(), pos.cuda(), plan), want, tol + 1e-8, s)


def test_positions_without_a_tensor_and_extreme_ones(handle):
    plan = la.Rotary(64, 1e6)
    freq, factor = frequencies(64, 1e6, None)
    x = torch.randn(6, 2, 64, generator=torch.Generator().manual_seed(3))
    for first in (0, -3, 2 ** 31 - 6, -(2 ** 31)):
        pos = np.arange(first, first + 6, dtype=np.int64)
        # 2^31 positions of half a unit of 2^-64 turns, and of the oracle's 2^-53: 1e-6 rad
        want, tol = plain(x, pos, freq, factor, False, False)
        got = run(handle, x.cuda(), first, plan)
        close(got, want, tol + (2e-6 if abs(first) > 1000 else 0.0), first)
        assert torch.equal(got, run(handle, x.cuda(), torch.from_numpy(pos).to(torch.int32).cuda(), plan))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_what_lies_beside(handle, dtype):
    """q and k heads of q|k|v rows into head-major order and back; nothing else is written; a head that is broadcast."""
    n, nh, nkv = 45, 6, 2
    g = torch.Generator().manual_seed(8)
    rows = torch.randn(n, (nh + 2 * nkv) * 64 + 8, generator=g).to(dtype).cuda()
    qk = rows[:, :(nh + 2 * nkv) * 64].view(n, nh + 2 * nkv, 64)[:, :nh + nkv]
    plan = la.Rotary(48, 1e4)
    freq, factor = frequencies(48, 1e4, None)
    want, tol = plain(qk.cpu(), np.arange(n) + 100, freq, factor, False, False)
    whole = torch.full((nh + nkv + 1, n + 2, 64), 3.0, dtype=dtype, device="cuda")
    head_major = whole[:nh + nkv, 1:n + 1].transpose(0, 1)
    close(run(handle, qk, 100, plan, out=head_major), want, tol, "head-major")
    assert (whole[nh + nkv] == 3).all() and (whole[:, 0] == 3).all() and (whole[:, n + 1] == 3).all()
    back = torch.empty_like(qk, memory_format=torch.contiguous_format)
    want2, tol2 = plain(head_major.cpu(), np.arange(n) + 100, freq, factor, False, True)
    close(run(handle, head_major, 100, plan, True, out=back), want2, tol2, "back")
    before = rows.clone()
    run(handle, qk, 100, plan, out=qk)
    assert torch.equal(rows[:, (nh + nkv) * 64:], before[:, (nh + nkv) * 64:]), "the rest of a row"
    assert torch.equal(qk, head_major)
    one = torch.randn(n, 1, 64, generator=g).to(dtype).cuda()
    out = run(handle, one.expand(n, 5, 64), 0, plan)
    assert torch.equal(out, run(handle, one, 0, plan).expand(n, 5, 64))
    for off in (1, 2, 3):   # rows that no wide access fits
        flat = torch.randn(n * 130 + 8, generator=g).to(dtype).cuda()
        view = flat[off:off + n * 130].view(n, 130)[:, :128].unflatten(1, (2, 64))
        want, tol = plain(view.cpu(), np.arange(n), freq, factor, False, False)
        close(run(handle, view, 0, plan), want, tol, off)


@pytest.mark.parametrize("interleaved", [False, True])
def test_infinities_and_nan_stay_in_their_pair(handle, interleaved):
    x = torch.randn(4, 2, 24)
    x[0, 0, 3], x[1, 1, 20], x[2, 0, 21] = math.inf, math.nan, -math.inf   # the last two behind the rotated part
    plan = la.Rotary(16, 1e4, interleaved=interleaved)
    got = run(handle, x.cuda(), 5, plan).cpu()
    bad = {(0, 0, 3), (0, 0, 2 if interleaved else 11), (1, 1, 20), (2, 0, 21)}
    assert {tuple(i) for i in torch.nonzero(~torch.isfinite(got)).tolist()} == bad
    assert got[2, 0, 21] == -math.inf


@pytest.mark.parametrize("s", [SCALINGS[0], SCALINGS[4]])
def test_the_inverse_is_the_gradient(handle, s):
    """f(x) = <dy, rotary(x)> is linear: its gradient along e is f(e), by differences (f(x + e) - f(x - e)) / 2, and <inverse(dy), e>."""
    n, heads, dim = 60, 5, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    x, e, dy = (torch.randn(n, heads, dim, device="cuda", generator=g) for _ in range(3))
    plan = la.Rotary(48, 1e4, s)
    dx = run(handle, dy, 77, plan, inverse=True).double()
    f = lambda v: (dy.double() * run(handle, v, 77, plan).double()).sum()  # noqa: E731
    diff, want = float(f(x + e) - f(x - e)) / 2, float((dx * e.double()).sum())
    # every product is off by 3e-7 (|a| + |b|) |dy| and the sum x + e rounds: 19200 of them, at random
    scale = float((dy.abs().double() * (x.abs() + e.abs()).double()).sum())
    assert abs(diff - want) <= 1e-6 * scale
    freq, factor = frequencies(48, 1e4, s)
    formula, tol = plain(dy.cpu(), np.arange(n) + 77, freq, factor, False, True)
    close(dx.float(), formula, tol, "formula")


def test_captured_replayed_and_on_another_stream(handle):
    n, heads = 64, 16
    x = torch.randn(n, heads, 64, device="cuda")
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    plan = la.Rotary(64, 1e6)
    out = torch.zeros_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        la.rotary(handle, out, x, pos, plan)
    for first in (0, 1000):
        pos.copy_(torch.arange(first, first + n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(handle, x, first, plan))
    got = torch.zeros_like(x)
    with torch.cuda.stream(side):
        la.rotary(handle, got, x, 1000, plan)
    side.synchronize()
    assert torch.equal(got, out)
    got.zero_()
    torch.cuda.synchronize()
    la.rotary(handle, got, x, 1000, plan, stream=side)
    side.synchronize()
    assert torch.equal(got, out)


def test_empty_and_beyond_32_bits(handle):
    plan = la.Rotary(64, 1e4)
    la.rotary(handle, torch.empty(0, 4, 64, device="cuda"), torch.empty(0, 4, 64, device="cuda"), 0, plan)
    la.rotary(handle, torch.empty(4, 0, 64, device="cuda"), torch.empty(4, 0, 64, device="cuda"), 0, plan)
    # two rows 2^31 + 64 elements apart
    far = torch.empty(2 ** 31 + 128, dtype=torch.bfloat16, device="cuda")
    x = far.as_strided((2, 1, 64), (2 ** 31 + 64, 64, 1))
    v = torch.randn(2, 1, 64, device="cuda").bfloat16()
    x.copy_(v)
    run(handle, x, 9, plan, out=x)
    assert torch.equal(x, run(handle, v, 9, plan))


def test_refusals(handle):
    x = torch.zeros(4, 2, 64, device="cuda")
    plan = la.Rotary(64, 1e4)
    bad = [lambda: la.rotary(handle, x, x.cpu(), 0, plan), lambda: la.rotary(handle, x[:3], x, 0, plan),
           lambda: la.rotary(handle, x.half(), x, 0, plan), lambda: la.rotary(handle, x.double(), x.double(), 0, plan),
           lambda: la.rotary(handle, x, x, torch.zeros(4, dtype=torch.int64, device="cuda"), plan),
           lambda: la.rotary(handle, x, x, torch.zeros(3, dtype=torch.int32, device="cuda"), plan),
           lambda: la.rotary(handle, x[..., :32], x[..., :32], 0, plan),          # more rotated than there is
           lambda: la.rotary(handle, x.transpose(1, 2), x.transpose(1, 2), 0, plan),
           lambda: la.rotary(handle, x[:1].expand(4, 2, 64), x, 0, plan),         # the rows of the output share memory
           lambda: la.rotary(handle, x.as_strided((4, 2, 64), (32, 64, 1)), x.clone(), 0, plan),
           lambda: la.rotary(handle, x, x.as_strided((4, 2, 64), (64, 256, 1)), 0, plan)]   # in place with other strides
    for call in bad:
        with pytest.raises(_lib.Mx230Error) as e:
            call()
        assert e.value.code == _lib.ERR_INVALID_ARG
