"""What the C entry points beside the attention step refuse before they touch the device: calls with a handle that no device stands
behind (all of these return before it is looked at), and the host-side table of rotary frequencies."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from mx230_b200 import _lib, serving
from mx230_b200 import llm_attention as la


@pytest.fixture(scope="module")
def L(lib_built):
    return _lib.lib()


FAKE = C.create_string_buffer(1 << 16)   # a handle of zeros
H = C.addressof(FAKE)
P = 1 << 20                              # an address that is never used, 16-byte aligned


def test_rotary_refuses(L):
    ok = dict(h=H, st=None, out=P, x=P + 4096, dt=0, pos=None, pos0=0, turns=P, factor=1.0, rows=4, heads=2, dim=64, rot=64, inter=0, inv=0,
              xr=128, xh=64, outr=128, outh=64)
    cases = [dict(h=None), dict(out=None), dict(x=None), dict(turns=None), dict(dt=3), dict(dt=-1), dict(rows=-1), dict(heads=-1), dict(rot=63),
             dict(rot=0), dict(rot=66), dict(dim=0), dict(xr=-1), dict(outh=-64), dict(outr=0), dict(outh=0), dict(outr=64), dict(outh=32),
             dict(outr=100, outh=64), dict(out=P + 4096, outr=256), dict(x=P + 4097), dict(out=P + 2), dict(turns=P + 4), dict(pos=P + 2)]
    for c in cases:
        assert L.mx230_rotary(*{**ok, **c}.values()) == _lib.ERR_INVALID_ARG, c
    assert L.mx230_rotary(*{**ok, "dim": 8192, "rot": 8192, "outh": 8192, "outr": 16384}.values()) == _lib.ERR_UNSUPPORTED
    assert L.mx230_rotary(*{**ok, "rows": 0}.values()) == 0 and L.mx230_rotary(*{**ok, "heads": 0}.values()) == 0


def test_rotary_table(L):
    t, f = (C.c_uint64 * 32)(), C.c_float()
    table = lambda *a: L.mx230_rotary_table(t, C.byref(f), *a)  # noqa: E731
    for bad in [(63, 1e4, 0, 1.0, 0.0, 0.0, 0), (0, 1e4, 0, 1.0, 0.0, 0.0, 0), (64, 0.0, 0, 1.0, 0.0, 0.0, 0), (64, math.inf, 0, 1.0, 0.0, 0.0, 0),
                (64, math.nan, 0, 1.0, 0.0, 0.0, 0), (64, 1e4, 5, 1.0, 0.0, 0.0, 0), (64, 1e4, 1, 0.0, 0.0, 0.0, 0), (64, 1e4, 2, math.nan, 0.0, 0.0, 0),
                (64, 1e4, 3, 8.0, 4.0, 1.0, 8192), (64, 1e4, 3, 8.0, 1.0, 4.0, 0), (64, 1e4, 4, 8.0, 1.0, 1.0, 8192), (64, 1.0, 4, 8.0, 1.0, 32.0, 8192)]:
        assert table(*bad) == _lib.ERR_INVALID_ARG, bad
    assert L.mx230_rotary_table(None, C.byref(f), 64, 1e4, 0, 1.0, 0.0, 0.0, 0) == _lib.ERR_INVALID_ARG
    assert table(64, 1e4, 0, 1.0, 0.0, 0.0, 0) == 0 and f.value == 1.0
    turns = np.array(t, np.uint64).astype(np.float64) / 2.0 ** 64
    want = 1e4 ** (-np.arange(32) / 32) / (2 * np.pi)
    # a power and a quotient in 64 bits on either side, and half a unit of 2^-64 turns: at 2e-5 turns that is 2^-49 of the value
    assert (np.abs(turns - want) <= 4 * 2.0 ** -53 * want + 2.0 ** -65).all()
    assert table(64, 0.001, 0, 1.0, 0.0, 0.0, 0) == 0   # frequencies above a turn a position: the remainder
    turns = np.array(t, np.uint64).astype(np.float64) / 2.0 ** 64
    want = np.mod(0.001 ** (-np.arange(32) / 32) / (2 * np.pi), 1.0)
    assert np.abs(turns - want).max() < 1e-12
    assert table(64, 1e4, 4, 16.0, 1.0, 32.0, 4096) == 0 and abs(f.value - (0.1 * math.log(16) + 1)) < 1e-7


def test_int4_refuses(L):
    ok = dict(h=H, st=None, y=P, x=P + 65536, packed=P, bias=None, add=None, rows=4, n_in=256, n_out=64, group=64, xs=256, ys=64, adds=0)
    cases = [dict(h=None), dict(y=None), dict(x=None), dict(packed=None), dict(rows=-1), dict(n_in=0), dict(n_out=0), dict(n_in=-5), dict(xs=-1),
             dict(ys=63), dict(ys=-64), dict(add=P + 64, adds=-1), dict(add=P, adds=0), dict(packed=P + 8), dict(y=P + 2), dict(x=P + 1), dict(bias=P + 2), dict(x=P), dict(bias=P),
             dict(rows=1, x=P)]
    for c in cases:
        assert L.mx230_gemv_int4(*{**ok, **c}.values()) == _lib.ERR_INVALID_ARG, c
    for g in (0, -64, 16, 48, 96, 31):
        assert L.mx230_gemv_int4(*{**ok, "group": g}.values()) == _lib.ERR_UNSUPPORTED, g
    assert L.mx230_gemv_int4(*{**ok, "rows": 1 << 30}.values()) == _lib.ERR_UNSUPPORTED
    assert L.mx230_gemv_int4(*{**ok, "n_in": 65537, "xs": 65537}.values()) == _lib.ERR_UNSUPPORTED
    assert L.mx230_gemv_int4(*{**ok, "rows": 0}.values()) == 0
    pk = dict(h=H, st=None, packed=P, codes=P, scales=P, zeros=None, n_in=256, n_out=64, group=64)
    for c in [dict(h=None), dict(packed=None), dict(codes=None), dict(scales=None), dict(packed=P + 4), dict(scales=P + 1), dict(n_in=0), dict(n_out=-1)]:
        assert L.mx230_pack_int4(*{**pk, **c}.values()) == _lib.ERR_INVALID_ARG, c
    assert L.mx230_pack_int4(*{**pk, "group": 40}.values()) == _lib.ERR_UNSUPPORTED
    # 16 x 64 tiles of 512 bytes, 64 bytes per 16 outputs and group
    assert L.mx230_int4_bytes(256, 64, 64) == 4 * 4 * 512 + 4 * 4 * 64 and L.mx230_int4_bytes(65, 17, 32) == 2 * 2 * 512 + 2 * 3 * 64
    assert L.mx230_int4_bytes(0, 64, 64) == 0 and L.mx230_int4_bytes(1 << 17, 1 << 19, 64) == (1 << 15) * (1 << 11) * 576


def test_sample_refuses(L):
    ok = dict(h=H, st=None, token=P, prob=None, logits=P, dt=0, rows=4, vocab=100, stride=100, u=P, t=1.0, ts=None, k=0, ks=None, p=1.0, ps=None,
              m=0.0, ms=None)
    cases = [dict(h=None), dict(token=None), dict(logits=None), dict(u=None), dict(dt=3), dict(rows=-1), dict(vocab=0), dict(vocab=-1), dict(stride=-1),
             dict(logits=P + 2), dict(logits=P + 1, dt=1), dict(token=P + 2), dict(prob=P + 1), dict(u=P + 2), dict(ts=P + 2), dict(ks=P + 1),
             dict(ps=P + 3), dict(ms=P + 2)]
    for c in cases:
        assert L.mx230_sample(*{**ok, **c}.values()) == _lib.ERR_INVALID_ARG, c
    assert L.mx230_sample(*{**ok, "vocab": (1 << 22) + 1}.values()) == _lib.ERR_UNSUPPORTED
    assert L.mx230_sample(*{**ok, "rows": 1 << 28}.values()) == _lib.ERR_UNSUPPORTED
    assert L.mx230_sample(*{**ok, "rows": 0}.values()) == 0


class _Lib:
    """In the library's place: a call of it fails the test."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


class _Handle:
    device, _h = 0, H


class _Tensor(torch.Tensor):
    """A tensor of the CPU that says that it lies on device 0."""

    def get_device(self):
        return 0


def t(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype).as_subclass(_Tensor)


@pytest.mark.parametrize("big", [1 << 31, (1 << 32) + 1, -(1 << 31) - 1, -(1 << 40)])
def test_numbers_beyond_32_bits(monkeypatch, big):
    """An int argument would lose its upper bits on the way into the library."""
    monkeypatch.setattr(_lib, "_lib", _Lib())
    h, x = _Handle(), t(3, 2, 8)
    plan = la.Rotary.__new__(la.Rotary)
    plan.rot_dim, plan.interleaved, plan.factor, plan._addr, plan._device = 8, 0, 1.0, P, 0
    refused = []
    for call in (lambda: la.rotary(h, x, x, big, plan, stream=0), lambda: la.Rotary(big, 1e4, device="cpu"),
                 lambda: la.Rotary(8, 1e4, {"kind": "yarn", "factor": 2.0, "slow": 1.0, "fast": 32.0, "length": big}, device="cpu"),
                 lambda: la.pack_int4(h, t(40, 8, dtype=torch.uint8), t(1, 8, dtype=torch.float16), group=big, stream=0),
                 lambda: serving.sample(h, t(3, dtype=torch.int32), t(3, 10), t(3), top_k=big, stream=0)):
        with pytest.raises(_lib.Mx230Error) as e:
            call()
        refused.append(e.value.code)
    assert refused == [_lib.ERR_INVALID_ARG] * 5


def test_lengths_beyond_32_bits(monkeypatch):
    monkeypatch.setattr(_lib, "_lib", _Lib())
    h, n = _Handle(), (1 << 32) + 1
    plan = la.Rotary.__new__(la.Rotary)
    plan.rot_dim, plan.interleaved, plan.factor, plan._addr, plan._device = 2, 0, 1.0, P, 0
    one = lambda dtype=torch.float32: t(1, dtype=dtype)  # noqa: E731
    many = lambda *shape, dtype=torch.float32: one(dtype).expand(*shape)  # noqa: E731
    w = la.Int4Weights.__new__(la.Int4Weights)
    w.packed, w.n_in, w.n_out, w.group, w._addr, w._device = None, 1, 1, 64, P, 0
    for call in (lambda: la.rotary(h, many(n, 1, 1), many(n, 1, 1), 0, plan, stream=0),
                 lambda: la.gemv_int4(h, many(n, 1), many(n, 1), w, stream=0),
                 lambda: serving.sample(h, many(n, dtype=torch.int32), many(n, 1), many(n), stream=0)):
        with pytest.raises(_lib.Mx230Error):
            call()


def test_seeds():
    for seed in (-1, 1 << 128):
        with pytest.raises(_lib.Mx230Error):
            serving.Sampler(_Handle(), seed)
    assert 0.0 <= serving.Sampler(_Handle(), (1 << 128) - 1).uniform(0, 0) < 1.0
