"""Host mirror of the reference engine's per-layer attention step
(03-llm-engine/src/gpu.rs:2570-2672 decode, :2808-2918 graph decode, :3204-3347 prefill
write path, :3530-3628 batched decode): RoPE -> KV write -> attention, with the kernel
chosen by (cache format, paging).  One Python function per reference kernel symbol,
same argument order; `KvCache` and `Paging` mirror gpu.rs:188-205 and :381-539.
Tensors are torch CUDA tensors; nothing here synchronises or allocates on the step path.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import addr, check, lib, ptr, require, require_int32
from .common import Handle, raw_stream, stream_ptr

KV_BLOCK = 16  # 03-llm-engine/src/gpu.rs:209


class KvCache:
    """One layer's KV cache: fp32 `[slots][n_kv_head*64]`, or int8 codes of that shape
    plus per-(slot, kv head) fp32 scale (and beta when `affine`), gpu.rs:188-205."""

    def __init__(self, slots: int, n_kv_head: int, head_dim: int = 64, quant: bool = False,
                 affine: bool = True, device="cuda"):
        self.slots, self.n_kv_head, self.head_dim = slots, n_kv_head, head_dim
        self.quant, self.affine = quant, affine
        kvd = n_kv_head * head_dim
        if quant:
            self.k = torch.zeros(slots, kvd, dtype=torch.int8, device=device)
            self.v = torch.zeros(slots, kvd, dtype=torch.int8, device=device)
            self.ks = torch.zeros(slots, n_kv_head, dtype=torch.float32, device=device)
            self.vs = torch.zeros(slots, n_kv_head, dtype=torch.float32, device=device)
            self.kb = torch.zeros(slots, n_kv_head, dtype=torch.float32, device=device) if affine else None
            self.vb = torch.zeros(slots, n_kv_head, dtype=torch.float32, device=device) if affine else None
        else:
            self.k = torch.zeros(slots, kvd, dtype=torch.float32, device=device)
            self.v = torch.zeros(slots, kvd, dtype=torch.float32, device=device)

    def q8_args(self):
        return tuple(ptr(x) for x in (self.k, self.v, self.ks, self.vs, self.kb, self.vb))

    def _q8_addrs(self):
        return (addr(self.k), addr(self.v), addr(self.ks), addr(self.vs), addr(self.kb), addr(self.vb))

    def nbytes(self) -> int:
        n = self.k.numel() * self.k.element_size() * 2
        if self.quant:
            n += self.ks.numel() * 4 * (4 if self.affine else 2)
        return n


class Paging:
    """Logical position -> physical row through a block table (gpu.rs:381-539):
    row = table[t // block_size] * block_size + t % block_size."""

    def __init__(self, table, block_size: int = KV_BLOCK):
        self.table_dev = table  # int32 CUDA tensor [n_log] or [n_seq][n_log]
        self.block_size = block_size
        self.n_log = table.shape[-1]

    def phys_row(self, host_table, pos: int) -> int:
        return int(host_table[pos // self.block_size]) * self.block_size + pos % self.block_size


# ---------------------------------------------------------------- rope
def rope(h: Handle, qkv, pos: int, n_head, n_kv_head, head_dim, theta, stream=None):
    check(lib().mx230_rope(h._h, stream_ptr(stream), addr(qkv), pos, n_head, n_kv_head, head_dim, theta))


def rope_dyn(h: Handle, qkv, pos_ptr, n_head, n_kv_head, head_dim, theta, stream=None):
    check(lib().mx230_rope_dyn(h._h, stream_ptr(stream), addr(qkv), addr(pos_ptr), n_head, n_kv_head,
                               head_dim, theta))


def rope_batch(h: Handle, qkv, pos0, n_tok, n_head, n_kv_head, head_dim, stride, theta, stream=None):
    check(lib().mx230_rope_batch(h._h, stream_ptr(stream), addr(qkv), pos0, n_tok, n_head, n_kv_head,
                                 head_dim, stride, theta))


def rope_seqpos(h: Handle, qkv, pos, n_seq, n_head, n_kv_head, head_dim, stride, theta, stream=None):
    check(lib().mx230_rope_seqpos(h._h, stream_ptr(stream), addr(qkv), addr(pos), n_seq, n_head,
                                  n_kv_head, head_dim, stride, theta))


# ---------------------------------------------------------------- rotary positions beyond the reference's forms
_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_SCALINGS = {"linear": (1, ()), "ntk": (2, ()), "wavelength": (3, ("low", "high", "length")), "yarn": (4, ("slow", "fast", "length"))}


def on_device(h: Handle, what: str, t, dtype=None):
    """A CUDA tensor of the handle's device, and of `dtype`."""
    require(isinstance(t, torch.Tensor) and t.get_device() == h.device, lambda: f"{what}: not a tensor of device {h.device}")
    require(dtype is None or t.dtype == dtype, lambda: f"{what}: {t.dtype}, not {dtype}")


class Rotary:
    """The frequencies of `rotary`, made once: theta^(-2i / rot_dim) for pair i of the first `rot_dim` values of a head.
    `scaling`: None, or how they are stretched for contexts longer than the trained one, as a dict with "kind" and "factor":
    "linear", "ntk", "wavelength" (with "low", "high", "length") or "yarn" (with "slow", "fast", "length"); the formulas stand
    in include/mx230_attn.h at MX230_ROTARY_*.  `interleaved`: pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)."""

    def __init__(self, rot_dim: int, theta: float, scaling: dict | None = None, interleaved: bool = False, device="cuda"):
        kind, names = (0, ()) if scaling is None else _SCALINGS.get(scaling.get("kind"), (None, ()))
        require(kind is not None, f"Rotary: scaling {scaling!r}")
        given = {} if scaling is None else {k: v for k, v in scaling.items() if k != "kind"}
        require(set(given) == ({"factor", *names} if kind else set()), f"Rotary: scaling {scaling!r} needs factor {' '.join(names)}")
        low, high, length = [given[n] for n in names] or (0.0, 0.0, 0)
        require_int32("Rotary", rot_dim, length)
        table, factor = (C.c_uint64 * max(1, rot_dim // 2))(), C.c_float()
        check(lib().mx230_rotary_table(table, C.byref(factor), rot_dim, theta, kind, given.get("factor", 1.0), low, high, length))
        self.rot_dim, self.interleaved, self.factor = rot_dim, int(interleaved), factor.value
        # (torch has no arithmetic on unsigned 64-bit words; only the bits matter)
        self.turns = torch.frombuffer(table, dtype=torch.int64).to(device)
        self._addr, self._device = self.turns.data_ptr(), self.turns.get_device()


def rotary(h: Handle, out, x, pos, plan: Rotary, inverse=False, stream=None):
    """Rotates the first plan.rot_dim values of every head of x [n_rows][n_head][head_dim] (fp32, fp16 or bf16; any strides between
    rows and heads) into `out` of the same shape, which may be x.  `pos`: an int32 tensor [n_rows], or the first row's position.
    `inverse` turns back; it takes the gradient of `out` to that of x."""
    shape, dtype, dev = x.shape, x.dtype, h.device
    require(len(shape) == 3 and out.shape == shape, lambda: f"rotary: x {tuple(x.shape)}, out {tuple(out.shape)}")
    require(dtype in _DTYPES and out.dtype == dtype, lambda: f"rotary: x {x.dtype}, out {out.dtype}")
    require(x.get_device() == dev and out.get_device() == dev and plan._device == dev, lambda: f"rotary: x, out or plan not on device {dev}")
    n, heads, dim = shape
    (xr, xh, xd), (outr, outh, outd) = x.stride(), out.stride()
    require(dim == 1 or (xd == 1 and outd == 1), "rotary: the values of a head must be contiguous")
    at, first = None, pos
    if isinstance(pos, torch.Tensor):
        on_device(h, "rotary: pos", pos, torch.int32)
        require(pos.shape == (n,) and (n < 2 or pos.stride(0) == 1), lambda: f"rotary: positions {tuple(pos.shape)} for {n} rows")
        at, first = pos.data_ptr(), 0
    require_int32("rotary", n, heads, dim, first)
    check(lib().mx230_rotary(h._h, raw_stream(stream, dev), out.data_ptr(), x.data_ptr(), _DTYPES[dtype], at, first, plan._addr, plan.factor,
                             n, heads, dim, plan.rot_dim, plan.interleaved, inverse, xr, xh, outr, outh))


# ---------------------------------------------------------------- fp32 KV write
def copy_kv(h: Handle, c: KvCache, qkv, pos: int, q_dim, kv_dim, stream=None):
    check(lib().mx230_copy_kv(h._h, stream_ptr(stream), addr(c.k), addr(c.v), addr(qkv), pos, q_dim, kv_dim))


def copy_kv_dyn(h: Handle, c: KvCache, qkv, pos_ptr, q_dim, kv_dim, stream=None):
    check(lib().mx230_copy_kv_dyn(h._h, stream_ptr(stream), addr(c.k), addr(c.v), addr(qkv),
                                  addr(pos_ptr), q_dim, kv_dim))


def copy_kv_paged_dyn(h: Handle, c: KvCache, qkv, pos_ptr, q_dim, kv_dim, pg: Paging, stream=None):
    check(lib().mx230_copy_kv_paged_dyn(h._h, stream_ptr(stream), addr(c.k), addr(c.v), addr(qkv),
                                        addr(pos_ptr), q_dim, kv_dim, addr(pg.table_dev), pg.block_size))


def copy_kv_batch(h: Handle, c: KvCache, qkv, pos0, n_tok, q_dim, kv_dim, stride, pg: Paging | None = None,
                  stream=None):
    if pg is None:
        check(lib().mx230_copy_kv_batch(h._h, stream_ptr(stream), addr(c.k), addr(c.v), addr(qkv), pos0,
                                        n_tok, q_dim, kv_dim, stride))
    else:
        check(lib().mx230_copy_kv_batch_paged(h._h, stream_ptr(stream), addr(c.k), addr(c.v), addr(qkv),
                                              pos0, n_tok, q_dim, kv_dim, stride, addr(pg.table_dev),
                                              pg.block_size))


def copy_kv_seqpos(h: Handle, c: KvCache, qkv, pos, n_seq, q_dim, kv_dim, qkv_stride, pg: Paging,
                   stream=None):
    check(lib().mx230_copy_kv_seqpos(h._h, stream_ptr(stream), addr(c.k), addr(c.v), addr(qkv), addr(pos),
                                     n_seq, q_dim, kv_dim, qkv_stride, addr(pg.table_dev),
                                     pg.block_size, pg.n_log))


# ---------------------------------------------------------------- int8 quantize-on-write
def quantize_kv(h: Handle, c: KvCache, qkv, pos: int, q_dim, n_kv_head, head_dim, stream=None):
    check(lib().mx230_quantize_kv(h._h, stream_ptr(stream), *c._q8_addrs(), addr(qkv), pos, q_dim,
                                  n_kv_head, head_dim))


def quantize_kv_dyn(h: Handle, c: KvCache, qkv, pos_ptr, q_dim, n_kv_head, head_dim, stream=None):
    check(lib().mx230_quantize_kv_dyn(h._h, stream_ptr(stream), *c._q8_addrs(), addr(qkv), addr(pos_ptr),
                                      q_dim, n_kv_head, head_dim))


def quantize_kv_paged_dyn(h: Handle, c: KvCache, qkv, pos_ptr, q_dim, n_kv_head, head_dim, pg: Paging,
                          stream=None):
    check(lib().mx230_quantize_kv_paged_dyn(h._h, stream_ptr(stream), *c._q8_addrs(), addr(qkv),
                                            addr(pos_ptr), q_dim, n_kv_head, head_dim,
                                            addr(pg.table_dev), pg.block_size))


def quantize_kv_batch(h: Handle, c: KvCache, qkv, pos0, n_tok, q_dim, n_kv_head, head_dim, stride,
                      pg: Paging | None = None, stream=None):
    if pg is None:
        check(lib().mx230_quantize_kv_batch(h._h, stream_ptr(stream), *c._q8_addrs(), addr(qkv), pos0,
                                            n_tok, q_dim, n_kv_head, head_dim, stride))
    else:
        check(lib().mx230_quantize_kv_batch_paged(h._h, stream_ptr(stream), *c._q8_addrs(), addr(qkv),
                                                  pos0, n_tok, q_dim, n_kv_head, head_dim, stride,
                                                  addr(pg.table_dev), pg.block_size))


def quantize_kv_seqpos(h: Handle, c: KvCache, qkv, pos, n_seq, q_dim, n_kv_head, head_dim, qkv_stride,
                       pg: Paging, stream=None):
    check(lib().mx230_quantize_kv_seqpos(h._h, stream_ptr(stream), *c._q8_addrs(), addr(qkv), addr(pos),
                                         n_seq, q_dim, n_kv_head, head_dim, qkv_stride,
                                         addr(pg.table_dev), pg.block_size, pg.n_log))


# ---------------------------------------------------------------- decode attention
def attn_decode(h: Handle, out, qkv, c: KvCache, t_cur: int, n_head, n_kv_head, head_dim,
                pg: Paging | None = None, stream=None):
    """attn_decode / attn_decode_paged / attn_decode_q8 / attn_decode_q8_paged, chosen by
    (cache format, paging) as gpu.rs:2607-2670."""
    s = stream_ptr(stream)
    L = lib()
    if c.quant:
        if pg is None:
            check(L.mx230_attn_decode_q8(h._h, s, addr(out), addr(qkv), *c._q8_addrs(), t_cur, n_head,
                                         n_kv_head, head_dim))
        else:
            check(L.mx230_attn_decode_q8_paged(h._h, s, addr(out), addr(qkv), *c._q8_addrs(), t_cur, n_head,
                                               n_kv_head, head_dim, addr(pg.table_dev), pg.block_size))
    else:
        if pg is None:
            check(L.mx230_attn_decode(h._h, s, addr(out), addr(qkv), addr(c.k), addr(c.v), t_cur, n_head,
                                      n_kv_head, head_dim))
        else:
            check(L.mx230_attn_decode_paged(h._h, s, addr(out), addr(qkv), addr(c.k), addr(c.v), t_cur,
                                            n_head, n_kv_head, head_dim, addr(pg.table_dev),
                                            pg.block_size))


def attn_decode_dyn(h: Handle, out, qkv, c: KvCache, pos_ptr, n_head, n_kv_head, head_dim,
                    pg: Paging | None = None, stream=None):
    """The `_dyn` forms of gpu.rs:2808-2918: position read from device memory."""
    s = stream_ptr(stream)
    L = lib()
    if c.quant:
        if pg is None:
            check(L.mx230_attn_decode_q8_dyn(h._h, s, addr(out), addr(qkv), *c._q8_addrs(), addr(pos_ptr),
                                             n_head, n_kv_head, head_dim))
        else:
            check(L.mx230_attn_decode_q8_paged_dyn(h._h, s, addr(out), addr(qkv), *c._q8_addrs(),
                                                   addr(pos_ptr), n_head, n_kv_head, head_dim,
                                                   addr(pg.table_dev), pg.block_size))
    else:
        if pg is None:
            check(L.mx230_attn_decode_dyn(h._h, s, addr(out), addr(qkv), addr(c.k), addr(c.v), addr(pos_ptr),
                                          n_head, n_kv_head, head_dim))
        else:
            check(L.mx230_attn_decode_paged_dyn(h._h, s, addr(out), addr(qkv), addr(c.k), addr(c.v),
                                                addr(pos_ptr), n_head, n_kv_head, head_dim,
                                                addr(pg.table_dev), pg.block_size))


def attn_decode_batched(h: Handle, out, qkv, c: KvCache, pos, n_seq, n_head, n_kv_head, head_dim,
                        pg: Paging, qkv_stride, out_stride, stream=None):
    """attn_decode_batched / attn_decode_q8_batched, gpu.rs:3530-3628."""
    s = stream_ptr(stream)
    if c.quant:
        check(lib().mx230_attn_decode_q8_batched(h._h, s, addr(out), addr(qkv), *c._q8_addrs(), addr(pos),
                                                 n_seq, n_head, n_kv_head, head_dim, addr(pg.table_dev),
                                                 pg.block_size, pg.n_log, qkv_stride, out_stride))
    else:
        check(lib().mx230_attn_decode_batched(h._h, s, addr(out), addr(qkv), addr(c.k), addr(c.v), addr(pos),
                                              n_seq, n_head, n_kv_head, head_dim, addr(pg.table_dev),
                                              pg.block_size, pg.n_log, qkv_stride, out_stride))


def _cache_args(c: KvCache):
    if c.quant:
        return (None, None) + c._q8_addrs()
    return (addr(c.k), addr(c.v), None, None, None, None, None, None)


def _table_args(pg: Paging | None):
    return (None, 0) if pg is None else (addr(pg.table_dev), pg.block_size)


def attn_decode_slab(h: Handle, out, qkv, c: KvCache, pos, n_seq, n_head, n_kv_head, head_dim,
                     seq_rows, qkv_stride, out_stride, stream=None):
    """Batched decode over contiguous per-sequence cache slabs of `seq_rows` rows."""
    check(lib().mx230_attn_decode_slab(h._h, stream_ptr(stream), addr(out), addr(qkv), *_cache_args(c),
                                       addr(pos), n_seq, n_head, n_kv_head, head_dim, seq_rows,
                                       qkv_stride, out_stride))


def attn_decode_partial(h: Handle, part_m, part_l, part_acc, qkv, c: KvCache, t0, t1, n_seq, n_head,
                        n_kv_head, head_dim, seq_rows, qkv_stride, stream=None):
    """Unnormalised (m, l, acc) of keys [t0, t1) per (sequence, query head)."""
    check(lib().mx230_attn_decode_partial(h._h, stream_ptr(stream), addr(part_m), addr(part_l),
                                          addr(part_acc), addr(qkv), *_cache_args(c), t0, t1, n_seq,
                                          n_head, n_kv_head, head_dim, seq_rows, qkv_stride))


def attn_decode_partial_push(h: Handle, comm, qkv, c: KvCache, t0, t1, n_seq, n_head, n_kv_head, head_dim, seq_rows,
                             qkv_stride, stream=None):
    """attn_decode_partial whose finishing CTAs store the triples into every rank's split-KV exchange region
    (`comm`: the mx230_splitkv_comm of `multi_gpu.PeerExchange`)."""
    check(lib().mx230_attn_decode_partial_push(h._h, stream_ptr(stream), comm, addr(qkv), *_cache_args(c), t0, t1,
                                               n_seq, n_head, n_kv_head, head_dim, seq_rows, qkv_stride))


def attn_decode_splitkv(h: Handle, comm, out, qkv, c: KvCache, t0, t1, n_seq, n_head, n_kv_head, head_dim, seq_rows,
                        qkv_stride, stream=None):
    """A whole split-KV step in one kernel: partial attention over keys [t0, t1), stores to every other rank's
    exchange region, wait for their triples, merged rows to out[n_seq * n_head][64]."""
    check(lib().mx230_attn_decode_splitkv(h._h, stream_ptr(stream), comm, addr(out), addr(qkv), *_cache_args(c), t0, t1,
                                          n_seq, n_head, n_kv_head, head_dim, seq_rows, qkv_stride))


def merge_partials(h: Handle, out, m, l, acc, parts, rows, head_dim=64, stream=None):
    check(lib().mx230_merge_partials(h._h, stream_ptr(stream), addr(out), addr(m), addr(l), addr(acc),
                                     parts, rows, head_dim))


def merge_partials_packed(h: Handle, out, gathered, parts, rows, head_dim=64, stream=None):
    """Merge straight from the all-gathered buffer [parts][m | l | acc] (rows even)."""
    check(lib().mx230_merge_partials_packed(h._h, stream_ptr(stream), addr(out), addr(gathered), parts, rows, head_dim))


# ---------------------------------------------------------------- the step
def decode_step(h: Handle, out, qkv, c: KvCache, pos: int, n_head, n_kv_head, head_dim, theta,
                pg: Paging | None = None, host_table=None, use_rope=True, stream=None):
    """One token of one sequence, as forward_layers does per layer (gpu.rs:2570-2672):
    RoPE, KV write at the host-resolved physical row, then attention over 0..=pos -- one launch."""
    phys = pos if pg is None else pg.phys_row(host_table, pos)
    check(lib().mx230_decode_step(h._h, stream_ptr(stream), addr(out), addr(qkv), *_cache_args(c), pos, None, phys, n_head,
                                  n_kv_head, head_dim, int(use_rope), theta, *_table_args(pg)))


def decode_step_dyn(h: Handle, out, qkv, c: KvCache, pos_ptr, n_head, n_kv_head, head_dim, theta,
                    pg: Paging | None = None, use_rope=True, stream=None):
    """The graph-capturable step of forward_body_dyn (gpu.rs:2808-2918)."""
    check(lib().mx230_decode_step(h._h, stream_ptr(stream), addr(out), addr(qkv), *_cache_args(c), -1, addr(pos_ptr), 0, n_head,
                                  n_kv_head, head_dim, int(use_rope), theta, *_table_args(pg)))


def batched_step(h: Handle, out, qkv, c: KvCache, pos, n_seq, n_head, n_kv_head, head_dim, theta,
                 pg: Paging, qkv_stride, out_stride, use_rope=True, stream=None):
    """One token for each of n_seq sequences, as forward_batched (gpu.rs:3530-3628) -- two launches, so that rows of the same
    sequence see one another."""
    check(lib().mx230_batched_step(h._h, stream_ptr(stream), addr(out), addr(qkv), *_cache_args(c), addr(pos), n_seq, n_head,
                                   n_kv_head, head_dim, int(use_rope), theta, addr(pg.table_dev), pg.block_size, pg.n_log,
                                   qkv_stride, out_stride))


# ---------------------------------------------------------------- prefill attention
def prefill_workspace_bytes(n_tok, n_keys, n_head, n_kv_head) -> int:
    return int(lib().mx230_prefill_workspace_bytes(n_tok, n_keys, n_head, n_kv_head))


def attn_prefill(h: Handle, out, qkv, c: KvCache, pos0, n_tok, n_head, n_kv_head, qkv_stride, out_stride,
                 pg: Paging | None = None, stream=None):
    """attn_prefill / _paged / _q8 / _q8_paged chosen by (cache format, paging) as
    batch_body_from does (gpu.rs:3269-3345).  The cache must already hold the new rows."""
    s = stream_ptr(stream)
    L = lib()
    if c.quant:
        if pg is None:
            check(L.mx230_attn_prefill_q8(h._h, s, addr(out), addr(qkv), *c._q8_addrs(), pos0, n_tok, n_head,
                                          n_kv_head, qkv_stride, out_stride))
        else:
            check(L.mx230_attn_prefill_q8_paged(h._h, s, addr(out), addr(qkv), *c._q8_addrs(), pos0, n_tok, n_head,
                                                n_kv_head, qkv_stride, out_stride, addr(pg.table_dev),
                                                pg.block_size))
    else:
        if pg is None:
            check(L.mx230_attn_prefill(h._h, s, addr(out), addr(qkv), addr(c.k), addr(c.v), pos0, n_tok, n_head,
                                       n_kv_head, qkv_stride, out_stride))
        else:
            check(L.mx230_attn_prefill_paged(h._h, s, addr(out), addr(qkv), addr(c.k), addr(c.v), pos0, n_tok,
                                             n_head, n_kv_head, qkv_stride, out_stride, addr(pg.table_dev),
                                             pg.block_size))


def prefill_step(h: Handle, out, qkv, c: KvCache, pos0, n_tok, n_head, n_kv_head, head_dim, theta,
                 qkv_stride, out_stride, pg: Paging | None = None, use_rope=True, stream=None):
    """The prefill attention step of batch_body_from (gpu.rs:3204-3347): RoPE on the n_tok rows,
    KV write of all of them, then causal attention over the cache -- two launches."""
    if head_dim != 64:   # the fused entry point knows 64 only; the separate ones decide what they take
        q_dim, kv_dim = n_head * head_dim, n_kv_head * head_dim
        if use_rope:
            rope_batch(h, qkv, pos0, n_tok, n_head, n_kv_head, head_dim, qkv_stride, theta, stream)
        if c.quant:
            quantize_kv_batch(h, c, qkv, pos0, n_tok, q_dim, n_kv_head, head_dim, qkv_stride, pg, stream)
        else:
            copy_kv_batch(h, c, qkv, pos0, n_tok, q_dim, kv_dim, qkv_stride, pg, stream)
        return attn_prefill(h, out, qkv, c, pos0, n_tok, n_head, n_kv_head, qkv_stride, out_stride, pg, stream)
    check(lib().mx230_prefill_step(h._h, stream_ptr(stream), addr(out), addr(qkv), *_cache_args(c), pos0, n_tok, n_head,
                                   n_kv_head, head_dim, int(use_rope), theta, qkv_stride, out_stride, *_table_args(pg)))


def attn_decode_q8_noalloc(out, qkv, c: KvCache, t_cur: int, n_head, n_kv_head, head_dim, stream=None):
    """Handle-free int8-cache decode of one sequence whose split-KV scratch is a fixed array inside
    the library: for hosts that may not call cudaMalloc (all HBM already owned by their KV pool, or
    only allowed to enqueue on a given stream).  Current device; see include/mx230_attn.h."""
    check(lib().mx230_attn_decode_q8_noalloc(stream_ptr(stream), addr(out), addr(qkv), *c._q8_addrs(), t_cur,
                                             n_head, n_kv_head, head_dim))


# ---------------------------------------------------------------- projections either side of attention
def gemv(h: Handle, y, x, w, b=None, accum=False, stream=None):
    """gemv / gemv_half (llm.cu:144-177; gpu.rs:1158-1198): y (+)= x W + b, W [n_in][n_out] fp32 or fp16."""
    n_in, n_out = w.shape
    check(lib().mx230_gemv(h._h, stream_ptr(stream), addr(y), addr(x), addr(w), int(w.dtype == torch.float16),
                           addr(b), n_in, n_out, int(accum)))


def gemm(h: Handle, c, a, w, b=None, stream=None):
    """gemm (gpu.rs:1291-1420) for the prefill-side projections: c [m][n] = a [m][k] . w [k][n] + b, `w` fp32 or
    fp16.  Grows the handle's workspace when it is too small for the staged operands."""
    m, k = a.shape
    n = w.shape[1]
    fp16 = 1 if w.dtype == torch.float16 else 0
    h.reserve(lib().mx230_gemm_workspace_bytes(m, n, k, fp16))
    check(lib().mx230_gemm(h._h, stream_ptr(stream), addr(c), addr(a), addr(w), fp16, addr(b), m, n, k))


def prefill_layer_attention(h: Handle, y, x, w_qkv, b_qkv, w_proj, b_proj, qkv, attn, c: KvCache, pos0, n_tok, n_head,
                            n_kv_head, head_dim, theta, pg: Paging | None = None, use_rope=True, stream=None):
    """The attention half of one layer for a prefill chunk, as batch_body_from runs it (gpu.rs:3187-3365):
    qkv = x W_qkv + b (gemm), RoPE, KV write, causal attention over the cache, y = attn W_proj + b (gemm).
    `qkv` [n_tok][q_dim + 2 kv_dim] and `attn` [n_tok][q_dim] are the caller's scratch rows (the reference's batch_qkv
    and batch_attn); the residual add that follows stays with the caller, as in the reference."""
    q_dim = n_head * head_dim
    gemm(h, qkv, x, w_qkv, b_qkv, stream)
    if w_proj.dtype == torch.float16 and head_dim == 64 and tuple(attn.shape) == (n_tok, q_dim):
        # attention leaves its rows in fp16 for the projection: one staging launch less
        check(lib().mx230_prefill_step_proj(h._h, stream_ptr(stream), addr(y), addr(w_proj), addr(b_proj), w_proj.shape[1],
                                            addr(attn), addr(qkv), *_cache_args(c), pos0, n_tok, n_head, n_kv_head, head_dim,
                                            int(use_rope), theta, qkv.shape[1], q_dim, *_table_args(pg)))
        return
    prefill_step(h, attn, qkv, c, pos0, n_tok, n_head, n_kv_head, head_dim, theta, qkv.shape[1], q_dim, pg, use_rope, stream)
    gemm(h, y, attn, w_proj, b_proj, stream)


def gemv_int8(h: Handle, y, x, w_packed, scales, b=None, accum=False, act_group=8, stream=None):
    """gemv_int8 (llm.cu:226-316): `w_packed` int32 [n_in / 4][n_out], four consecutive input rows per word."""
    n_in, n_out = w_packed.shape[0] * 4, w_packed.shape[1]
    check(lib().mx230_gemv_int8(h._h, stream_ptr(stream), addr(y), addr(x), addr(w_packed), addr(scales), addr(b),
                                n_in, n_out, int(accum), act_group))


class Int4Weights:
    """A matrix [n_in][n_out] of 4-bit weights in the layout of `gemv_int4` (made by `pack_int4`)."""

    def __init__(self, packed, n_in: int, n_out: int, group: int):
        self.packed, self.n_in, self.n_out, self.group = packed, n_in, n_out, group
        self._addr, self._device = packed.data_ptr(), packed.get_device()

    def nbytes(self) -> int:
        return self.packed.numel()


def pack_int4(h: Handle, codes, scales, zeros=None, group: int | None = None, stream=None) -> Int4Weights:
    """Lays out weights scale * (code - zero) once for `gemv_int4`: `codes` uint8 [n_in][n_out] (low four bits), `scales` fp16 and
    `zeros` uint8 [groups][n_out] (None: 8).  A group is 32 inputs or a multiple of 64; `group` may be left out where the
    number of groups determines it among the powers of two.  Allocates the result, on `stream`: not for the step path."""
    require(codes.dim() == 2 and scales.dim() == 2 and scales.shape[1] == codes.shape[1], "pack_int4: codes [n_in][n_out], scales [groups][n_out]")
    n_in, n_out = codes.shape
    groups = scales.shape[0]
    if group is None:
        fits = [g for g in (32, 64, 128, 256, 512, 1024) if -(-n_in // g) == groups]
        require(len(fits) == 1, lambda: f"pack_int4: {groups} groups of {n_in} inputs: give the group")
        group = fits[0]
    require(group > 0 and -(-n_in // group) == groups, lambda: f"pack_int4: {groups} groups of {group} for {n_in} inputs")
    require_int32("pack_int4", n_in, n_out, group)
    on_device(h, "pack_int4: codes", codes, torch.uint8), on_device(h, "pack_int4: scales", scales, torch.float16)
    require(codes.is_contiguous() and scales.is_contiguous(), "pack_int4: codes and scales must be contiguous")
    if zeros is not None:
        on_device(h, "pack_int4: zeros", zeros, torch.uint8)
        require(zeros.shape == scales.shape and zeros.is_contiguous(), "pack_int4: zeros must be contiguous, of the scales' shape")
    on = raw_stream(stream, h.device)
    # (on the stream that writes it: memory that was freed on another one may still be in use there)
    with torch.cuda.stream(None if stream is None else torch.cuda.ExternalStream(on, device=codes.device)):
        packed = torch.empty(lib().mx230_int4_bytes(n_in, n_out, group), dtype=torch.uint8, device=codes.device)
    check(lib().mx230_pack_int4(h._h, on, packed.data_ptr(), addr(codes), addr(scales), addr(zeros), n_in, n_out, group))
    return Int4Weights(packed, n_in, n_out, group)


def gemv_int4(h: Handle, y, x, w: Int4Weights, b=None, add=None, stream=None):
    """y = x W + b + add over 4-bit weights: x [n_in] or [n_rows][n_in], y and add (which may be y: the residual row) with n_out.
    A row's bits do not depend on the rows beside it."""
    xs, ys, dev, f32 = x.shape, y.shape, h.device, torch.float32
    rows, n_out = xs[:-1], w.n_out
    require(0 < len(xs) < 3 and xs[-1] == w.n_in and ys == (*rows, n_out), lambda: f"gemv_int4: x {tuple(xs)}, y {tuple(ys)}, weights [{w.n_in}][{n_out}]")
    require(x.dtype == f32 and y.dtype == f32 and x.get_device() == dev and y.get_device() == dev and w._device == dev,
            lambda: f"gemv_int4: x {x.dtype}, y {y.dtype} must be fp32, they and the weights on device {dev}")
    xd, yd = x.stride(), y.stride()
    require((w.n_in == 1 or xd[-1] == 1) and (n_out == 1 or yd[-1] == 1), "gemv_int4: the values of a row must be contiguous")
    bias = plus = None
    ad = (0,)
    if b is not None:
        on_device(h, "gemv_int4: bias", b, f32)
        require(b.shape == (n_out,) and (n_out == 1 or b.stride(0) == 1), "gemv_int4: bias must be [n_out], contiguous")
        bias = b.data_ptr()
    if add is not None:
        on_device(h, "gemv_int4: add", add, f32)
        ad, plus = add.stride(), add.data_ptr()
        require(add.shape == ys and (n_out == 1 or ad[-1] == 1), "gemv_int4: add must have the shape of y, its rows contiguous")
    n = rows[0] if rows else 1
    require_int32("gemv_int4", n)
    check(lib().mx230_gemv_int4(h._h, raw_stream(stream, dev), y.data_ptr(), x.data_ptr(), w._addr, bias, plus, n, w.n_in,
                                n_out, w.group, xd[0], yd[0], ad[0]))


def qkv_rope_kvwrite(h: Handle, qkv, x, w, b, pos, c: KvCache, n_head, n_kv_head, theta, pg: Paging | None = None,
                     stream=None, w_scales=None, act_group=8):
    """The qkv step of one decode token in one launch (gemv + rope + KV write of gpu.rs:2558-2646):
    `pos` is a host int or an int32 device tensor (the graph-captured form)."""
    int8 = w.dtype == torch.int32   # packed int8 weights
    n_in = w.shape[0] * (4 if int8 else 1)
    kind = 2 if int8 else int(w.dtype == torch.float16)
    dyn = not isinstance(pos, int)
    caches = (None, None, *c._q8_addrs()) if c.quant else (addr(c.k), addr(c.v), None, None, None, None, None, None)
    check(lib().mx230_qkv_rope_kvwrite(h._h, stream_ptr(stream), addr(qkv), addr(x), addr(w),
                                       kind, addr(w_scales), act_group, addr(b), n_in, 0 if dyn else pos,
                                       addr(pos) if dyn else None, n_head, n_kv_head, 64, theta, *caches,
                                       addr(pg.table_dev) if pg else None, pg.block_size if pg else 0))
