"""Continuous batching over the batched decode attention step.

Mirror of `Engine::run_continuous` (03-llm-engine/src/gpu.rs:3800-3915) on the C ABI's
`mx230_sched_*` state machine.  The reference scheduler is welded to its model; here the model is
whatever the caller passes in: an object with

    prefill(request_index, prompt_tokens, table: np.ndarray[int32, n_log]) -> int   # first generated token
    decode_batched(cur: np.ndarray[uint32, n], pos: np.ndarray[int32, n],
                   tables: np.ndarray[int32, n x n_log]) -> sequence of n next tokens

whose attention runs through `llm_attention.prefill_step` / `batched_step` with those block tables.  With a `Sampler` both
return logits instead (device tensors, [vocab] and [n][vocab]), and the tokens are drawn here by each request's settings.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field

import numpy as np

from ._lib import ERR_INVALID_ARG, Mx230Error, check, lib, require, require_int32
from .common import Handle, raw_stream
from .paging import KvPool

torch = None   # brought in by the first draw: the scheduler runs on hosts without it


def _need_torch() -> None:
    global torch, _DTYPES, on_device
    import torch
    from .llm_attention import _DTYPES, on_device


@dataclass
class Request:
    """Request, gpu.rs:356-359, and how its tokens are drawn where a `Sampler` draws them (the settings of `sample`;
    temperature 0: the most likely one)."""
    prompt: list
    max_new: int
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


@dataclass
class ServeStats:
    """ServeStats, gpu.rs:366-370."""
    decode_steps: int = 0
    seq_decodes: int = 0
    admitted: int = 0
    ended: list = field(default_factory=list)   # requests that ended before their last token (see run_continuous)


class Scheduler:
    def __init__(self, pool: KvPool, n_ctx: int, max_batch: int, requests: list[Request]):
        self._s = C.c_void_p()
        self.pool, self.max_batch, self.n_req = pool, max_batch, len(requests)
        pl = np.ascontiguousarray([len(r.prompt) for r in requests], np.int32)
        mn = np.ascontiguousarray([r.max_new for r in requests], np.int32)
        check(lib().mx230_sched_create(C.byref(self._s), pool._p, n_ctx, max_batch,
                                       pl.ctypes.data_as(C.c_void_p), mn.ctypes.data_as(C.c_void_p), len(requests)))
        self.n_log = lib().mx230_sched_n_log(self._s)

    def close(self):
        """Requests that are still being served end here; their blocks go back to the pool."""
        if self._s:
            if self.pool._p:
                lib().mx230_sched_end(self._s, -1)
            lib().mx230_sched_destroy(self._s)
            self._s = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def admit(self):
        """(request index, block table) of the next admission, or None."""
        r = C.c_int(-1)
        table = np.empty(self.n_log, np.int32)
        check(lib().mx230_sched_admit(self._s, C.byref(r), table.ctypes.data_as(C.c_void_p)))
        return None if r.value < 0 else (r.value, table)

    def admitted(self, request: int, first_token: int) -> None:
        check(lib().mx230_sched_admitted(self._s, request, int(first_token)))

    def batch(self):
        """(cur, pos, tables) of the active set; cur is empty when everything has been served."""
        n = C.c_int(0)
        cur = np.empty(self.max_batch, np.uint32)
        pos = np.empty(self.max_batch, np.int32)
        tables = np.empty((self.max_batch, self.n_log), np.int32)
        check(lib().mx230_sched_batch(self._s, C.byref(n), cur.ctypes.data_as(C.c_void_p),
                                      pos.ctypes.data_as(C.c_void_p), tables.ctypes.data_as(C.c_void_p)))
        return cur[:n.value], pos[:n.value], tables[:n.value]

    def requests(self) -> list[int]:
        """The request of each row of the batch."""
        out = np.empty(self.max_batch, np.int32)
        return out[:lib().mx230_sched_requests(self._s, out.ctypes.data_as(C.c_void_p), out.size)].tolist()

    def step_done(self, next_tokens) -> None:
        nt = np.ascontiguousarray(next_tokens, np.uint32)
        check(lib().mx230_sched_step_done(self._s, nt.ctypes.data_as(C.c_void_p)))

    def end(self, request: int) -> None:
        """Ends a request that awaits its first token or is being decoded (within a step: with `step_done`, which does not take its token)."""
        check(lib().mx230_sched_end(self._s, request))

    def result(self, request: int) -> list[int]:
        n = C.c_int(0)
        check(lib().mx230_sched_result(self._s, request, None, 0, C.byref(n)))
        out = np.empty(max(1, n.value), np.uint32)
        check(lib().mx230_sched_result(self._s, request, out.ctypes.data_as(C.c_void_p), out.size, C.byref(n)))
        return out[:n.value].tolist()

    def stats(self) -> ServeStats:
        f = lib().mx230_sched_stat
        return ServeStats(f(self._s, 0), f(self._s, 1), f(self._s, 2))


def sample(h: Handle, token, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, prob=None, stream=None):
    """The next token of each row of `logits` [n][vocab] (fp32, fp16 or bf16; the values of a row contiguous) into `token` int32 [n],
    from random numbers `u` fp32 [n] in [0, 1); its probability among what could be drawn into `prob` fp32 [n].  Each setting
    is a number or a tensor [n] (fp32, top_k int32).  include/mx230_attn.h has the definition at mx230_sample: of the entries in
    falling order the first top_k, of those the shortest prefix with top_p of their weight, cut at min_p times the largest
    weight; among what is kept, in the order of the vocabulary, the token is where the running weight passes u's share.  -1
    where a row is masked throughout."""
    if torch is None:
        _need_torch()
    dev, dtype = h.device, _DTYPES.get(logits.dtype)
    require(logits.dim() == 2 and dtype is not None, lambda: f"sample: logits {tuple(logits.shape)} of {logits.dtype}")
    (n, vocab), (row, one) = logits.shape, logits.stride()
    on_device(h, "sample: logits", logits)
    require(vocab < 2 or one == 1, "sample: the logits of a row must be contiguous")

    def vector(what, t, ty):
        on_device(h, what, t, ty)
        require(t.shape == (n,) and (n < 2 or t.stride(0) == 1), lambda: f"{what} {tuple(t.shape)} for {n} rows")
        return t.data_ptr()

    t, ts = (0.0, vector("sample: temperature", temperature, torch.float32)) if isinstance(temperature, torch.Tensor) else (temperature, None)
    k, ks = (0, vector("sample: top_k", top_k, torch.int32)) if isinstance(top_k, torch.Tensor) else (top_k, None)
    p, ps = (0.0, vector("sample: top_p", top_p, torch.float32)) if isinstance(top_p, torch.Tensor) else (top_p, None)
    m, ms = (0.0, vector("sample: min_p", min_p, torch.float32)) if isinstance(min_p, torch.Tensor) else (min_p, None)
    require_int32("sample", n, vocab, k)
    check(lib().mx230_sample(h._h, raw_stream(stream, dev), vector("sample: token", token, torch.int32),
                             None if prob is None else vector("sample: prob", prob, torch.float32), logits.data_ptr(), dtype, n, vocab, row,
                             vector("sample: u", u, torch.float32), t, ts, k, ks, p, ps, m, ms))


class MaskedLogits(Mx230Error):
    """Every logit of some rows is masked: `tokens` has -1 for those, and the tokens of the others."""

    def __init__(self, tokens, what: str):
        super().__init__(ERR_INVALID_ARG, what)
        self.tokens = tokens


class Sampler:
    """Draws the tokens of `run_continuous`.  The random number of a request's t-th token depends on (seed, request, t) alone, so a
    request's tokens do not depend on what is served beside it."""

    def __init__(self, h: Handle, seed: int = 0):
        require(0 <= seed < 1 << 128, f"Sampler: seed {seed} (0 to 2^128 - 1)")
        self.h, self.seed = h, seed

    def uniform(self, request: int, step: int) -> float:
        bits = np.random.Philox(key=self.seed, counter=[request, step, 0, 0]).random_raw()
        return (int(bits) >> 40) * 2.0 ** -24

    def draw(self, logits, rows) -> list[int]:
        """One token for each of `rows`, (request index, step, Request), from its row of `logits` [rows][vocab], or [vocab] for one.
        Raises `MaskedLogits` where a row has none."""
        if torch is None:
            _need_torch()
        if logits.dim() == 1:
            logits = logits[None]
        require(logits.dim() == 2 and logits.shape[0] == len(rows), lambda: f"logits {tuple(logits.shape)} for {len(rows)} sequences")
        dev = lambda a, t: torch.tensor(a, dtype=t, device=logits.device)  # noqa: E731
        token = torch.empty(len(rows), dtype=torch.int32, device=logits.device)
        sample(self.h, token, logits, dev([self.uniform(r, t) for r, t, _ in rows], torch.float32),
               dev([q.temperature for *_, q in rows], torch.float32), dev([q.top_k for *_, q in rows], torch.int32),
               dev([q.top_p for *_, q in rows], torch.float32), dev([q.min_p for *_, q in rows], torch.float32))
        out = token.tolist()
        if min(out, default=0) < 0:
            raise MaskedLogits(out, ", ".join(f"request {r}: every logit of token {t} is masked" for (r, t, _), tok in zip(rows, out) if tok < 0))
        return out


def run_continuous(model, pool: KvPool, n_ctx: int, requests: list[Request], max_batch: int, trace=None,
                   sampler: Sampler | None = None):
    """Serves `requests` keeping up to `max_batch` sequences decoding together; returns each
    request's generated tokens (request order) and the occupancy statistics.  `trace`, when given,
    receives one tuple per event (for tests).  `sampler`: the model returns logits, and it draws the tokens; a request whose logits are
    masked throughout ends with the tokens that it has, is named in the statistics, and the others go on."""
    s = Scheduler(pool, n_ctx, max_batch, requests)
    ended = []   # requests that ended early

    def draw(logits, rows):
        try:
            return sampler.draw(logits, rows)
        except MaskedLogits as e:
            for (r, t, _), tok in zip(rows, e.tokens):
                if tok < 0:
                    s.end(r)
                    ended.append(r)
                    if trace is not None:
                        trace.append(("end", r, t))
            return [max(tok, 0) for tok in e.tokens]

    try:
        while True:
            while (adm := s.admit()) is not None:
                r, table = adm
                first = model.prefill(r, requests[r].prompt, table)
                if sampler is not None:
                    first = draw(first, [(r, 0, requests[r])])[0]
                    if r in ended:
                        continue
                if trace is not None:
                    trace.append(("admit", r, table.tolist(), int(first)))
                s.admitted(r, first)
            cur, pos, tables = s.batch()
            if cur.size == 0:
                break
            nxt = model.decode_batched(cur.copy(), pos.copy(), tables.copy())
            if sampler is not None:
                nxt = draw(nxt, [(r, int(p) - len(requests[r].prompt) + 1, requests[r]) for r, p in zip(s.requests(), pos)])
            if trace is not None:
                trace.append(("step", cur.tolist(), pos.tolist(), tables.tolist(), [int(x) for x in nxt]))
            s.step_done(nxt)
        stats = s.stats()
        stats.ended = sorted(ended)
        return [s.result(r) for r in range(len(requests))], stats
    finally:
        s.close()
