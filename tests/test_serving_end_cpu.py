"""Requests that end early, and serving that is left by an error: every block is back in the pool, and the others are served as before
(no GPU: a pure function in place of the model)."""
import gc
import os
import subprocess
import sys

import pytest
import torch

from mx230_b200 import serving
from mx230_b200._lib import Mx230Error
from mx230_b200.paging import KvPool
from mx230_b200.serving import MaskedLogits, Request, Sampler, Scheduler, run_continuous

BS, N_CTX = 16, 64


class Model:
    def prefill(self, r, prompt, table):
        return sum(prompt) * 31 % 1000

    def decode_batched(self, cur, pos, tables):
        return [(int(c) * 131 + int(p) * 17) % 1000 for c, p in zip(cur, pos)]


REQUESTS = [Request([1, 2, 3], 9), Request([4] * 20, 1), Request([5] * 10, 30), Request([6] * 33, 12), Request([7], 20)]


class Stop(Exception):
    pass


@pytest.mark.parametrize("where", ["prefill", "decode_batched"])
@pytest.mark.parametrize("calls", [0, 1, 3])
def test_an_error_of_the_model_gives_the_blocks_back(where, calls):
    pool, model, left = KvPool(30 * BS, BS), Model(), [calls]
    plain = getattr(model, where)

    def failing(*a):
        left[0] -= 1
        if left[0] < 0:
            raise Stop
        return plain(*a)

    setattr(model, where, failing)
    with pytest.raises(Stop):
        run_continuous(model, pool, N_CTX, REQUESTS, 3)
    assert pool.free_blocks == 30
    pool.audit()
    setattr(model, where, plain)
    out, _ = run_continuous(model, pool, N_CTX, REQUESTS, 3)
    assert [len(o) for o in out] == [r.max_new for r in REQUESTS] and pool.free_blocks == 30


def serve(pool, ends=()):
    """The loop of run_continuous, with requests ended at (request, tokens so far)."""
    s, m, ended = Scheduler(pool, N_CTX, 3, REQUESTS), Model(), set()
    while True:
        while (adm := s.admit()) is not None:
            r, table = adm
            if (r, 0) in ends:
                s.end(r)
                ended.add(r)
            else:
                s.admitted(r, m.prefill(r, REQUESTS[r].prompt, table))
        cur, pos, tables = s.batch()
        if not cur.size:
            break
        for r in range(len(REQUESTS)):
            if r not in ended and (r, len(s.result(r))) in ends:
                s.end(r)
                ended.add(r)
                with pytest.raises(Mx230Error):
                    s.end(r)   # in this step already
        s.step_done(m.decode_batched(cur, pos, tables))
    got = [s.result(r) for r in range(len(REQUESTS))]
    for r in (0, len(REQUESTS) - 1, len(REQUESTS)):
        with pytest.raises(Mx230Error):
            s.end(r)   # not being served (any more)
    s.close()
    return got


def test_requests_that_end_early():
    pool = KvPool(30 * BS, BS)
    want = serve(pool)
    for ends in [{(0, 1)}, {(2, 0)}, {(2, 29), (0, 4)}, {(1, 0), (3, 11), (4, 1)}, {(4, 19), (0, 8)}, {(0, 0), (1, 0), (2, 0), (3, 0), (4, 0)}]:
        got = serve(pool, ends)
        cut = dict(ends)
        assert got == [w[:cut.get(r, len(w))] for r, w in enumerate(want)], ends
        assert pool.free_blocks == 30
        pool.audit()


def test_a_scheduler_that_is_left_in_the_middle():
    for step in range(4):
        pool = KvPool(30 * BS, BS)
        s = Scheduler(pool, N_CTX, 3, REQUESTS)
        r, _ = s.admit()
        if step > 0:
            s.admitted(r, 7)
        if step > 1:
            s.batch()
        if step > 2:
            s.end(r)
        assert pool.free_blocks < 30
        s.close()
        assert pool.free_blocks == 30, step
        pool.audit()
    s = Scheduler(pool, N_CTX, 3, REQUESTS)
    s.admit()
    pool.close()   # the pool first: nothing is given back to it
    s.close()
    del s, pool
    gc.collect()


class Draws:
    """Tokens from (request, step) alone; none for the ones that are named."""

    def __init__(self, masked=()):
        self.masked = masked

    def draw(self, logits, rows):
        out = [-1 if (r, t) in self.masked else (r * 37 + t * 11) % 1000 for r, t, _ in rows]
        if min(out) < 0:
            raise MaskedLogits(out, "masked")
        return out


def test_masked_logits_end_their_request_alone():
    pool = KvPool(30 * BS, BS)
    want, st = run_continuous(Model(), pool, N_CTX, REQUESTS, 3, sampler=Draws())
    assert st.ended == [] and [len(w) for w in want] == [r.max_new for r in REQUESTS]
    for masked in [{(1, 0)}, {(0, 0), (2, 7)}, {(0, 4), (2, 4), (3, 3)}, {(4, 19)}, {(r, 0) for r in range(5)}]:
        trace = []
        got, st = run_continuous(Model(), pool, N_CTX, REQUESTS, 3, trace=trace, sampler=Draws(masked))
        cut = dict(masked)
        assert got == [w[:cut.get(r, len(w))] for r, w in enumerate(want)], masked
        assert st.ended == sorted(cut) and sorted(e[1:] for e in trace if e[0] == "end") == sorted(masked)
        assert pool.free_blocks == 30
        pool.audit()
    assert issubclass(MaskedLogits, Mx230Error)


def test_another_error_of_the_draw_gives_the_blocks_back():
    class Failing(Draws):
        def draw(self, logits, rows):
            if rows[0][1] == 3:
                raise Stop
            return super().draw(logits, rows)

    pool = KvPool(30 * BS, BS)
    with pytest.raises(Stop):
        run_continuous(Model(), pool, N_CTX, REQUESTS, 3, sampler=Failing())
    assert pool.free_blocks == 30


def test_the_draw_is_told_the_requests_by_the_scheduler(monkeypatch):
    """Not by their blocks: a table whose first block is another request's too changes nothing."""
    asked = []

    class Asking(Draws):
        def draw(self, logits, rows):
            asked.append([(r, t, q is REQUESTS[r]) for r, t, q in rows])
            return super().draw(logits, rows)

    want, _ = run_continuous(Model(), KvPool(30 * BS, BS), N_CTX, REQUESTS, 3, sampler=Asking())
    plain, batch, admit = asked.copy(), Scheduler.batch, Scheduler.admit
    asked.clear()

    def first_block(table):
        table[..., 0] = 5
        return table

    monkeypatch.setattr(Scheduler, "batch", lambda s: (lambda c, p, t: (c, p, first_block(t)))(*batch(s)))
    monkeypatch.setattr(Scheduler, "admit", lambda s: (lambda a: None if a is None else (a[0], first_block(a[1])))(admit(s)))
    got, _ = run_continuous(Model(), KvPool(30 * BS, BS), N_CTX, REQUESTS, 3, sampler=Asking())
    assert got == want and asked == plain and all(same for rows in asked for *_, same in rows)


@pytest.mark.parametrize("shape,n", [((8, 50), 4), ((4, 50), 8), ((100,), 2), ((50,), 0), ((2, 2, 25), 4), ((1, 1, 50), 1), ((), 1), ((3, 50), 1)])
def test_logits_of_another_number_of_rows(monkeypatch, shape, n):
    """As of a step that is padded to the largest batch: its rows are not regrouped."""
    from types import SimpleNamespace

    def drawn(*a, **k):
        raise AssertionError("drawn")

    monkeypatch.setattr(serving, "sample", drawn)
    sampler = Sampler(SimpleNamespace(device=0))
    with pytest.raises(Mx230Error) as e:
        sampler.draw(torch.zeros(shape), [(r, 0, REQUESTS[0]) for r in range(n)])
    assert not isinstance(e.value, MaskedLogits)
    for shape in ((50,), (1, 50)):
        with pytest.raises(AssertionError, match="drawn"):
            sampler.draw(torch.zeros(shape), [(0, 0, REQUESTS[0])])


WITHOUT_TORCH = """
import sys
sys.modules["torch"] = None
from mx230_b200.paging import KvPool
from mx230_b200.serving import Request, Sampler, Scheduler
s = Scheduler(KvPool(64), 64, 2, [Request([1, 2], 3)])
assert s.admit()[0] == 0
"""


def test_the_scheduler_needs_no_torch(lib_built):
    done = subprocess.run([sys.executable, "-c", WITHOUT_TORCH], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, done.stderr[-2000:]
