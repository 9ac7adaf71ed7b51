"""A 4-bit model's serving path as a program puts it together: 4-bit projections, rotary positions scaled for a long context on part of
each head, the KV write and attention over a paged cache, 4-bit logits, and tokens drawn by each request's settings inside
`run_continuous`.  Served together and one at a time the tokens are the same, and the logits are those of the same
layer in 64 bits."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from mx230_b200 import _lib
from mx230_b200 import llm_attention as la
from mx230_b200 import serving
from mx230_b200.paging import KvPool
from mx230_b200.serving import Request, Sampler, run_continuous
from tests.conftest import assert_close

pytestmark = pytest.mark.gpu

NH, NKV, E, VOCAB, BS, N_CTX, ROT, THETA = 8, 2, 448, 1003, 16, 160, 48, 1e5
QD, KVD = NH * 64, NKV * 64
STRIDE = QD + 2 * KVD
FIRST = 50_000   # positions of the rotation start here, as behind a long document
SCALING = {"kind": "yarn", "factor": 8.0, "slow": 1.0, "fast": 32.0, "length": 8192}


class FourBitModel:
    def __init__(self, handle, n_slots, quant):
        g = torch.Generator(device="cuda").manual_seed(31)
        self.h, self.quant = handle, quant
        self.cache = la.KvCache(n_slots, NKV, 64, quant)
        self.emb = torch.randn(VOCAB, E, device="cuda", generator=g)
        self.bias = torch.randn(STRIDE, device="cuda", generator=g) * 0.1
        self.plan = la.Rotary(ROT, THETA, SCALING)
        self.w, self.dense = {}, {}
        for name, n_in, n_out, group, scale in (("qkv", E, STRIDE, 32, 0.012), ("out", QD, E, 64, 0.01), ("logits", E, VOCAB, 128, 0.04)):
            codes = torch.randint(0, 16, (n_in, n_out), device="cuda", generator=g, dtype=torch.uint8)
            groups = -(-n_in // group)
            s = ((0.5 + torch.rand(groups, n_out, device="cuda", generator=g)) * scale).half()
            z = torch.randint(6, 10, (groups, n_out), device="cuda", generator=g, dtype=torch.uint8)
            self.w[name] = la.pack_int4(handle, codes, s, z, group=group)
            at = torch.arange(n_in, device="cuda") // group
            self.dense[name] = (codes.double() - z.double()[at]) * s.double()[at]
        self.seen = {}   # (tokens so far) -> logits

    def rows(self, tokens, pos):
        x = self.emb[tokens]
        qkv = torch.empty(len(tokens), STRIDE, device="cuda")
        la.gemv_int4(self.h, qkv, x, self.w["qkv"], self.bias)
        qk = qkv.unflatten(1, (NH + 2 * NKV, 64))[:, :NH + NKV]
        la.rotary(self.h, qk, qk, pos, self.plan)
        return x, qkv

    def logits(self, x, attn):
        y, out = torch.empty_like(x), torch.empty(len(x), VOCAB, device="cuda")
        la.gemv_int4(self.h, y, attn, self.w["out"], add=x)
        la.gemv_int4(self.h, out, y, self.w["logits"])
        return out

    def prefill(self, r, prompt, table):
        n = len(prompt)
        x, qkv = self.rows(torch.tensor(prompt, device="cuda"), FIRST)
        out = torch.empty(n, QD, device="cuda")
        pg = la.Paging(torch.from_numpy(np.ascontiguousarray(table)).cuda(), BS)
        la.prefill_step(self.h, out, qkv, self.cache, 0, n, NH, NKV, 64, THETA, STRIDE, QD, pg, use_rope=False)
        return self.logits(x[-1:], out[-1:].contiguous())[0]

    def decode_batched(self, cur, pos, tables):
        n = len(cur)
        p = torch.from_numpy(pos).cuda()
        x, qkv = self.rows(torch.from_numpy(cur.astype(np.int64)).cuda(), p + FIRST)
        out = torch.empty(n, QD, device="cuda")
        pg = la.Paging(torch.from_numpy(np.ascontiguousarray(tables)).cuda(), BS)
        la.batched_step(self.h, out, qkv, self.cache, p, n, NH, NKV, 64, THETA, pg, STRIDE, QD, use_rope=False)
        lg = self.logits(x, out)
        for i in range(n):
            self.seen[(int(tables[i][0]), int(pos[i]))] = lg[i].double().cpu().numpy()
        return lg

    def plain(self, tokens):
        """Logits behind the last of `tokens` in 64 bits."""
        n = len(tokens)
        x = self.emb[torch.tensor(tokens, device="cuda")].double()
        qkv = (x @ self.dense["qkv"] + self.bias.double()).unflatten(1, (NH + 2 * NKV, 64))
        i = torch.arange(ROT // 2, device="cuda", dtype=torch.float64)
        f = THETA ** (-2 * i / ROT)
        pair = lambda turns: ROT * np.log(SCALING["length"] / (turns * 2 * np.pi)) / (2 * np.log(THETA))  # noqa: E731
        lo, hi = np.floor(pair(32.0)), np.ceil(pair(1.0))
        part = ((i - lo) / (hi - lo)).clamp(0, 1)
        f = part * f / 8 + (1 - part) * f
        ang = (FIRST + torch.arange(n, device="cuda").double())[:, None] * f
        c, s = (t[:, None] * (0.1 * np.log(8.0) + 1) for t in (ang.cos(), ang.sin()))
        a, b = qkv[:, :NH + NKV, :ROT // 2].clone(), qkv[:, :NH + NKV, ROT // 2:ROT].clone()
        qkv[:, :NH + NKV, :ROT // 2], qkv[:, :NH + NKV, ROT // 2:ROT] = a * c - b * s, a * s + b * c
        q, k, v = qkv[-1, :NH].unflatten(0, (NKV, NH // NKV)), qkv[:, NH:NH + NKV], qkv[:, NH + NKV:]
        pr = torch.softmax(torch.einsum("kgd,tkd->kgt", q, k) / 8, -1)
        y = torch.einsum("kgt,tkd->kgd", pr, v).reshape(1, QD) @ self.dense["out"] + x[-1:]
        return (y @ self.dense["logits"])[0].cpu().numpy()


@pytest.mark.parametrize("quant", [False, True])
def test_served_together_and_alone(handle, quant):
    g = np.random.default_rng(12)
    settings = [(0.0, 0, 1.0, 0.0), (0.9, 40, 0.9, 0.0), (1.1, 0, 0.95, 0.0), (0.7, 0, 1.0, 0.05), (1.0, 0, 1.0, 0.0)]
    reqs = [Request(g.integers(0, VOCAB, size=int(g.integers(3, 50))).tolist(), int(g.integers(1, 30)), *settings[i % 5]) for i in range(9)]
    n_slots = 40 * BS
    handle.set_option(_lib.OPT_DECODE_CHUNK, 256)   # (the key split, and with it the order of the sums, does not go by the batch)
    try:
        model = FourBitModel(handle, n_slots, quant)
        trace = []
        together, st = run_continuous(model, KvPool(n_slots, BS), N_CTX, reqs, 4, trace=trace, sampler=Sampler(handle, 7))
        alone, _ = run_continuous(FourBitModel(handle, n_slots, quant), KvPool(n_slots, BS), N_CTX, reqs, 1, sampler=Sampler(handle, 7))
        other, _ = run_continuous(FourBitModel(handle, n_slots, quant), KvPool(n_slots, BS), N_CTX, reqs, 4, sampler=Sampler(handle, 8))
    finally:
        handle.set_option(_lib.OPT_DECODE_CHUNK, 0)
    handle.check_status()
    assert together == alone and [len(t) for t in together] == [r.max_new for r in reqs]
    assert st.seq_decodes / st.decode_steps > 2.0
    greedy = [i for i, r in enumerate(reqs) if r.temperature == 0]
    assert other != together and all(other[i] == together[i] for i in greedy)
    if quant:
        return
    # the logits of the last step of some requests against 64 bits (the prompt's attention has bf16 operands)
    last = max((i for i, t in enumerate(together) if len(t) > 2), key=lambda i: reqs[i].max_new)
    tokens = reqs[last].prompt + together[last][:-1]
    table = next(e[2] for e in trace if e[0] == "admit" and e[1] == last)
    got = model.seen[(table[0], len(tokens) - 1)]
    assert_close(got / np.abs(got).max(), model.plain(tokens) / np.abs(got).max(), "logits")


def test_a_masked_row_is_an_error(handle):
    sampler = Sampler(handle)
    with pytest.raises(_lib.Mx230Error):
        sampler.draw(torch.full((1, 50), float("-inf"), device="cuda"), [(3, 0, Request([1], 1))])


FIRST_CALLS = """
import torch
from mx230_b200 import llm_attention as la, serving
from mx230_b200.common import Handle
torch.cuda.set_device(0)
h = Handle(0, 16 << 20)
g = torch.Generator(device="cuda").manual_seed(0)
plan = la.Rotary(64, 1e4, device="cuda")
made = []
for n_in, n_out, rows in ((896, 300, 1), (4864, 896, 6), (14336, 512, 3)):
    codes = torch.randint(0, 16, (n_in, n_out), device="cuda", dtype=torch.uint8, generator=g)
    w = la.pack_int4(h, codes, torch.rand(-(-n_in // 64), n_out, device="cuda", generator=g).half(), group=64)
    made.append((torch.empty(rows, n_out, device="cuda"), torch.randn(rows, n_in, device="cuda", generator=g), w))
x = torch.randn(5, 4, 64, device="cuda", generator=g)
out = torch.empty_like(x)
logits, u = torch.randn(3, 70000, device="cuda", generator=g), torch.rand(3, device="cuda", generator=g)
token = torch.empty(3, dtype=torch.int32, device="cuda")
def calls():
    for y, a, w in made:
        la.gemv_int4(h, y, a, w)
    la.rotary(h, out, x, 7, plan)
    serving.sample(h, token, logits, u, top_p=0.9)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls()
graph.replay()
torch.cuda.synchronize()
results = [y for y, *_ in made] + [out, token]
captured = [r.clone() for r in results]
for r in results:
    r.zero_()
calls()
assert all(torch.equal(a, b) for a, b in zip(results, captured))
h.check_status()
"""


def test_the_first_calls_of_a_process_may_be_captured():
    """What the host asks and sets once (attributes, clusters that fit) it may do while a stream is captured."""
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300,
                          cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert done.returncode == 0, done.stderr[-2000:]


def test_two_streams_at_once(handle):
    """No call has a workspace: two of a kind on two streams, over and over, with the results of one after the other."""
    g = torch.Generator(device="cuda").manual_seed(3)
    codes = torch.randint(0, 16, (14336, 1024), device="cuda", dtype=torch.uint8, generator=g)
    w = la.pack_int4(handle, codes, torch.rand(224, 1024, device="cuda", generator=g).half(), group=64)
    xs = [torch.randn(n, 14336, device="cuda", generator=g) for n in (3, 8)]
    logits = [torch.randn(n, 128000, device="cuda", generator=g) * 3 for n in (2, 40)]
    us = [torch.rand(l.shape[0], device="cuda", generator=g) for l in logits]
    ys = [torch.empty(x.shape[0], 1024, device="cuda") for x in xs]
    tokens = [torch.empty(l.shape[0], dtype=torch.int32, device="cuda") for l in logits]

    def calls(i, **kw):
        la.gemv_int4(handle, ys[i], xs[i], w, **kw)
        serving.sample(handle, tokens[i], logits[i], us[i], top_p=0.95, **kw)

    calls(0), calls(1)
    want = [t.clone() for t in ys + tokens]
    torch.cuda.synchronize()
    for t in ys + tokens:
        t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        calls(0, stream=streams[0]), calls(1, stream=streams[1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ys + tokens, want))
    handle.check_status()
