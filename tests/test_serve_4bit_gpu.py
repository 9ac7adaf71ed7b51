"""A 4-bit model's serving path as a program puts it together: 4-bit projections, rotary positions scaled for a long context on part of
each head, the KV write and attention over a paged cache, 4-bit logits, and tokens drawn by each request's settings inside
`run_continuous`.  Served together and one at a time the tokens are the same, and the logits are those of the same
layer in 64 bits."""
import numpy as np
import pytest
import torch

from mx230_b200 import _lib
from mx230_b200 import llm_attention as la
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
