"""Sampling from given random numbers against its definition, row by row with Python's whole numbers.

Tokens have to be equal.  A weight of the kernel is within 2^-48 of the definition's, far below half of the unit of 2^-40, so two
whole numbers differ only where a weight lies that close to the middle of two: one in 2^8 of the largest, and then by one unit in
a sum of 2^40 or more.  A token can differ only where the target lies within those few units of a border: below 1e-9 for a row
here, and the inputs are seeded.  prob: a quotient in 64 bits of sums that may be off by a few units, rounded to fp32: 1e-7.
"""
import math

import numpy as np
import pytest
import torch

from mx230_b200 import _lib, serving

pytestmark = pytest.mark.gpu


def draw(row, u, t, k, p, m):
    """(token, probability) of one row of logits, from the definition."""
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    u, t, p, m = f32(u), f32(t), f32(p), f32(m)
    big = float(np.finfo(np.float32).max)
    row = [(min(float(v), big), i) for i, v in enumerate(row) if not math.isnan(v) and v != -math.inf]
    if not row:
        return -1, 0.0
    row.sort(key=lambda e: (-e[0], e[1]))
    if not t > 0 or p <= 0:
        return row[0][1], 1.0
    t, top = min(t, f32(1e30)), row[0][0]
    if k > 0:
        row = row[:k]
    w = [math.exp((v - top) / t) for v, _ in row]
    mass = [math.floor(x * 2 ** 40 + 0.5) for x in w]
    n = len(row)
    if p < 1:
        target, run, n = p * float(sum(mass)), 0, 0
        while n < len(row) and run < target:
            run += mass[n]
            n += 1
    if m > 0:
        n = min(n, sum(x >= min(m, 1.0) for x in w))
    total = sum(mass[:n])
    u = min(u, 1.0) if u > 0 else 0.0
    target, run = min(math.floor(u * float(total)), total - 1), 0
    for i in range(n):
        run += mass[i]
        if run > target:
            return row[i][1], mass[i] / total
    raise AssertionError


def check(handle, logits, u, t=1.0, k=0, p=1.0, m=0.0, what=""):
    n = logits.shape[0]
    token, prob = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.full((n,), math.nan, device="cuda")
    dev = lambda v, ty: torch.tensor(v, dtype=ty, device="cuda") if isinstance(v, list) else v  # noqa: E731
    x = logits if logits.is_cuda else logits.cuda()
    serving.sample(handle, token, x, dev(u, torch.float32), dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32),
                   dev(m, torch.float32), prob)
    rows = x.float().cpu().numpy()
    pick = lambda v, r: v[r] if isinstance(v, list) else v  # noqa: E731
    want = [draw(rows[r], u[r], pick(t, r), pick(k, r), pick(p, r), pick(m, r)) for r in range(n)]
    got = token.tolist()
    assert got == [w[0] for w in want], (what, [(r, g, w) for r, (g, w) in enumerate(zip(got, want)) if g != w[0]][:8])
    assert np.abs(prob.cpu().numpy() - np.array([w[1] for w in want])).max() < 1e-7, what
    return token


def logits_of(n, vocab, spread, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, vocab, generator=g) * spread).to(dtype)


def uniforms(n, seed):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed)).tolist()


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7, k=40, p=0.9), dict(p=0.95), dict(k=50, m=0.05), dict(t=1.5, m=0.01), dict(k=1), dict(k=700),
            dict(t=0.3, k=5000, p=0.999), dict(p=1e-6), dict(t=4.0, p=0.5, m=0.2), dict(t=100.0, k=3000, p=0.7)]


@pytest.mark.parametrize("s", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab,dtype", [(1, torch.float32), (2, torch.float16), (61, torch.float32), (1000, torch.bfloat16), (4099, torch.float32),
                                         (32000, torch.float32), (50257, torch.bfloat16), (50257, torch.float16), (128001, torch.float32)])
def test_matches_the_definition(handle, vocab, dtype, s):
    n = 6 if vocab < 60000 else 3
    x = logits_of(n, vocab, 2.5, vocab + len(str(s)), dtype)
    check(handle, x, uniforms(n, vocab), **s, what=(vocab, s))


@pytest.mark.parametrize("vocab", [2, 3, 31, 33, 127, 128, 129, 130, 511, 512, 513, 1023, 1024, 1025])
def test_lists_of_every_length(handle, vocab):
    """Rows that are looked at whole, however long the list: equal logits among them, and the last entry drawn."""
    x = logits_of(5, vocab, 1.0, vocab)
    x[1] = x[1].round()
    x[2] = 0.5
    x[3, : vocab // 2] = -math.inf
    for s in (dict(k=vocab - 1), dict(p=0.99), dict(t=2.0, k=vocab // 2 + 1, p=0.8), dict(m=0.1)):
        check(handle, x, [0.5, 0.97, 0.999, 0.2, 1.0], **s, what=(vocab, s))


def test_the_largest_vocabulary(handle):
    x = logits_of(1, 1 << 22, 2.0, 5, torch.float32)
    for s in (dict(p=0.9), dict(k=50), dict(t=50.0, k=100_000, p=0.9)):
        check(handle, x, [0.3], **s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab", [(40, 128000), (160, 50257), (300, 7001), (19, 200003)])
def test_batches_of_every_size(handle, n, vocab, dtype):
    """Rows over eight CTAs to one, kept in shared memory or read again: the tokens of the same rows by themselves, and some rows
    against the definition."""
    x = logits_of(4, vocab, 2.0, vocab, dtype).repeat(-(-n // 4), 1)[:n].cuda()
    u = torch.rand(n, generator=torch.Generator().manual_seed(n)).cuda()
    for s in (dict(top_p=0.95), dict(temperature=0.8, top_k=40, top_p=0.9), dict(min_p=0.02), dict(temperature=0.0), dict(temperature=3.0, top_k=3000)):
        token, one, prob = (torch.empty(n, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.float32))
        serving.sample(handle, token, x, u, **s, prob=prob)
        for r in range(0, n, 7):
            serving.sample(handle, one[r:r + 1], x[r:r + 1], u[r:r + 1], **s)
        assert torch.equal(token[::7], one[::7]), s
        rows = x[:2].float().cpu().numpy()
        for r in range(2):
            want = draw(rows[r], u[r].item(), s.get("temperature", 1.0), s.get("top_k", 0), s.get("top_p", 1.0), s.get("min_p", 0.0))
            assert token[r].item() == want[0] and abs(prob[r].item() - want[1]) < 1e-7, (s, r)


def test_settings_of_each_row(handle):
    n = 97
    g = np.random.default_rng(3)
    x = logits_of(n, 3001, 3.0, 17)
    x[5], x[6, 1:], x[7, :2999] = -math.inf, -math.inf, -math.inf
    check(handle, x, uniforms(n, 9), g.choice([0.0, -1.0, math.nan, 0.5, 1.0, 2.0, 1e-30, math.inf], n).tolist(),
          g.choice([0, -5, 1, 2, 30, 600, 3001, 2 ** 31 - 1], n).tolist(), g.choice([1.0, 2.0, 0.0, -1.0, math.nan, 0.1, 0.9, 0.9999], n).tolist(),
          g.choice([0.0, -1.0, math.nan, 1e-9, 0.1, 1.0, 7.0], n).tolist())


@pytest.mark.parametrize("s", [dict(), dict(p=0.5), dict(k=7), dict(k=1500), dict(k=1500, p=0.25), dict(m=1.0), dict(t=0.0), dict(t=1e-20, k=3)], ids=str)
@pytest.mark.parametrize("vocab", [9, 5000, 70001])
def test_equal_logits_go_by_index(handle, vocab, s):
    """Rows of one value, of two, of a few (more equal entries than a list holds), and masks of the lowest number."""
    x = torch.zeros(5, vocab)
    x[1, vocab // 2:] = 1.0
    x[2] = torch.randint(0, 4, (vocab,), generator=torch.Generator().manual_seed(1)).float() * 0.5
    x[3] = torch.finfo(torch.float32).min
    x[3, vocab // 3:] = -2.0
    x[4] = torch.finfo(torch.float32).min
    for seed in range(2):
        check(handle, x, uniforms(5, seed), **s, what=(vocab, s))


def test_masked_rows_infinities_and_zeros(handle):
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    rows = [[-inf] * 6, [nan] * 6, [nan, -inf, 3.0, nan, -inf, -inf], [inf, 1.0, inf, nan, -inf, 2.0], [low] * 5 + [-inf], [0.0, -0.0, 0.0, -0.0, -1e-45, 1e-45],
            [1e38, -1e38, 3e38, -3e38, 0.0, 1.0], [-inf, -inf, -inf, -inf, -inf, low]]
    for s in (dict(), dict(t=0.0), dict(k=2), dict(p=0.5), dict(m=0.5), dict(t=1e38, p=0.9), dict(t=1e-40)):
        for u in (0.0, 0.4, 0.9999999):
            check(handle, torch.tensor(rows), [u] * len(rows), **s, what=(s, u))
    half = torch.tensor([[-inf, 6e4, inf, -6e4, 0.0]]).half()
    check(handle, half, [0.6])


def test_random_numbers_at_and_outside_the_ends(handle):
    u = [0.0, -1.0, math.nan, 1.0, 2.0, math.inf, -math.inf, 1 - 2.0 ** -24]
    x = logits_of(1, 3000, 2.0, 2).expand(len(u), 3000)   # the same row for all
    for s in (dict(), dict(k=20), dict(p=0.9), dict(k=20, m=0.1)):
        check(handle, x, u, **s, what=s)


def test_strides_and_a_row_does_not_depend_on_the_others(handle):
    for dtype, off in ((torch.float32, 1), (torch.float32, 3), (torch.bfloat16, 5), (torch.float16, 0)):
        store = logits_of(40, 5011, 3.0, 21, dtype).cuda()
        x = store[:, off:off + 5000]
        u = uniforms(40, 4)
        token = check(handle, x, u, 0.9, 300, 0.95)
        for r in (0, 17, 39):
            assert check(handle, x[r:r + 1], u[r:r + 1], 0.9, 300, 0.95).item() == token[r].item()
    many = logits_of(1, 700, 2.0, 6).cuda().expand(5000, 700)
    token = torch.empty(5000, dtype=torch.int32, device="cuda")
    u = torch.arange(5000, device="cuda", dtype=torch.float32) / 5000
    serving.sample(handle, token, many, u, top_k=0)
    # shares of the draws against the probabilities: 5000 equal steps of u, so each entry's share is off by a step at either end
    w = torch.softmax(many[0].double(), 0)
    share = torch.bincount(token.long(), minlength=700).double() / 5000
    assert float((share - w).abs().max()) <= 2 / 5000


def test_captured_replayed_and_on_another_stream(handle):
    x = logits_of(8, 20000, 2.5, 12).cuda()
    u, token, prob = torch.rand(8, device="cuda"), torch.empty(8, dtype=torch.int32, device="cuda"), torch.empty(8, device="cuda")
    k = torch.full((8,), 40, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    serving.sample(handle, token, x, u, 0.8, k, 0.9, prob=prob)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        serving.sample(handle, token, x, u, 0.8, k, 0.9, prob=prob)
    for seed in (1, 2, 3):
        x.copy_(logits_of(8, 20000, 2.5, 100 + seed)), u.copy_(torch.tensor(uniforms(8, seed))), k.fill_(10 * seed)
        graph.replay()
        torch.cuda.synchronize()
        want = check(handle, x, u.tolist(), 0.8, 10 * seed, 0.9)
        assert torch.equal(want, token)
    other = torch.empty_like(token)
    torch.cuda.synchronize()
    serving.sample(handle, other, x, u, 0.8, k, 0.9, stream=side)   # two at once
    serving.sample(handle, token, x, u, 0.8, k, 0.9)
    torch.cuda.synchronize()
    assert torch.equal(other, token)


def test_refusals(handle):
    x = torch.zeros(3, 10, device="cuda")
    u, tok = torch.zeros(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    serving.sample(handle, tok[:0], x[:0], u[:0])
    bad = [lambda: serving.sample(handle, tok, x.cpu(), u), lambda: serving.sample(handle, tok, x.double(), u), lambda: serving.sample(handle, tok, x[0], u),
           lambda: serving.sample(handle, tok.long(), x, u), lambda: serving.sample(handle, tok, x, u[:2]), lambda: serving.sample(handle, tok[:2], x, u),
           lambda: serving.sample(handle, tok, x.t().contiguous().t(), u), lambda: serving.sample(handle, tok, x, u.half()),
           lambda: serving.sample(handle, tok, x, u, top_k=u), lambda: serving.sample(handle, tok, x, u, top_p=u[:2]),
           lambda: serving.sample(handle, tok, x, u, prob=tok), lambda: serving.sample(handle, tok, x[:, :0], u)]
    for call in bad:
        with pytest.raises(_lib.Mx230Error) as e:
            call()
        assert e.value.code == _lib.ERR_INVALID_ARG
    with pytest.raises(_lib.Mx230Error) as e:
        serving.sample(handle, tok[:1], torch.zeros(1, (1 << 22) + 1, device="cuda"), u[:1])
    assert e.value.code == _lib.ERR_UNSUPPORTED
