"""The draw of the next token against its definition: what top-k, top-p and min-p keep, and among that the first entry in the order of the
vocabulary whose running weight passes u's part of the sum.

Tokens have to be equal.  The kernel's weights are within 4e-14 of e^((l - max) / T), that is 0.04 units of 2^-40 at the most, and NumPy's
within 2^-52: so of the largest whole numbers up to one in twelve differs by one unit, and of smaller ones fewer.  A sum over weights
of together S is then off by less than S / 12 units of S 2^40.  A token (or the end of what is kept) differs only where its target lies
that close to one of the borders: with 2^17 entries in 2^17 2 / 12 / 2^40, 2e-8 of the rows here, whose inputs are seeded.  prob: a
quotient in 64 bits of such sums, 2^-40 of it, rounded to fp32: 1e-7.
"""
import math

import numpy as np
import pytest
import torch

from mx230_b200 import serving

pytestmark = pytest.mark.gpu

BIG = float(np.finfo(np.float32).max)


def draw(row, u, t, k, p, m):
    """(token, probability) of one row of logits, from the definition."""
    u, t, p, m = (float(np.float32(v)) for v in (u, t, p, m))
    index = np.flatnonzero(~np.isnan(row) & (row != -np.inf))
    if not index.size:
        return -1, 0.0
    value = np.minimum(row[index].astype(np.float64), BIG)
    order = np.lexsort((index, -value))
    if not t > 0 or p <= 0:
        return int(index[order[0]]), 1.0
    if k > 0:
        order = order[:k]
    with np.errstate(over="ignore"):
        w = np.exp((value[order] - value[order[0]]) / min(t, float(np.float32(1e30))))
    mass = np.floor(w * 2.0 ** 40 + 0.5).astype(np.int64)
    if p < 1:
        before = np.cumsum(mass) - mass
        mass = np.where(before < p * float(mass.sum()), mass, 0)
    if m > 0:
        mass = np.where(w >= min(m, 1.0), mass, 0)
    back = np.argsort(index[order], kind="stable")   # in the order of the vocabulary
    run = np.cumsum(mass[back])
    total = int(run[-1])
    target = min(math.floor((min(u, 1.0) if u > 0 else 0.0) * float(total)), total - 1)
    at = int(np.searchsorted(run, target, side="right"))
    return int(index[order[back[at]]]), int(mass[back[at]]) / total


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
    return (torch.randn(n, vocab, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


def uniforms(n, seed):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed)).tolist()


def test_in_the_order_of_the_vocabulary(handle):
    """Weights 1, 3, 2 and one that is cut off: the shares of u are those of the entries as they stand, not of the largest first."""
    x = torch.tensor([[0.0, math.log(3.0), -50.0, math.log(2.0)]]).expand(6, 4)
    u = [0.0, 0.16, 0.17, 0.66, 0.67, 0.99]
    assert check(handle, x, u).tolist() == [0, 0, 1, 1, 3, 3]
    for cut in (dict(k=2), dict(p=0.8), dict(m=0.5)):   # 3 and 2 are left: three fifths
        assert check(handle, x, u, **cut).tolist() == [1, 1, 1, 3, 3, 3]


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7, k=40, p=0.9), dict(p=0.95), dict(k=50, m=0.05), dict(t=1.5, m=0.01), dict(k=1), dict(k=700),
            dict(k=20000), dict(k=20000, p=0.99, m=0.001), dict(t=0.3, k=5000, p=0.999), dict(p=1e-6), dict(t=4.0, p=0.5, m=0.2), dict(t=100.0, k=3000, p=0.7),
            dict(t=3.0, p=0.8)]


@pytest.mark.parametrize("s", SETTINGS, ids=str)
@pytest.mark.parametrize("vocab,dtype", [(1, torch.float32), (2, torch.float16), (61, torch.float32), (1000, torch.bfloat16), (4099, torch.float32),
                                         (32000, torch.float32), (50257, torch.bfloat16), (50257, torch.float16), (128001, torch.float32)])
def test_matches_the_definition(handle, vocab, dtype, s):
    n = 6 if vocab < 60000 else 3
    check(handle, logits_of(n, vocab, 2.5, vocab + len(str(s)), dtype), uniforms(n, vocab), **s, what=(vocab, s))


@pytest.mark.parametrize("vocab", [2, 3, 31, 33, 127, 128, 129, 130, 511, 512, 513, 1023, 1024, 1025])
def test_lists_of_every_length(handle, vocab):
    x = logits_of(5, vocab, 1.0, vocab)
    x[1] = x[1].round()
    x[2] = 0.5
    x[3, : vocab // 2] = -math.inf
    for s in (dict(k=vocab - 1), dict(p=0.99), dict(t=2.0, k=vocab // 2 + 1, p=0.8), dict(m=0.1), dict(k=vocab - 1, m=0.3)):
        check(handle, x, [0.5, 0.97, 0.999, 0.2, 1.0], **s, what=(vocab, s))


def test_the_largest_vocabulary(handle):
    """A CTA has an eighth of a row, or all of it."""
    x = logits_of(1, 1 << 22, 2.0, 5).cuda()
    row, u = x[0].cpu().numpy(), [0.3, 0.9999999]
    for s in (dict(), dict(p=0.9), dict(k=50), dict(t=50.0, k=100_000, p=0.9)):
        want = [draw(row, v, s.get("t", 1.0), s.get("k", 0), s.get("p", 1.0), 0.0)[0] for v in u]
        for n in (2, 150):
            token = torch.empty(n, dtype=torch.int32, device="cuda")
            serving.sample(handle, token, x.expand(n, 1 << 22), torch.tensor(u * (n // 2), device="cuda"), s.get("t", 1.0), s.get("k", 0), s.get("p", 1.0))
            assert token.tolist() == want * (n // 2), (n, s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,vocab", [(40, 128000), (160, 50257), (300, 7001), (19, 200003)])
def test_batches_of_every_size(handle, n, vocab, dtype):
    """Rows over eight CTAs to one, kept in shared memory or read again: the tokens of the same rows by themselves, and some rows
    against the definition."""
    x = logits_of(4, vocab, 2.0, vocab, dtype).repeat(-(-n // 4), 1)[:n].cuda()
    u = torch.rand(n, generator=torch.Generator().manual_seed(n)).cuda()
    for s in (dict(), dict(top_p=0.95), dict(temperature=0.8, top_k=40, top_p=0.9), dict(min_p=0.02), dict(temperature=0.0), dict(temperature=3.0, top_k=3000)):
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
    for vocab in (3001, 30011):
        x = logits_of(n, vocab, 3.0, 17)
        x[5], x[6, 1:], x[7, :vocab - 2] = -math.inf, -math.inf, -math.inf
        check(handle, x, uniforms(n, 9), g.choice([0.0, -1.0, math.nan, 0.5, 1.0, 2.0, 1e-30, math.inf], n).tolist(),
              g.choice([0, -5, 1, 2, 30, 600, 3001, 2 ** 31 - 1], n).tolist(), g.choice([1.0, 2.0, 0.0, -1.0, math.nan, 0.1, 0.9, 0.9999], n).tolist(),
              g.choice([0.0, -1.0, math.nan, 1e-9, 0.1, 1.0, 7.0], n).tolist())


@pytest.mark.parametrize("s", [dict(), dict(p=0.5), dict(k=7), dict(k=1500), dict(k=1500, p=0.25), dict(m=1.0), dict(t=0.0), dict(t=1e-20, k=3), dict(k=1500, p=0.25, m=1.0)],
                         ids=str)
@pytest.mark.parametrize("vocab", [9, 5000, 70001])
def test_equal_logits(handle, vocab, s):
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
    check(handle, torch.tensor([[-inf, 6e4, inf, -6e4, 0.0]]).half(), [0.6])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_infinities_than_a_list(handle, dtype):
    """They count as the largest number, one as much as another: the first ones by index are kept."""
    x = logits_of(4, 40000, 2.0, 3, dtype)
    x[0, 100:9000] = math.inf
    x[1, ::3] = math.inf
    x[2, 7], x[2, 39999] = math.inf, math.inf
    x[3, 1::2], x[3, ::2] = math.inf, -math.inf
    for s in (dict(), dict(k=1500), dict(k=1500, p=0.5), dict(p=0.3), dict(k=3), dict(m=0.5), dict(t=0.0), dict(k=20000, m=1.0)):
        check(handle, x, [0.0, 0.5, 0.7, 0.9999], **s, what=s)


@pytest.mark.parametrize("t", [1e-45, 1e-44, 1e-42, 1e-40, 3e-39, 8e-39, 1.2e-38, 1e-37, 1e-36, 1e-30])
@pytest.mark.parametrize("scale", [1.0, 20.0, 1000.0, 1e5])
def test_the_smallest_temperatures(handle, t, scale):
    """Logits as close to each other as such a temperature tells apart, at 0 and where floats are farther apart, and others far below."""
    t = float(np.float32(t))
    g = np.random.default_rng(int(scale))
    x = (g.random((6, 3001)) * -t * scale).astype(np.float32)
    x[:, 0], x[:, 1], x[:, 2] = 0.0, -1e-37, -2.0
    x[1] += np.float32(3e-38)
    x[2] += np.float32(1e-33)
    x[3, 1700:] = -math.inf
    x[4] -= np.float32(1e-37)
    x[5] *= 1e30
    for s in (dict(), dict(p=0.9), dict(k=2), dict(k=1500), dict(k=1500, p=0.5), dict(m=0.5), dict(p=0.9, m=0.01)):
        check(handle, torch.from_numpy(x), [0.0, 0.3, 0.5, 0.7, 0.9, 0.99], t=t, **s, what=s)


def test_random_numbers_at_and_outside_the_ends(handle):
    u = [0.0, -1.0, math.nan, 1.0, 2.0, math.inf, -math.inf, 1 - 2.0 ** -24]
    for vocab in (3000, 40000):
        x = logits_of(1, vocab, 2.0, 2).expand(len(u), vocab)   # the same row for all
        for s in (dict(), dict(k=20), dict(p=0.9), dict(k=20, m=0.1), dict(k=2000)):
            check(handle, x, u, **s, what=s)


def test_the_shares_of_the_draws(handle):
    """Equal steps of u: an entry's share of the draws is its probability, off by a step at either end."""
    many = logits_of(1, 700, 2.0, 6).cuda().expand(5000, 700)
    token = torch.empty(5000, dtype=torch.int32, device="cuda")
    serving.sample(handle, token, many, torch.arange(5000, device="cuda", dtype=torch.float32) / 5000)
    share = torch.bincount(token.long(), minlength=700).double() / 5000
    assert float((share - torch.softmax(many[0].double(), 0)).abs().max()) <= 2 / 5000
    assert (token[1:] >= token[:-1]).all()


def test_captured_strided_and_on_another_stream(handle):
    store = logits_of(8, 20011, 2.5, 12).cuda()
    x = store[:, 3:20003]
    u, token, prob = torch.rand(8, device="cuda"), torch.empty(8, dtype=torch.int32, device="cuda"), torch.empty(8, device="cuda")
    k = torch.full((8,), 40, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        serving.sample(handle, token, x, u, 0.8, k, 0.9, prob=prob)
    for seed in (1, 2, 3):
        x.copy_(logits_of(8, 20000, 2.5, 100 + seed)), u.copy_(torch.tensor(uniforms(8, seed))), k.fill_((10, 600, 0)[seed - 1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(check(handle, x, u.tolist(), 0.8, (10, 600, 0)[seed - 1], 0.9), token)
    other = torch.empty_like(token)
    torch.cuda.synchronize()
    serving.sample(handle, other, x, u, 0.8, k, 0.9, stream=side)   # two at once
    serving.sample(handle, token, x, u, 0.8, k, 0.9)
    torch.cuda.synchronize()
    assert torch.equal(other, token)


def test_a_masked_row_among_others(handle):
    """The sampler says which row has no token, and has the others'."""
    sampler, x = serving.Sampler(handle, 3), logits_of(4, 500, 2.0, 1).cuda()
    rows = [(r, r + 1, serving.Request([1], 9, 0.8, 40, 0.9)) for r in range(4)]
    want = sampler.draw(x, rows)
    x[2] = math.nan
    with pytest.raises(serving.MaskedLogits, match="request 2") as e:
        sampler.draw(x, rows)
    assert e.value.tokens == [*want[:2], -1, want[3]]
    x[2, 7] = 1.0
    assert sampler.draw(x, rows) == [*want[:2], 7, want[3]]
