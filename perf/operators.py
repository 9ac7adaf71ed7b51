"""What a decode step does outside attention, as cases that can be timed and compared with a plain form.

  int4     rows times a matrix of 4-bit weights with group scales: y = x W + b, plus a residual (`llm_attention.gemv_int4`)
  rotary   rotary positions of q and k heads, or the gradient through them (`llm_attention.rotary`)
  sample   the next token of each row of logits, from given random numbers (`serving.sample`)
"""
import math

import numpy as np
import torch

own = False

MASS = 2.0 ** 40   # the weight of a row's largest logit in `sample`; weights are whole numbers
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}

_handle = None


def handle():
    """The program's handle: one per device, kept for the life of the process."""
    global _handle
    if _handle is None:
        from mx230_b200.common import Handle
        _handle = Handle(torch.cuda.current_device(), 64 << 20)
    return _handle


def listed():
    return [
        # The q, k, v projection of one token, 14 query and 2 key/value heads: the smallest product of a decode step.
        {"name": "int4 896>1152 x1", "op": "int4", "n_in": 896, "n_out": 1152, "rows": 1, "group": 32, "zeros": False, "bias": True, "add": False},
        # A larger model's up projection for one token, weights with zero points.
        {"name": "int4 4096>14336 x1", "op": "int4", "n_in": 4096, "n_out": 14336, "rows": 1, "group": 128, "zeros": True, "bias": False, "add": False},
        # The way back, eight sequences decoding together, added to the residual row.
        {"name": "int4 14336>4096 x8", "op": "int4", "n_in": 14336, "n_out": 4096, "rows": 8, "group": 64, "zeros": True, "bias": False, "add": True},
        # The logits of four sequences: the largest matrix of a step.
        {"name": "int4 4096>128000 x4", "op": "int4", "n_in": 4096, "n_out": 128000, "rows": 4, "group": 128, "zeros": False, "bias": False, "add": False},
        # One token's q and k heads at a far position, host-launched.
        {"name": "rotary 1x16x64 fp32", "op": "rotary", "rows": 1, "heads": 16, "dim": 64, "rot": 64, "dtype": "fp32", "interleaved": False,
         "inverse": False, "head_major": False, "first": 130001, "scaling": "wavelength"},
        # The q and k heads of a prompt's chunk behind 100000 tokens, rows of the q|k|v projection, ragged.
        {"name": "rotary 1900x36x64 fp32", "op": "rotary", "rows": 1900, "heads": 36, "dim": 64, "rot": 64, "dtype": "fp32", "interleaved": False,
         "inverse": False, "head_major": False, "first": 100000, "scaling": "yarn"},
        # A quarter of each head rotated, interleaved pairs, an odd number of rows.
        {"name": "rotary 4097x12x80/20 fp16", "op": "rotary", "rows": 4097, "heads": 12, "dim": 80, "rot": 20, "dtype": "fp16", "interleaved": True,
         "inverse": False, "head_major": False, "first": 0, "scaling": "none"},
        # Training: the gradient of 16384 tokens back from the head-major order in which attention takes them.
        {"name": "rotary 16384x40x128 bf16 grad", "op": "rotary", "rows": 16384, "heads": 40, "dim": 128, "rot": 128, "dtype": "bf16", "interleaved": False,
         "inverse": True, "head_major": True, "first": 0, "scaling": "linear"},
        # One interactive sequence with the usual three limits.
        {"name": "sample 1x32000 fp32", "op": "sample", "rows": 1, "vocab": 32000, "dtype": "fp32", "filters": "k40 p.9", "masked": 0.0, "spread": 2.5},
        # A full serving batch that is cut by probability alone: long nuclei.
        {"name": "sample 64x128000 fp32", "op": "sample", "rows": 64, "vocab": 128000, "dtype": "fp32", "filters": "p.95", "masked": 0.0, "spread": 2.0},
        # Every request with settings of its own, an odd vocabulary, logits in 16 bits (many ties).
        {"name": "sample 200x50257 bf16", "op": "sample", "rows": 200, "vocab": 50257, "dtype": "bf16", "filters": "mixed", "masked": 0.0, "spread": 3.0},
        # Constrained output: a grammar masks most of the vocabulary.
        {"name": "sample 16x128000 masked", "op": "sample", "rows": 16, "vocab": 128000, "dtype": "fp32", "filters": "k50 m.05", "masked": 0.97, "spread": 2.5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["int4", "rotary", "sample"])
    if op == "int4":
        n_in = rng.choice([_log_int(rng, 64, 16384), 64 * _log_int(rng, 1, 256)])
        n_out = _log_int(rng, 64, min(131072, 500_000_000 // n_in))
        return {"op": op, "n_in": n_in, "n_out": n_out, "rows": rng.choice([1, 1, rng.randint(2, 8), rng.randint(2, 16)]),
                "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "bias": rng.random() < 0.5, "add": rng.random() < 0.3}
    if op == "rotary":
        dim = rng.choice([64, 64, 80, 128, 96, 256])
        heads = _log_int(rng, 1, 48)
        rows = _log_int(rng, 1, min(32768, 80_000_000 // (heads * dim)))
        return {"op": op, "rows": rows, "heads": heads, "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4]),
                "dtype": rng.choice(["fp32", "fp16", "bf16"]), "interleaved": rng.random() < 0.5, "inverse": rng.random() < 0.4,
                "head_major": rng.random() < 0.4, "first": rng.choice([0, _log_int(rng, 1, 1_000_000)]),
                "scaling": rng.choice(["none", "linear", "ntk", "wavelength", "yarn"])}
    vocab = _log_int(rng, 1000, 200_000)
    return {"op": op, "rows": _log_int(rng, 1, min(256, 8_000_000 // vocab)), "vocab": vocab, "dtype": rng.choice(["fp32", "fp32", "fp16", "bf16"]),
            "filters": rng.choice(["greedy", "plain", "k40 p.9", "p.95", "k50 m.05", "mixed"]), "masked": rng.choice([0.0, 0.0, 0.5, 0.97]),
            "spread": rng.uniform(1.0, 4.0)}


# ---------------------------------------------------------------- inputs
THETA = 5e5
SCALING = {"none": None, "linear": {"kind": "linear", "factor": 4.0}, "ntk": {"kind": "ntk", "factor": 8.0},
           "wavelength": {"kind": "wavelength", "factor": 8.0, "low": 1.0, "high": 4.0, "length": 8192},
           "yarn": {"kind": "yarn", "factor": 16.0, "fast": 32.0, "slow": 1.0, "length": 8192}}


def _frequencies(rot, scaling):
    """Radians per position of each pair, and the factor on both outputs."""
    half, s = rot // 2, SCALING[scaling]
    f, factor = [THETA ** (-2.0 * i / rot) for i in range(half)], 1.0
    if scaling == "linear":
        f = [x / s["factor"] for x in f]
    elif scaling == "ntk":
        theta = THETA * s["factor"] ** (rot / (rot - 2.0)) if rot > 2 else THETA
        f = [theta ** (-2.0 * i / rot) for i in range(half)]
    elif scaling == "wavelength":
        for i, x in enumerate(f):
            turns = s["length"] * x / (2 * math.pi)   # turns over the trained length
            part = min(1.0, max(0.0, (turns - s["low"]) / (s["high"] - s["low"])))
            f[i] = part * x + (1 - part) * x / s["factor"]
    elif scaling == "yarn":
        at = [rot * math.log(s["length"] / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (s["fast"], s["slow"])]
        lo, hi = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
        for i, x in enumerate(f):
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))   # 1: interpolated
            f[i] = part * x / s["factor"] + (1 - part) * x
        factor = 0.1 * math.log(s["factor"]) + 1.0
    return f, factor


def _filters(case, g):
    """temperature, top_k, top_p, min_p: numbers for all rows, or one per row."""
    n = case["rows"]
    if case["filters"] == "greedy":
        return 0.0, 0, 1.0, 0.0
    if case["filters"] == "plain":
        return 1.0, 0, 1.0, 0.0
    if case["filters"] == "k40 p.9":
        return 0.8, 40, 0.9, 0.0
    if case["filters"] == "p.95":
        return 1.0, 0, 0.95, 0.0
    if case["filters"] == "k50 m.05":
        return 0.7, 50, 1.0, 0.05
    pick = lambda a: torch.tensor(a, device="cuda")[torch.randint(0, len(a), (n,), device="cuda", generator=g)]  # noqa: E731
    return (pick([0.0, 0.6, 0.8, 1.0, 1.3]), pick([0, 1, 20, 200, 2000]).to(torch.int32), pick([1.0, 0.5, 0.9, 0.99]), pick([0.0, 0.0, 0.02, 0.1]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    st = {"case": case}
    if case["op"] == "int4":
        n_in, n_out, rows = case["n_in"], case["n_out"], case["rows"]
        groups = -(-n_in // case["group"])
        st["codes"] = torch.randint(0, 16, (n_in, n_out), device="cuda", generator=g, dtype=torch.uint8)
        st["scales"] = ((0.5 + torch.rand(groups, n_out, device="cuda", generator=g)) * (0.25 / math.sqrt(n_in))).half()
        st["zeros"] = torch.randint(4, 12, (groups, n_out), device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
        st["bias"] = normal(n_out) * 0.1 if case["bias"] else None
        st["x"], st["old"], st["y"] = normal(rows, n_in), normal(rows, n_out), torch.empty(rows, n_out, device="cuda")
        if own:
            from mx230_b200 import llm_attention as la
            st["weights"] = la.pack_int4(handle(), st["codes"], st["scales"], st["zeros"])
    elif case["op"] == "rotary":
        n, heads, dim = case["rows"], case["heads"], case["dim"]
        # the heads of q and k lie in rows of the q|k|v projection, an eighth more heads behind them; or each head by itself
        more = heads + max(1, heads // 8)
        st["x"] = normal(heads, n, dim).to(TYPES[case["dtype"]]).transpose(0, 1) if case["head_major"] else \
            normal(n, more, dim).to(TYPES[case["dtype"]])[:, :heads]
        st["y"] = torch.empty(n, heads, dim, device="cuda", dtype=TYPES[case["dtype"]])
        st["pos"] = torch.arange(case["first"], case["first"] + n, device="cuda", dtype=torch.int32)
        f, st["factor"] = _frequencies(case["rot"], case["scaling"])
        st["freq"] = torch.tensor(f, device="cuda", dtype=torch.float64)
        if own:
            from mx230_b200 import llm_attention as la
            st["plan"] = la.Rotary(case["rot"], THETA, scaling=SCALING[case["scaling"]], interleaved=case["interleaved"])
    else:
        n, vocab = case["rows"], case["vocab"]
        logits = normal(n, vocab) * case["spread"]
        # a few likely continuations stand out, as a trained model's do
        top = torch.randint(0, vocab, (n, 8), device="cuda", generator=g)
        logits.scatter_(1, top, case["spread"] * 4 + normal(n, 8) * 2)
        if case["masked"]:
            logits = logits.masked_fill(torch.rand(n, vocab, device="cuda", generator=g) < case["masked"], -math.inf)
        st["logits"] = logits.to(TYPES[case["dtype"]])
        st["u"] = torch.rand(n, device="cuda", generator=g)
        st["filters"] = _filters(case, g)
        st["token"], st["prob"] = torch.empty(n, device="cuda", dtype=torch.int32), torch.empty(n, device="cuda")
    return st


# ---------------------------------------------------------------- one pass
def _run_own(st):
    from mx230_b200 import llm_attention as la
    from mx230_b200 import serving
    case = st["case"]
    if case["op"] == "int4":
        la.gemv_int4(handle(), st["y"], st["x"], st["weights"], st["bias"], add=st["old"] if case["add"] else None)
        return st["y"]
    if case["op"] == "rotary":
        la.rotary(handle(), st["y"], st["x"], st["pos"], st["plan"], inverse=case["inverse"])
        return st["y"]
    t, k, p, m = st["filters"]
    serving.sample(handle(), st["token"], st["logits"], st["u"], temperature=t, top_k=k, top_p=p, min_p=m, prob=st["prob"])
    return {"token": st["token"], "prob": st["prob"]}


def _plain_int4(st):
    case = st["case"]
    at = torch.arange(case["n_in"], device="cuda") // case["group"]
    zero = st["zeros"].float()[at] if st["zeros"] is not None else 8.0
    w = (st["codes"].float() - zero) * st["scales"].float()[at]
    y = st["x"] @ w
    if st["bias"] is not None:
        y = y + st["bias"]
    return y + st["old"] if case["add"] else y


def _plain_rotary(st):
    case, x, half = st["case"], st["x"], st["case"]["rot"] // 2
    angle = st["pos"].double()[:, None] * st["freq"]
    sign = -1.0 if case["inverse"] else 1.0
    cos, sin = (torch.cos(angle) * st["factor"]).float()[:, None], (torch.sin(angle) * (sign * st["factor"])).float()[:, None]
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
    y = x.float().clone()
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a] = xa * cos - xb * sin
    y[..., b] = xa * sin + xb * cos
    return y.to(x.dtype)


def _column(v, n, dtype):
    return (v.to(dtype) if isinstance(v, torch.Tensor) else torch.full((n,), v, device="cuda", dtype=torch.float32).to(dtype))[:, None]


def _plain_sample(st):
    n, vocab = st["logits"].shape
    t, k, p, m = (_column(v, n, torch.float64) for v in st["filters"])
    order = torch.sort(st["logits"].double(), dim=1, descending=True, stable=True)
    d = order.values - order.values[:, :1]
    # weights of the sorted entries; temperature 0 leaves the first alone
    w = torch.where(t > 0, torch.exp(d / torch.where(t > 0, t, 1.0)), 0.0)
    first = torch.arange(vocab, device="cuda")[None] == 0
    w = torch.where(first, 1.0, w)
    mass = torch.floor(w * MASS + 0.5).long()
    rank = torch.arange(vocab, device="cuda")[None]
    mass = torch.where((k <= 0) | (rank < k), mass, 0)
    before = torch.cumsum(mass, 1) - mass
    total = mass.sum(1, keepdim=True)
    mass = torch.where((p >= 1) | (before.double() < p * total.double()), mass, 0)
    mass = torch.where(w >= m, mass, 0)
    kept = torch.zeros_like(mass).scatter_(1, order.indices, mass)   # in the order of the vocabulary
    run = torch.cumsum(kept, 1)
    total = run[:, -1:]
    token = (run <= torch.floor(st["u"].double()[:, None] * total.double()).long()).sum(1)
    prob = kept.gather(1, token[:, None]).double() / total.double()
    return {"token": token.to(torch.int32), "prob": prob[:, 0].float()}


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_int4(state) if op == "int4" else _plain_rotary(state) if op == "rotary" else _plain_sample(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "int4":
        n_in, n_out, rows = case["n_in"], case["n_out"], case["rows"]
        groups = -(-n_in // case["group"])
        # codes, fp16 scales, 4-bit zero points, x, y (and what is added to it), bias
        b = n_in * n_out / 2 + groups * n_out * (2.5 if case["zeros"] else 2) + 4 * rows * (n_in + n_out * (2 if case["add"] else 1)) + \
            (4 * n_out if case["bias"] else 0)
        return {"bytes": b, "flops": 2.0 * rows * n_in * n_out}
    if case["op"] == "rotary":
        n = case["rows"] * case["heads"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2.0 * n * case["dim"] * size + 4 * case["rows"], "flops": 3.0 * n * case["rot"]}
    size = 4 if case["dtype"] == "fp32" else 2
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size + 12.0 * case["rows"], "flops": (1.0 if case["filters"] == "greedy" else 4.0) * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_int4(case, st):
    x, cols = st["x"].double(), []
    group = torch.arange(case["n_in"], device="cuda").div(case["group"], rounding_mode="floor")
    for o in range(0, case["n_out"], 4096):   # sum_i x_i s_i q_i - sum_i x_i s_i z_i, some columns at a time
        s = st["scales"][:, o:o + 4096].double().index_select(0, group)
        q = st["codes"][:, o:o + 4096].double()
        z = st["zeros"][:, o:o + 4096].double().index_select(0, group) if st["zeros"] is not None else torch.full_like(q, 8.0)
        cols.append(x @ (q * s - z * s))
    y = torch.cat(cols, 1)
    if case["bias"]:
        y += st["bias"].double()
    return y + st["old"].double() if case["add"] else y


def _exact_rotary(case, st):
    x, half = st["x"].double(), case["rot"] // 2
    turn = torch.exp(1j * torch.outer(st["pos"].double(), st["freq"])) * st["factor"]
    if case["inverse"]:
        turn = turn.conj()
    part = x[..., :2 * half]
    pairs = part.reshape(*part.shape[:-1], half, 2) if case["interleaved"] else part.reshape(*part.shape[:-1], 2, half).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(pairs[..., 0].contiguous(), pairs[..., 1].contiguous()) * turn[:, None])
    if not case["interleaved"]:
        z = z.transpose(-1, -2)
    return torch.cat([z.reshape(part.shape), x[..., 2 * half:]], -1)


def _exact_sample(case, st):
    n, vocab = case["rows"], case["vocab"]
    logits, u = st["logits"].float().cpu().numpy().astype(np.float64), st["u"].cpu().numpy().astype(np.float64)
    t, k, p, m = (v.cpu().numpy().astype(np.float64) if isinstance(v, torch.Tensor) else np.full(n, np.float32(v), np.float64) for v in st["filters"])
    prob = np.zeros(n)
    for r in range(n):
        row = logits[r]
        if t[r] <= 0:
            prob[r] = 1.0
            continue
        likely = np.flatnonzero(row > row.max() - 30 * t[r])   # (the others weigh less than half a unit)
        likely = likely[np.lexsort((likely, -row[likely]))]
        if k[r] > 0:
            likely = likely[:int(k[r])]
        w = np.exp((row[likely] - row[likely[0]]) / t[r])
        mass = [int(v) for v in np.floor(w * MASS + 0.5)]
        if p[r] < 1:
            limit, so_far, keep = p[r] * float(sum(mass)), 0, 0
            while keep < len(mass) and so_far < limit:
                so_far += mass[keep]
                keep += 1
            likely, w, mass = likely[:keep], w[:keep], mass[:keep]
        held = sorted((int(i), v) for i, v, x in zip(likely, mass, w) if x >= m[r])
        total, at = sum(v for _, v in held), 0
        limit = math.floor(u[r] * float(total))
        for _, v in held:
            at += v
            if at > limit:
                prob[r] = v / total
                break
    return {"token": None, "prob": torch.from_numpy(prob)}


def exact(case, seed):
    st = prepare(case, seed)
    return {"int4": _exact_int4, "rotary": _exact_rotary, "sample": _exact_sample}[case["op"]](case, st)
