"""The measured cases of the embedding, dropout and 8-bit linear operators.

A case is a dict of plain values; its ``op`` says which operator it calls:

  lookup   rows of a table by token id, scaled:        Y[i] = s T[id_i]
  bag      weighted sums of rows over ragged bags:     Y[b] = s sum_j w_j T[id_j]
  grad     the table's gradient from the rows' ones:   dT[v] = s sum_{id_j = v} w_j dY[row_j]
  dropout  x / (1 - p) where a counter's bits keep it, and the gradient's pass
  fp8      x W + b with e4m3 operands and a power-of-two scale for every 128 of K

Ids outside the table (an unseen word is -1) read nothing: zeros, and no
gradient.  Token ids follow the rank-frequency law that ids ordered by
frequency have (the chance of rank r falls as 1/r).
"""

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one short document looked up for scoring: nothing but latency
        dict(name="lookup one document", op="lookup", n=61, vocab=20000, dim=64,
             dtype="f32", scale=1.0),
        # a training batch's token embeddings, scaled by sqrt(dim)
        dict(name="lookup batch", op="lookup", n=262144, vocab=100000, dim=512,
             dtype="bf16", scale=22.627416997969522),
        # naive Bayes scores of 2000 sparse documents over 20 newsgroups
        dict(name="bag class scores", op="bag", bags=2000, mean_len=210,
             vocab=100000, dim=20, dtype="f32", weighted=True, scale=1.0),
        # pooled embeddings of a large batch of ragged documents
        dict(name="bag pooled", op="bag", bags=32768, mean_len=100,
             vocab=100000, dim=256, dtype="f16", weighted=True, scale=1.0),
        # a small mini-batch's gradient, odd sizes, sort included
        dict(name="grad small batch", op="grad", bags=777, mean_len=1,
             vocab=20000, dim=100, dtype="f32", weighted=False, scale=1.0,
             kept_plan=False),
        # an unpooled batch's gradient, the sort included, as every step pays
        dict(name="grad batch", op="grad", bags=1048576, mean_len=1,
             vocab=100000, dim=256, dtype="bf16", weighted=False, scale=16.0,
             kept_plan=False),
        # X^T D of binary logistic regression on review n-grams: the rows stay
        # the same through the fit, so the program keeps the sorted plan
        dict(name="grad logistic", op="grad", bags=65536, mean_len=120,
             vocab=100000, dim=2, dtype="f32", weighted=True, scale=1.0,
             kept_plan=True),
        # a small batch of random features
        dict(name="dropout small", op="dropout", rows=128, cols=1000,
             dtype="f32", p=0.1),
        # a large batch of wide features
        dict(name="dropout large", op="dropout", rows=32768, cols=8192,
             dtype="bf16", p=0.5),
        # one image's Fisher vector scored over 1000 classes
        dict(name="fp8 one row", op="fp8", rows=1, inner=16384, cols=1000,
             dtype="f32"),
        # speech frames' cosine features scored over 147 phones
        dict(name="fp8 phones", op="fp8", rows=1021, inner=8192, cols=147,
             dtype="f32"),
        # 8192 images' Fisher vectors scored over 1000 classes
        dict(name="fp8 images", op="fp8", rows=8192, inner=65536, cols=1000,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "bag", "grad", "dropout", "fp8"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "lookup":
        dim = _log(rng, 1, 1100)
        return dict(op=op, n=_log(rng, 1, min(262144, 134217728 // dim)),
                    vocab=_log(rng, 1, 200000), dim=dim, dtype=dtype,
                    scale=rng.choice([1.0, math.sqrt(dim)]))
    if op == "bag":
        dim, mean = _log(rng, 1, 600), _log(rng, 1, 400)
        most = max(1, min(32768, 3276800 // mean, 838860800 // (mean * dim)))
        return dict(op=op, bags=max(_log(rng, 1, most), 64 // mean),
                    mean_len=mean, vocab=_log(rng, 2, 200000), dim=dim, dtype=dtype,
                    weighted=rng.random() < 0.7, scale=1.0)
    if op == "grad":
        dim, mean = _log(rng, 1, 600), rng.choice([1, _log(rng, 2, 300)])
        most = max(1, min(1048576, 4194304 // mean,
                          268435456 // (mean * dim)))
        return dict(op=op, bags=max(_log(rng, 1, most), 64 // mean),
                    mean_len=mean, vocab=_log(rng, 2, 150000), dim=dim, dtype=dtype,
                    weighted=rng.random() < 0.5,
                    scale=rng.choice([1.0, 0.5]), kept_plan=rng.random() < 0.5)
    if op == "dropout":
        cols = _log(rng, 1, 20000)
        rows = _log(rng, 1, max(2, 134217728 // cols))
        return dict(op=op, rows=max(rows, -(-64 // cols)), cols=cols, dtype=dtype,
                    p=round(rng.uniform(0.01, 0.9), 4))
    inner, cols = _log(rng, 64, 40000), _log(rng, 2, 2000)
    return dict(op=op, rows=_log(rng, 1, min(8192, 2 ** 39 // (inner * cols))),
                inner=inner, cols=cols, dtype=dtype)


# ------------------------------------------------------------------ inputs
def _ids(n, vocab, g):
    """Ranks with chance about 1/rank; 2 in 100 words are unseen (-1)."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.exp(u * math.log(vocab + 1)).long().clamp_(1, vocab) - 1
    unseen = torch.rand(n, generator=g, device="cuda") < 0.02
    return torch.where(unseen, torch.full_like(ids, -1), ids)


def _lengths(bags, mean, g):
    """Document lengths: exponential about their mean, so some are empty and
    a few are many times longer."""
    u = torch.rand(bags, generator=g, device="cuda", dtype=torch.float64)
    return (-(1 - u).log() * mean).long().clamp_(max=20 * mean)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def number(most):
        return int(torch.randint(0, most, (1,), generator=g, device="cuda"))

    c, t = case, TYPES[case["dtype"]]
    s = {"case": c}
    if c["op"] == "lookup":
        s["table"] = normal(c["vocab"], c["dim"]).to(t)
        s["ids"] = _ids(c["n"], c["vocab"], g)
    elif c["op"] in ("bag", "grad"):
        one = c["op"] == "grad" and c["mean_len"] == 1  # not pooled
        lens = None if one else _lengths(c["bags"], c["mean_len"], g)
        n = c["bags"] if one else int(lens.sum())
        s["ids"], s["offsets"] = _ids(n, c["vocab"], g), None
        if not one:
            s["offsets"] = torch.zeros(c["bags"] + 1, dtype=torch.int64,
                                       device="cuda")
            torch.cumsum(lens, 0, out=s["offsets"][1:])
        # square roots of term counts
        s["weights"] = (1 + 3 * torch.rand(n, generator=g, device="cuda") ** 4
                        ).sqrt() if c["weighted"] else None
        if c["op"] == "bag":
            s["table"] = normal(c["vocab"], c["dim"]).to(t)
        else:
            s["dy"] = (0.1 * normal(c["bags"], c["dim"])).to(t)
    elif c["op"] == "dropout":
        s["x"] = normal(c["rows"], c["cols"]).to(t)
        s["dy"] = normal(c["rows"], c["cols"]).to(t)
        s["seed"], s["step"] = number(1 << 62), number(1 << 40)
    else:
        # power-normalised rows of unlike size, and W's columns too
        x = normal(c["rows"], c["inner"])
        x = x.sign() * x.abs().sqrt() * torch.exp(normal(c["rows"], 1))
        s["x"], s["bias"] = x.to(t), normal(c["cols"])
        W = normal(c["inner"], c["cols"]) / math.sqrt(c["inner"])
        s["W"] = W * torch.exp(0.5 * normal(1, c["cols"]))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "grad" and case["kept_plan"]:
        s["plan"] = _plan(s)
    elif case["op"] == "fp8":  # the weights as a server keeps them
        W = s.pop("W")
        if own:
            from keystone_amd import hip
            s["packed"] = hip.fp8_pack(W)
        else:
            q, s["W_scale"] = _blocks_of_128(W.t())
            s["W_e4m3"] = q.to(torch.float8_e4m3fn)
    return s


def _plan(s):
    """The order of the tokens that a program keeps while its rows stay."""
    c = s["case"]
    if own:
        from keystone_amd import hip
        return hip.embedding_plan(s["ids"], c["vocab"], s["offsets"])
    keep = (s["ids"] >= 0).nonzero().squeeze(1)
    rows = keep
    if s["offsets"] is not None:
        rows = torch.searchsorted(s["offsets"], keep, right=True) - 1
    return keep, s["ids"][keep], rows


# ------------------------------------------------------------- plain forms
def _philox(block, step, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011) in 64-bit integers:
    four 32-bit words for each block index."""
    m = 0xFFFFFFFF
    c = [block & m, (block >> 32) & m, torch.full_like(block, step & m),
         torch.full_like(block, (step >> 32) & m)]
    k0, k1 = seed & m, (seed >> 32) & m
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & m) ^ c[1] ^ k0, b & m,
             ((a >> 32) & m) ^ c[3] ^ k1, a & m]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return c


def _dropout(x, p, seed, step):
    n, t = x.numel(), round(p * 65536)
    words = _philox(torch.arange((n + 7) // 8, device=x.device), step, seed)
    bits = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1)
    keep = bits.reshape(-1)[:n].reshape(x.shape) >= t
    y = x.float() * (65536 / (65536 - t))
    return torch.where(keep, y, torch.zeros((), device=x.device)).to(x.dtype)


def _blocks_of_128(x):
    """Rows' values divided by their block's scale and rounded to e4m3, and
    the scales: the least power of two that brings the block under 448."""
    rows, n = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -n % 128)).view(rows, -1, 128)
    m, e = torch.frexp(x.abs().amax(2))
    e = torch.where(m > 0, e - 9 + (m > 0.875).int(), torch.zeros_like(e))
    scale = torch.ldexp(torch.ones_like(m), e.clamp(min=-127))
    q = (x / scale.unsqueeze(2)).to(torch.float8_e4m3fn)
    return q.float().view(rows, -1)[:, :n], scale


def _wide(scale, n):
    return scale.repeat_interleave(128, 1)[:, :n]


def run(state):
    s, c = state, state["case"]
    if own:
        from keystone_amd import hip
    if c["op"] == "lookup":
        if own:
            return hip.embedding_lookup(s["table"], s["ids"], c["scale"])
        keep = s["ids"] >= 0
        y = s["table"][s["ids"].clamp(min=0)].float() * c["scale"]
        return torch.where(keep.unsqueeze(1), y, torch.zeros_like(y)
                           ).to(s["table"].dtype)
    if c["op"] == "bag":
        if own:
            return hip.embedding_bag(s["table"], s["ids"], s["offsets"],
                                     s["weights"], c["scale"])
        keep, ids, rows = _plan(s)
        y = s["table"][ids].float()
        if s["weights"] is not None:
            y = y * s["weights"][keep].unsqueeze(1)
        out = torch.zeros(c["bags"], c["dim"], device=y.device)
        return (out.index_add_(0, rows, y) * c["scale"]).to(s["table"].dtype)
    if c["op"] == "grad":
        plan = s["plan"] if c["kept_plan"] else _plan(s)
        if own:
            return hip.embedding_grad(s["dy"], plan, s["weights"], c["scale"])
        keep, ids, rows = plan
        g = s["dy"][rows].float()
        if s["weights"] is not None:
            g = g * s["weights"][keep].unsqueeze(1)
        out = torch.zeros(c["vocab"], c["dim"], device=g.device)
        return out.index_add_(0, ids, g) * c["scale"]
    if c["op"] == "dropout":
        f = hip.dropout if own else _dropout
        return {"y": f(s["x"], c["p"], s["seed"], s["step"]),
                "dx": f(s["dy"], c["p"], s["seed"], s["step"])}
    if own:
        return hip.fp8_linear(s["x"], s["packed"], s["bias"])
    q, e = _blocks_of_128(s["x"])
    x = q * _wide(e, c["inner"])
    w = s["W_e4m3"].float() * _wide(s["W_scale"], c["inner"])
    return (x @ w.t() + s["bias"]).to(s["x"].dtype)


# -------------------------------------------------------------------- work
def _touched(n, vocab):
    """How many rows n tokens of the rank-frequency law touch, on average."""
    r = np.arange(1, vocab + 1, dtype=np.float64)
    p = np.log1p(1 / r) / math.log(vocab + 1) * 0.98
    return float(-np.expm1(n * np.log1p(-p)).sum())


def work(case):
    c, z = case, BYTES[case["dtype"]]
    if c["op"] == "lookup":
        b = 8 * c["n"] + z * c["dim"] * (_touched(c["n"], c["vocab"]) + c["n"])
        return {"bytes": b, "flops": c["n"] * c["dim"]}
    if c["op"] in ("bag", "grad"):
        one = c["op"] == "grad" and c["mean_len"] == 1
        n = c["bags"] * (1 if one else max(c["mean_len"] - 0.5, 0.5))
        b = n * (8 + 4 * c["weighted"]) + (0 if one else 8 * c["bags"])
        if c["op"] == "bag":
            b += z * c["dim"] * (_touched(n, c["vocab"]) + c["bags"])
        else:
            b += c["dim"] * (z * c["bags"] + 4 * c["vocab"])
        return {"bytes": b, "flops": 2 * n * c["dim"]}
    if c["op"] == "dropout":
        return {"bytes": 4 * z * c["rows"] * c["cols"],
                "flops": 2 * c["rows"] * c["cols"]}
    m, k, n = c["rows"], c["inner"], c["cols"]
    return {"bytes": z * m * (k + n) + k * n + n * (k + 127) // 128 + 4 * n,
            "flops": 2 * m * k * n}


# ------------------------------------------------------------------- exact
def _exact_bits(n, seed, step):
    """The generator's 16-bit numbers, its 32 x 32 products made of 16-bit
    parts."""
    def high_low(a, k):
        a0, a1, k0, k1 = a & 65535, a >> 16, k & 65535, k >> 16
        mid = (a0 * k0 >> 16) + (a1 * k0 & 65535) + (a0 * k1 & 65535)
        low = (a0 * k0 & 65535) | ((mid & 65535) << 16)
        return a1 * k1 + (a1 * k0 >> 16) + (a0 * k1 >> 16) + (mid >> 16), low

    b = torch.arange(-(-n // 8), device="cuda")
    x, y = b % 2 ** 32, b // 2 ** 32
    z, w = (torch.full_like(b, step % 2 ** 32),
            torch.full_like(b, step // 2 ** 32))
    for r in range(10):
        ka = (seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32
        kb = (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32
        hx, lx = high_low(x, 0xD2511F53)
        hz, lz = high_low(z, 0xCD9E8D57)
        x, y, z, w = hz ^ y ^ ka, lz, hx ^ w ^ kb, lx
    out = torch.empty(b.numel(), 8, dtype=torch.int64, device="cuda")
    for i, v in enumerate((x, y, z, w)):
        out[:, 2 * i], out[:, 2 * i + 1] = v % 65536, v // 65536
    return out.view(-1)[:n]


def _exact_e4m3(x):
    """x [rows, K] in 64 bits as the values that 8 bits hold of it: in each
    block of 128 multiples of 2^(exponent - 3), halves to even, from 2^-9 of
    the block's scale on."""
    rows, n = x.shape
    out = torch.empty_like(x)
    for k in range(0, n, 128):
        b = x[:, k:k + 128]
        top = b.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(top / 448))
        # the logarithm may be off by one at a border
        e = torch.where(torch.exp2(e - 1) * 448 >= top, e - 1, e)
        e = torch.where(torch.exp2(e) * 448 < top, e + 1, e)
        scale = torch.exp2(torch.where(top > 0, e, torch.zeros_like(e)))
        v = b / scale
        power = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
        power = torch.where(torch.exp2(power) > v.abs().clamp(min=2.0 ** -6),
                            power - 1, power)
        power = torch.where(torch.exp2(power + 1) <= v.abs(), power + 1, power)
        unit = torch.exp2(power - 3)
        out[:, k:k + 128] = torch.round(v / unit) * unit * scale
    return out


def exact(case, seed):
    s, c = _inputs(case, seed), case
    if c["op"] == "lookup":
        y = torch.zeros(c["n"], c["dim"], dtype=torch.float64, device="cuda")
        seen = s["ids"] >= 0
        y[seen] = s["table"].double()[s["ids"][seen]] * c["scale"]
        return y
    if c["op"] in ("bag", "grad"):
        at = torch.arange(s["ids"].numel(), device="cuda")
        if s["offsets"] is not None:
            at = torch.repeat_interleave(
                torch.arange(c["bags"], device="cuda"), s["offsets"].diff())
        w = torch.ones(at.numel(), dtype=torch.float64, device="cuda")
        if s["weights"] is not None:
            w = s["weights"].double()
        w = torch.where(s["ids"] >= 0, w, torch.zeros_like(w)) * c["scale"]
        ids = s["ids"].clamp(min=0)
        src, dst, data, size = (ids, at, s["table"], c["bags"]) \
            if c["op"] == "bag" else (at, ids, s["dy"], c["vocab"])
        out = torch.zeros(size, c["dim"], dtype=torch.float64, device="cuda")
        for i in range(0, at.numel(), 1 << 20):
            j = slice(i, i + (1 << 20))
            out.index_add_(0, dst[j], data[src[j]].double() * w[j, None])
        return out
    if c["op"] == "dropout":
        t = int(c["p"] * 65536 + 0.5)
        keep = _exact_bits(c["rows"] * c["cols"], s["seed"], s["step"]) >= t
        keep = keep.view(c["rows"], c["cols"])
        f = torch.where(keep, 65536.0 / (65536 - t), 0.0).double()
        return {"y": s["x"].double() * f, "dx": s["dy"].double() * f}
    x = _exact_e4m3(s["x"].double())
    w = _exact_e4m3(s["W"].double().t().contiguous())
    return x @ w.t().contiguous() + s["bias"].double()
