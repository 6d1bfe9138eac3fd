"""Cases of the ranking operators: rows held in 4 bits with a scale for every 32 of them, their products with queries, the
scores of candidate lists, and log probabilities over scores with their gradient.

A case is a dict of plain values; `op` says which operator it passes through:

  quantize   n rows of d values of a type into 4-bit codes and scales, and back into values of that type
  product    nq queries against all n rows: an nq x n matrix of scores in a type
  score      nq queries against their lists of candidates (CSR) out of n rows: a score for each candidate
  log_probs  log probabilities of given entries, entropy, and the k most likely ones: over the rows of an nq x n
             matrix (lists false) or over lists of candidates (lists true, mean their mean length)
  backward   the gradient of those log probabilities and entropies with respect to the scores

`type` is the type of the rows, of the scores, or of the product; `pad` makes the rows of a matrix that many entries
further apart than they are long.
"""
import math

import torch

own = False  # True: the framework's kernels; False: the plain forms below

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "f64": 8}
DEV = "cuda"


def _c(name, op, type, n, d=0, nq=0, metric="dot", lists=False, mean=0, k=0, temperature=1.0, pad=0, law="normal"):
    c = dict(op=op, type=type, n=n, d=d, nq=nq, metric=metric, lists=lists, mean=mean, k=k, temperature=temperature,
             pad=pad, law=law)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a small collection of odd shape, half precision as an encoder leaves it
        _c("quantize_small_odd", "quantize", "bf16", 1_001, 100),
        # the million descriptors of the benchmark
        _c("quantize_million", "quantize", "f32", 1_000_000, 128, law="counts"),
        # one query of an online service against every row: exhaustive search
        _c("product_one_query", "product", "f32", 1_000_000, 128, nq=1, metric="cosine"),
        # a batch of queries against every row, the exact side of a recall measurement
        _c("product_batch", "product", "bf16", 1_000_000, 128, nq=1_000),
        # long embeddings, both sides large: the arithmetic counts
        _c("product_long_rows", "product", "bf16", 32_771, 2_048, nq=4_099),
        # the quick-start shape: a hundred queries, short lists
        _c("score_few", "score", "f32", 10_000, 128, nq=100, mean=150),
        # the benchmark's ten thousand queries and the candidates that thirty-two tables give them
        _c("score_batch", "score", "f32", 1_000_000, 128, nq=10_000, mean=18_000, metric="cosine", law="counts"),
        # one query's distribution over every row
        _c("log_probs_one_query", "log_probs", "f32", 1_000_000, nq=1, k=10),
        # a batch's distributions over every row, half precision
        _c("log_probs_batch", "log_probs", "bf16", 1_000_000, nq=1_000, k=10),
        # distributions over the candidate lists of the benchmark, and the ten nearest of each
        _c("log_probs_lists", "log_probs", "f32", 1_000_000, nq=10_000, lists=True, mean=18_000, k=10, temperature=0.05),
        # a training step of a query encoder over short lists of hard negatives
        _c("backward_lists", "backward", "f32", 100_000, nq=1_000, lists=True, mean=200, temperature=0.05),
        # the same over every row of an odd collection, half precision
        _c("backward_batch", "backward", "bf16", 200_003, nq=1_000),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "score", "score", "log_probs", "log_probs", "backward"])
    law = rng.choice(["normal", "counts", "wide"])
    metric = rng.choice(["dot", "cosine", "euclidean"])
    pad = rng.choice([0, 0, 1, 8, 13])
    if op == "quantize":
        d = _log(rng, 1, 4_096)
        return _c(None, op, rng.choice(["f32", "f32", "f16", "bf16", "f64"]), _log(rng, 1, 64_000_000 // d), d, law="normal", pad=pad)
    if op == "product":
        d = _log(rng, 1, 4_096)
        n = _log(rng, 1, min(1_000_000, 128_000_000 // d))
        nq = _log(rng, 1, max(1, min(5_000, 500_000_000 // n)))
        return _c(None, op, rng.choice(["f32", "f16", "bf16"]), n, d, nq=nq, metric="dot", pad=pad)
    if op == "score":
        d = _log(rng, 1, 2_048)
        n = _log(rng, 2, min(1_000_000, 128_000_000 // d))
        mean = _log(rng, 1, max(1, n // 4))
        nq = _log(rng, 1, max(1, min(10_000, 10_000_000_000 // (mean * max(d, 64)))))
        return _c(None, op, rng.choice(["f32", "f16", "bf16", "f64"]), n, d, nq=nq, mean=mean, metric=metric, law=law)
    lists = rng.random() < 0.5
    k = rng.choice([0, 1, 5, 10, 32, 100]) if op == "log_probs" else 0
    t = rng.choice([1.0, 0.05, 0.3])
    kind = rng.choice(["f32", "f16", "bf16"])
    n = _log(rng, 2, 1_000_000)
    if lists:
        mean = _log(rng, 1, max(1, n // 4))
        return _c(None, op, kind, n, nq=_log(rng, 1, max(1, min(20_000, 100_000_000 // mean))), lists=True, mean=mean, k=k, temperature=t)
    return _c(None, op, kind, n, nq=_log(rng, 1, max(1, min(20_000, 300_000_000 // n))), k=k, temperature=t, pad=pad)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _rows(gen, n, d, law, dtype):
    """Vectors: standard normals, non-negative counts with a heavy tail, or normals of widely different magnitudes."""
    if law == "counts":
        z = torch.randn(n, d, generator=gen, device=DEV)
        x = (20.0 * z * z).round_().clamp_(0, 255)
    else:
        x = torch.randn(n, d, generator=gen, device=DEV)
        if law == "wide":
            x *= torch.exp2(torch.randint(-12, 13, (n, d), generator=gen, device=DEV).float())
    return x.to(dtype)


def _apart(x, pad):
    """The same matrix with its rows `pad` entries further apart."""
    if not pad:
        return x
    y = x.new_zeros(x.shape[0], x.shape[1] + pad)
    y[:, :x.shape[1]] = x
    return y[:, :x.shape[1]]


def _lists(gen, nq, n, mean):
    """Ascending lists of distinct ids below n, of very different lengths around a mean, some of them empty.  A case has the
    same lengths whatever the seed: outputs are as long as the lists."""
    u = torch.rand(nq, generator=torch.Generator(device=DEV).manual_seed(7 * nq + mean), device=DEV)
    length = (-torch.log1p(-u.clamp(max=0.999)) * mean).long().clamp_(max=max(1, min(n, 4 * mean)))
    offsets = torch.zeros(nq + 1, dtype=torch.int64, device=DEV)
    offsets[1:] = torch.cumsum(length, 0)
    total = int(offsets[-1])
    q = torch.repeat_interleave(torch.arange(nq, device=DEV), length, output_size=total)
    step = (n // length.clamp(min=1))[q]
    at = torch.arange(total, device=DEV) - offsets[q]
    ids = at * step + (torch.rand(total, generator=gen, device=DEV, dtype=torch.float64) * step).long().clamp_(max=n)
    return ids.clamp_(max=n - 1).to(torch.int32), offsets


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = TYPES[c["type"]]
    s = {"case": c}
    if c["op"] == "quantize":
        s["X"] = _apart(_rows(gen, c["n"], c["d"], c["law"], dtype), c["pad"])
        return s
    if c["op"] in ("product", "score"):
        # the program keeps its rows in 4 bits and no longer has the others
        s["codes"], s["scales"], s["norms"] = _pack(_rows(gen, c["n"], c["d"], c["law"], torch.float32))
        s["Q"] = _rows(gen, c["nq"], c["d"], c["law"], dtype if c["op"] == "score" else torch.float32)
        if c["op"] == "score":
            s["ids"], s["offsets"] = _lists(gen, c["nq"], c["n"], c["mean"])
        else:
            s["Q"] = _apart(s["Q"], c["pad"])
        return s
    nq, n = c["nq"], c["n"]
    spread = 2.0 * min(1.0, 2.0 * c["temperature"])  # cosines where the temperature is low
    if c["lists"]:
        s["ids"], s["offsets"] = _lists(gen, nq, n, c["mean"])
        s["scores"] = (torch.randn(s["ids"].shape[0], generator=gen, device=DEV) * spread).to(dtype)
        if s["ids"].shape[0]:  # given ids: one of the list, or any
            at = s["offsets"][:-1] + (torch.rand(nq, generator=gen, device=DEV) * (s["offsets"][1:] - s["offsets"][:-1])).long()
            near = s["ids"][at.clamp(max=s["ids"].shape[0] - 1)].long()
        else:
            near = torch.zeros(nq, dtype=torch.int64, device=DEV)
        far = torch.randint(0, n, (nq,), generator=gen, device=DEV)
        s["targets"] = torch.where(torch.rand(nq, generator=gen, device=DEV) < 0.9, near, far)
    else:
        x = torch.empty(nq, n + c["pad"], dtype=dtype, device=DEV)[:, :n]
        x.copy_(torch.randn(nq, n, generator=gen, device=DEV, dtype=dtype if dtype != torch.float64 else torch.float32)).mul_(spread)
        masked = torch.rand(n, generator=gen, device=DEV) < 0.02  # rows that were deleted, or that a filter takes out
        x[:, masked] = -math.inf
        if nq > 4:
            x[nq // 2] = -math.inf  # a query for which the filter leaves nothing
        s["scores"] = x
        s["targets"] = torch.randint(0, n, (nq,), generator=gen, device=DEV)
        s["targets"][torch.rand(nq, generator=gen, device=DEV) < 0.02] = -1
    if c["op"] == "backward":  # what the forward pass left, and what comes from the loss
        r = _log_probs(s["scores"], s["targets"], s.get("ids"), s.get("offsets"), c["temperature"], 0)
        s["lse"], s["entropy"] = r[2], r[1]
        s["grad_log_probs"] = torch.randn(nq, generator=gen, device=DEV)
        s["grad_entropy"] = 0.1 * torch.randn(nq, generator=gen, device=DEV)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # a value on one goes to the code that is even


def _quantize(X):
    """Codes and scale exponents of rows: blocks of 32, scale 2^(floor(log2 max) - 2), values rounded to the nearest of the
    levels, ties to the even code, larger ones to 6.  (codes [n, blocks, 32], exponents [n, blocks])"""
    n, d = X.shape
    groups = -(-d // 128)
    x = torch.nn.functional.pad(X if X.dtype == torch.float64 else X.float(), (0, groups * 128 - d)).view(n, groups * 4, 32)
    top = x.abs().amax(2)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    y = torch.ldexp(x, -e[:, :, None].to(x.dtype))
    mid = torch.tensor(_MIDDLES, dtype=x.dtype, device=x.device)
    a = y.abs()
    low, high = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)
    code = torch.where(low % 2 == 0, low, high).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    return code, e


def _pack(X):
    """Codes two to a byte, the first in the low half, rows padded to 128 values; scale bytes 127 + exponent in tiles of 128 rows
    by 128 values [tile, group, row % 32, row // 32 % 4, block % 4]; squared norms of what is held."""
    n, d = X.shape
    code, e = _quantize(X)
    codes = code.view(n, -1, 2)
    codes = codes[:, :, 0] | (codes[:, :, 1] << 4)
    tiles = -(-n // 128)
    b = torch.zeros(tiles * 128, e.shape[1], dtype=torch.uint8, device=X.device)
    b[:n] = (e + 127).to(torch.uint8)
    scales = b.view(tiles, 4, 32, -1, 4).permute(0, 3, 2, 1, 4).contiguous()
    v = _decode(code, e).view(n, -1)
    return codes.contiguous(), scales, (v * v).sum(1)


def _decode(code, e):
    v = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device=code.device)[code.long()]
    return torch.ldexp(v, e[:, :, None].float())


def _unpack(codes, scales, n):
    code = torch.stack((codes & 15, codes >> 4), 2).view(n, -1, 32)
    e = scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:n].int() - 127
    return _decode(code, e).view(n, -1)


def _metric(dot, metric, q2, x2):
    """Dot products, cosines, or negative squared distances from dot products and squared norms."""
    if metric == "cosine":
        s = (q2 * x2).sqrt()
        return torch.where(s > 0, dot / s, torch.zeros_like(dot))
    if metric == "euclidean":
        return 2 * dot - q2 - x2
    return dot


def _product(s):
    c = s["case"]
    x = _unpack(s["codes"], s["scales"], c["n"])
    q = _decode(*_quantize(s["Q"])).view(c["nq"], -1)
    dot = q @ x.T
    return _metric(dot, c["metric"], (q * q).sum(1)[:, None], s["norms"][None, :]).to(TYPES[c["type"]])


_CHUNK = 8_000_000  # candidates whose rows are gathered at a time


def _score(s):
    c = s["case"]
    q, d = s["Q"].float(), c["d"]
    x = _unpack(s["codes"], s["scales"], c["n"])[:, :d]
    ids, offsets = s["ids"].long(), s["offsets"]
    owner = torch.repeat_interleave(torch.arange(c["nq"], device=DEV), offsets[1:] - offsets[:-1], output_size=ids.shape[0])
    step = max(1, min(ids.shape[0], _CHUNK * 128 // max(d, 32)))
    dot = torch.cat([(x[i] * q[o]).sum(1) for i, o in zip(ids.split(step), owner.split(step))]) if ids.shape[0] else q.new_zeros(0)
    return _metric(dot, c["metric"], (q * q).sum(1)[owner], s["norms"][ids])


def _dense(scores, ids, offsets):
    """Lists as rows of a matrix, -inf behind their ends, and whether an entry is one of its list."""
    length = offsets[1:] - offsets[:-1]
    at = torch.arange(max(1, int(length.max())), device=DEV)[None, :]
    real = at < length[:, None]
    place = torch.where(real, offsets[:-1, None] + at, torch.zeros_like(at))
    if not scores.shape[0]:
        return torch.full(real.shape, -math.inf, dtype=scores.dtype, device=DEV), place, real
    return torch.where(real, scores[place], torch.full((), -math.inf, dtype=scores.dtype, device=DEV)), place, real


def _log_probs(scores, targets, ids, offsets, temperature, k):
    """(log probability of the target, entropy, log of the sum of exponentials, log probabilities and ids of the k most likely)"""
    if offsets is not None:
        x, place, real = _dense(scores, ids, offsets)
        names = ids[place] if ids.shape[0] else place.int()
        hit = real & (names == targets[:, None])
    else:
        x, names = scores, None
    z = x.float() / temperature
    top = z.amax(1, keepdim=True)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(z - base)
    total = p.sum(1, keepdim=True)
    lse = (base + torch.log(total))[:, 0]
    weighted = torch.where(p > 0, p * (z - base), torch.zeros_like(p)).sum(1)
    entropy = torch.where(lse == -math.inf, torch.zeros_like(lse), torch.log(total[:, 0]) - weighted / total[:, 0])
    del p
    if offsets is not None:
        mine = torch.where(hit, z, torch.full_like(z, -math.inf)).amax(1)
    else:
        inside = (targets >= 0) & (targets < z.shape[1])
        mine = torch.where(inside, z.gather(1, targets.clamp(0, z.shape[1] - 1)[:, None])[:, 0], torch.full_like(lse, -math.inf))
    logp = torch.where(mine == -math.inf, mine, mine - lse)
    if not k:
        return logp, entropy, lse
    # the largest first, the lowest place among equal ones: one whole number for each entry that says both
    bits = (x.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    order = order * 4294967296 + (4294967295 - torch.arange(x.shape[1], device=DEV))[None, :]
    kk = min(k, x.shape[1])
    at = 4294967295 - (torch.topk(order, kk, dim=1).values & 4294967295)
    del order, bits
    zt = z.gather(1, at)
    found = zt > -math.inf
    value = torch.where(found, zt - lse[:, None], zt)
    name = at.int() if names is None else names.gather(1, at)
    name = torch.where(found, name, torch.full_like(name, -1))
    pad = (0, k - kk)
    return (logp, entropy, lse, torch.nn.functional.pad(value, pad, value=-math.inf), torch.nn.functional.pad(name, pad, value=-1))


def _backward(s):
    c = s["case"]
    scores, targets = s["scores"], s["targets"][:, None]
    if c["lists"]:
        x, place, real = _dense(scores, s["ids"], s["offsets"])
        hit = real & (s["ids"][place] == targets) if scores.shape[0] else real
    else:
        x, hit = scores, torch.arange(scores.shape[1], device=DEV)[None, :] == targets
    z = x.float() / c["temperature"]
    lse, h = s["lse"][:, None], s["entropy"][:, None]
    g, ge = s["grad_log_probs"][:, None], s["grad_entropy"][:, None]
    alive = z > -math.inf
    logp = torch.where(alive, z - lse, torch.zeros_like(z))
    p = torch.where(alive, torch.exp(logp), torch.zeros_like(z))
    g = torch.where((hit & alive).any(1, keepdim=True), g, torch.zeros_like(g))  # an entry of no probability stays where it is
    grad = ((hit & alive) * g - g * p - ge * p * (logp + h)) / c["temperature"]
    grad = grad.to(scores.dtype)
    return grad[real] if c["lists"] else grad


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        import culsh_b200 as culsh

        if c["op"] == "quantize":
            rows = culsh.MXRows(state["X"])
            return rows.dequantize(TYPES[c["type"]]), rows.norms
        if c["op"] == "product":
            rows = culsh.MXRows.from_parts(state["codes"], state["scales"], state["norms"], c["d"])
            return rows.product(state["Q"], metric=c["metric"], dtype=TYPES[c["type"]])
        if c["op"] == "score":
            rows = culsh.MXRows.from_parts(state["codes"], state["scales"], state["norms"], c["d"])
            return rows.score(state["Q"], (state["ids"], state["offsets"]), metric=c["metric"])
        lists = (state["ids"], state["offsets"]) if c["lists"] else None
        if c["op"] == "log_probs":
            r = culsh.log_probs(state["scores"], state["targets"], lists, top_k=c["k"], temperature=c["temperature"])
            return tuple(r) if c["k"] else tuple(r)[:3]
        return culsh.log_probs_backward(state["scores"], state["targets"], state["lse"], state["entropy"], state["grad_log_probs"],
                                        state["grad_entropy"], lists, temperature=c["temperature"])
    if c["op"] == "quantize":
        values = _decode(*_quantize(state["X"])).view(c["n"], -1)
        return values[:, :c["d"]].to(TYPES[c["type"]]).contiguous(), (values * values).sum(1)
    if c["op"] == "product":
        return _product(state)
    if c["op"] == "score":
        return _score(state)
    if c["op"] == "log_probs":
        return _log_probs(state["scores"], state["targets"], state.get("ids"), state.get("offsets"), c["temperature"], c["k"])
    return _backward(state)


def work(case):
    c, z = case, SIZE[case["type"]]
    n, d, nq = c["n"], c["d"], c["nq"]
    held = n * (-(-d // 32)) * 17 + 4 * n  # 32 codes and a scale are 17 bytes; a norm
    if c["op"] == "quantize":
        return {"bytes": 2 * n * d * z + 4 * n, "flops": 6 * n * d}
    if c["op"] == "product":
        return {"bytes": held + 4 * nq * d + nq * n * z, "flops": 2 * nq * n * d}
    if c["op"] == "score":
        total = nq * c["mean"]
        return {"bytes": min(held, total * (held // n)) + nq * d * z + 8 * total + 8 * nq, "flops": 2 * total * d}
    entries = nq * (c["mean"] if c["lists"] else n)
    if c["op"] == "log_probs":
        return {"bytes": entries * z + nq * (20 + 8 * c["k"]), "flops": 5 * entries}
    return {"bytes": 2 * entries * z + 24 * nq, "flops": 8 * entries}


# ---- in 64 bits, from the definitions -------------------------------------------------------------------------------
def _held64(codes, scales, n, d):
    """Values that packed rows stand for: sign, two bits of exponent, one of fraction; times the block's power of two."""
    c = codes.long()
    c = torch.cat((c % 16, c // 16), 1).view(n, 2, -1).transpose(1, 2).reshape(n, -1)
    exponent, fraction = c // 2 % 4, (c % 2).double()
    size = torch.where(exponent == 0, fraction / 2, (1 + fraction / 2) * 2.0 ** (exponent.double() - 1))
    row, block = torch.arange(n, device=DEV)[:, None], torch.arange(codes.shape[1] // 16, device=DEV)[None, :]
    byte = scales[row // 128, block // 4, row % 32, row // 32 % 4, block % 4]
    scale = 2.0 ** (byte.double() - 127)
    return (torch.where(c >= 8, -size, size) * scale.repeat_interleave(32, 1))[:, :d]


def _nearest64(X):
    """Values of rows by distance to every level: the nearest, the even code of two as near."""
    n, d = X.shape
    x = torch.zeros(n, -(-d // 32) * 32, dtype=torch.float64, device=DEV)
    x[:, :d] = X
    out = torch.empty_like(x)
    level = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    even_first = [0, 2, 4, 6, 1, 3, 5, 7]
    for at in range(0, n, 100_000):
        y = x[at:at + 100_000].view(-1, 32)
        top = y.abs().amax(1, keepdim=True)
        low = torch.log2(torch.where(top > 0, top, torch.ones_like(top))).round()
        low = torch.where(torch.exp2(low) > top, low - 1, low)  # the largest power of two that is no more than the largest value
        unit = torch.exp2((low - 2).clamp(-127, 127))
        y = y / unit
        best = torch.full_like(y, math.inf)
        value = torch.zeros_like(y)
        for i in even_first:
            far = (y.abs() - level[i]).abs()
            value = torch.where(far < best, level[i], value)
            best = torch.minimum(far, best)
        out[at:at + 100_000] = (torch.copysign(value, y) * unit).view(-1, out.shape[1])
    return out[:, :d]


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    n, d, nq = c["n"], c["d"], c["nq"]
    if c["op"] == "quantize":
        v = _nearest64(s["X"].double())
        return v, (v * v).sum(1)
    if c["op"] == "product":
        x, q = _held64(s["codes"], s["scales"], n, d), _nearest64(s["Q"].double())
        dot = q @ x.T
        q2, x2 = (q * q).sum(1)[:, None], (x * x).sum(1)[None, :]
        if c["metric"] == "cosine":
            return torch.nan_to_num(dot / torch.sqrt(q2) / torch.sqrt(x2), nan=0.0)
        return dot if c["metric"] == "dot" else -(q2 + x2 - 2 * dot)
    if c["op"] == "score":
        x, q = _held64(s["codes"], s["scales"], n, d), s["Q"].double()
        out = torch.empty(s["ids"].shape[0], dtype=torch.float64, device=DEV)
        x2, q2 = (x * x).sum(1), (q * q).sum(1)
        ends = s["offsets"].tolist()
        for i in range(nq):
            mine = s["ids"][ends[i]:ends[i + 1]].long()
            v = x[mine] @ q[i]
            if c["metric"] == "cosine":
                v = torch.nan_to_num(v / torch.sqrt(q2[i]) / torch.sqrt(x2[mine]), nan=0.0)
            elif c["metric"] == "euclidean":
                v = -(q2[i] + x2[mine] - 2 * v)
            out[ends[i]:ends[i + 1]] = v
        return out
    ends = s["offsets"].tolist() if c["lists"] else None
    few = torch.zeros(nq, 3, dtype=torch.float64, device=DEV)
    best = torch.full((nq, c["k"]), -math.inf, dtype=torch.float64, device=DEV)
    grads = torch.zeros(s["scores"].shape, dtype=torch.float64, device=DEV) if c["op"] == "backward" else None
    targets = s["targets"].tolist()
    if c["op"] == "backward":
        g1, g2 = s["grad_log_probs"].double().tolist(), s["grad_entropy"].double().tolist()
    for i in range(nq):
        z = (s["scores"][ends[i]:ends[i + 1]] if c["lists"] else s["scores"][i]).double() / c["temperature"]
        lse = torch.logsumexp(z, 0) if z.numel() else torch.tensor(-math.inf, dtype=torch.float64, device=DEV)
        logp = z - lse
        p = torch.nan_to_num(torch.exp(logp), nan=0.0)
        plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
        h = -plogp.sum()
        if c["lists"]:
            hit = torch.nonzero(s["ids"][ends[i]:ends[i + 1]] == targets[i])[:, 0]
        else:
            hit = torch.arange(targets[i], targets[i] + 1, device=DEV) if targets[i] >= 0 else torch.arange(0, device=DEV)
        lp = logp[hit].sum() if hit.numel() and torch.isfinite(z[hit]).all() else torch.tensor(-math.inf, dtype=torch.float64, device=DEV)
        if c["op"] == "backward":
            g = -g2[i] * (plogp + p * h)
            if torch.isfinite(lp):
                g -= g1[i] * p
                g[hit] += g1[i]
            (grads[ends[i]:ends[i + 1]] if c["lists"] else grads[i]).copy_(g / c["temperature"])
            continue
        few[i, 0], few[i, 1], few[i, 2] = lp, h, lse
        kk = min(c["k"], z.numel())
        if kk:
            best[i, :kk] = torch.nan_to_num(torch.topk(logp, kk).values, nan=-math.inf, neginf=-math.inf)
    if c["op"] == "backward":
        return grads
    r = (few[:, 0].contiguous(), few[:, 1].contiguous(), few[:, 2].contiguous())
    return r + (best, None) if c["k"] else r
