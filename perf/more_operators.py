"""Cases of rows held in 8 bits, and of the loss that an encoder is trained with against every row.

A case is a dict of plain values; `op` says which operator it passes through:

  quantize   n rows of d values of a type into 8-bit integers with a scale for each row, and back into values of that type
  product    nq queries, held in 8 bits as well, against all n rows: an nq x n matrix of scores in a type
  score      nq queries against their lists of candidates (CSR) out of n rows: a score for each candidate
  loss       the softmax cross entropy of nq queries over all n rows, whose scores are not kept: losses and logs of the sums
  gradient   its gradient with respect to the queries and the rows

`type` is the type of the rows, of the scores, or of both sides of the loss; `pad` makes the rows of a matrix that many entries
further apart than they are long.  `bias`: a term for each row is added to its scores: the log of how often it was drawn, taken
off, and -inf for rows that are masked.
"""
import math

import torch

own = False  # True: the framework's kernels; False: the plain forms below

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "f64": 8}
DEV = "cuda"


def _c(name, op, type, n, d, nq=0, metric="dot", mean=0, temperature=1.0, bias=False, pad=0, law="normal"):
    c = dict(op=op, type=type, n=n, d=d, nq=nq, metric=metric, mean=mean, temperature=temperature, bias=bias, pad=pad, law=law)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # a small collection of odd shape, half precision as an encoder leaves it
        _c("rows8_small_odd", "quantize", "bf16", 1_001, 100),
        # the million descriptors of the benchmark
        _c("rows8_million", "quantize", "f32", 1_000_000, 128, law="counts"),
        # one query of an online service against every row: exhaustive search
        _c("product8_one_query", "product", "f32", 1_000_000, 128, nq=1, metric="cosine"),
        # a batch of queries against every row, the exact side of a recall measurement
        _c("product8_batch", "product", "bf16", 1_000_000, 128, nq=1_000),
        # long embeddings, or a layer of an encoder: both sides large, the arithmetic counts
        _c("product8_long_rows", "product", "bf16", 32_771, 2_048, nq=4_099),
        # the quick-start shape: a hundred queries, short lists
        _c("score8_few", "score", "f32", 10_000, 128, nq=100, mean=150),
        # the benchmark's ten thousand queries and candidates of a few tables
        _c("score8_batch", "score", "f32", 1_000_000, 128, nq=10_000, mean=1_500, metric="cosine", law="counts"),
        # a small encoder's validation loss, single precision, with the correction for rows that are drawn more often
        _c("loss_small", "loss", "f32", 1_000, 100, nq=64, temperature=0.05, bias=True),
        # a training batch against the million rows of the benchmark
        _c("loss_batch", "loss", "bf16", 1_000_000, 128, nq=4_096, temperature=0.05),
        # the gradient of a small batch
        _c("gradient_small", "gradient", "f32", 1_000, 100, nq=64, temperature=0.05, bias=True),
        # the gradient of a training batch, for the encoder and for the rows
        _c("gradient_batch", "gradient", "bf16", 1_000_000, 128, nq=4_096, temperature=0.05),
        # long embeddings, odd numbers of both sides, half precision
        _c("gradient_long", "gradient", "f16", 32_771, 2_048, nq=4_099, temperature=0.05),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "score", "loss", "loss", "gradient", "gradient", "gradient"])
    pad = rng.choice([0, 0, 1, 8, 13])
    metric = rng.choice(["dot", "cosine", "euclidean"])
    if op == "quantize":
        d = _log(rng, 1, 4_096)
        return _c(None, op, rng.choice(["f32", "f32", "f16", "bf16", "f64"]), _log(rng, 1, 64_000_000 // d), d, law=rng.choice(["normal", "wide"]), pad=pad)
    if op == "product":
        d = _log(rng, 1, 4_096)
        n = _log(rng, 1, min(1_000_000, 128_000_000 // d))
        nq = _log(rng, 1, max(1, min(5_000, 500_000_000 // n)))
        return _c(None, op, rng.choice(["f32", "f16", "bf16"]), n, d, nq=nq, metric=metric, pad=pad)
    if op == "score":
        d = _log(rng, 1, 2_048)
        n = _log(rng, 2, min(1_000_000, 128_000_000 // d))
        mean = _log(rng, 1, max(1, n // 4))
        nq = _log(rng, 1, max(1, min(10_000, 1_500_000_000 // (mean * max(d, 64)))))
        return _c(None, op, rng.choice(["f32", "f16", "bf16", "f64"]), n, d, nq=nq, mean=mean, metric=metric, law=rng.choice(["normal", "counts"]))
    d = _log(rng, 1, 2_048)
    n = _log(rng, 1, min(1_000_000, 128_000_000 // d))
    kind = rng.choice(["f32", "f16", "bf16"])
    most = 500_000_000_000 // (8 if kind == "f32" else 1)
    nq = _log(rng, 1, max(1, min(5_000, most // (n * max(d, 64)))))
    return _c(None, op, kind, n, d, nq=nq, temperature=rng.choice([1.0, 0.05, 0.3]), bias=rng.random() < 0.3, pad=pad)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _rows(gen, n, d, law, dtype):
    """Vectors: standard normals, non-negative counts with a heavy tail, or normals whose rows are of widely different magnitudes."""
    x = torch.randn(n, d, generator=gen, device=DEV)
    if law == "counts":
        x = (20.0 * x * x).round_().clamp_(0, 255)
    elif law == "wide":
        x *= torch.exp2(torch.randint(-12, 13, (n, 1), generator=gen, device=DEV).float())
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
    dtype, n, d, nq = TYPES[c["type"]], c["n"], c["d"], c["nq"]
    s = {"case": c}
    if c["op"] == "quantize":
        s["X"] = _apart(_rows(gen, n, d, c["law"], dtype), c["pad"])
        return s
    if c["op"] in ("product", "score"):
        # the program keeps its rows in 8 bits and no longer has the others
        s["codes"], s["scales"], s["squares"] = _pack(_rows(gen, n, d, c["law"], torch.float32))
        s["Q"] = _rows(gen, nq, d, c["law"], dtype if c["op"] == "score" else torch.float32)
        if c["op"] == "score":
            s["ids"], s["offsets"] = _lists(gen, nq, n, c["mean"])
        else:
            s["Q"] = _apart(s["Q"], c["pad"])
        return s
    # embeddings of length 1, each query a copy of the row that it should find under 2.5 times as much noise, as early in training;
    # a few queries have no target
    X = torch.nn.functional.normalize(torch.randn(n, d, generator=gen, device=DEV))
    targets = torch.randint(0, n, (nq,), generator=gen, device=DEV)
    Q = torch.nn.functional.normalize(X[targets] + torch.randn(nq, d, generator=gen, device=DEV) * (2.5 / d ** 0.5))
    targets[torch.rand(nq, generator=gen, device=DEV) < 0.02] = -1
    s["Q"], s["X"], s["targets"], s["bias"] = _apart(Q.to(dtype), c["pad"]), _apart(X.to(dtype), c["pad"]), targets, None
    if c["bias"]:
        s["bias"] = -torch.log(0.1 + torch.rand(n, generator=gen, device=DEV))
        s["bias"][torch.rand(n, generator=gen, device=DEV) < 0.02] = -math.inf
    if c["op"] == "gradient":  # what the forward pass left, and what comes from the loss
        s["losses"], s["lse"], s["lse_low"] = _loss(s)
        mean = 1 if c["type"] == "f16" else nq  # of the mean loss; in half precision scaled up, as its range demands
        s["grad_losses"] = (1.0 + 0.2 * torch.randn(nq, generator=gen, device=DEV)) / mean
        s["grad_lse"] = 0.01 * torch.randn(nq, generator=gen, device=DEV) / mean
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _quantize(X):
    """Codes of rows and their scales: scale = largest magnitude / 127 in 32 bits, codes the nearest whole numbers to x / scale,
    ties to the even one.  The quotients are next to borders now and then: 64 bits."""
    x = X.double()
    scale = (x.abs().amax(1) / 127).float().clamp(min=2.0 ** -126)
    return torch.round(x / scale.double()[:, None]).to(torch.int8), scale


def _pack(X):
    """Codes in rows padded with zeros to a multiple of 16, scales, and the sums of the codes' squares."""
    codes, scales = _quantize(X)
    squares = (codes.int() * codes.int()).sum(1).to(torch.int32)
    return torch.nn.functional.pad(codes, (0, -X.shape[1] % 16)), scales, squares


def _metric(dot, metric, q_scale, q2, x_scale, x2):
    """Scores from whole numbers: dot products of codes, the scales, and the sums of the codes' squares."""
    if metric == "cosine":
        s = torch.sqrt(q2.float()) * torch.sqrt(x2.float())
        return torch.where(s > 0, dot / s, torch.zeros_like(dot))
    v = dot * (q_scale * x_scale)
    if metric == "euclidean":
        return 2 * v - q2.float() * (q_scale * q_scale) - x2.float() * (x_scale * x_scale)
    return v


def _product(s):
    c = s["case"]
    q_codes, q_scale = _quantize(s["Q"])
    q2 = (q_codes.int() * q_codes.int()).sum(1)
    dot = q_codes.float() @ s["codes"][:, :c["d"]].float().T
    return _metric(dot, c["metric"], q_scale[:, None], q2[:, None], s["scales"][None, :], s["squares"][None, :]).to(TYPES[c["type"]])


def _score(s):
    c = s["case"]
    q_codes, q_scale = _quantize(s["Q"])
    q2 = (q_codes.int() * q_codes.int()).sum(1)
    ids, offsets = s["ids"].long(), s["offsets"]
    owner = torch.repeat_interleave(torch.arange(c["nq"], device=DEV), offsets[1:] - offsets[:-1], output_size=ids.shape[0])
    dot = (s["codes"][:, :c["d"]].float()[ids] * q_codes.float()[owner]).sum(1)
    return _metric(dot, c["metric"], q_scale[owner], q2[owner], s["scales"][ids], s["squares"][ids])


def _scores(s):
    """Scores of every row by the temperature, and the rows' terms, [nq, n] in 32 bits."""
    z = s["Q"].float() @ s["X"].float().T
    z /= s["case"]["temperature"]
    if s["bias"] is not None:
        z += s["bias"]
    return z


def _target(s):
    """Targets as columns, and whether there is one."""
    t = s["targets"]
    real = (t >= 0) & (t < s["case"]["n"])
    return torch.where(real, t, torch.zeros_like(t))[:, None], real


def _loss(s):
    """(losses, logs of the sums, what these leave behind their last bits)"""
    z = _scores(s)
    at, real = _target(s)
    mine = z.gather(1, at)[:, 0]
    top = z.amax(1)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    z -= base[:, None]
    lse = base.double() + torch.log(z.exp_().sum(1).double())
    losses = torch.where(real, lse - mine.double(), torch.zeros_like(lse))
    losses = torch.where(real & (mine == -math.inf), torch.full_like(lse, math.inf), losses)
    high = lse.float()
    low = torch.where(torch.isfinite(lse), lse - high.double(), torch.zeros_like(lse))
    return losses.float(), high, low.float()


def _gradient(s):
    t = s["case"]["temperature"]
    z = _scores(s)
    z -= s["lse"][:, None]
    z -= s["lse_low"][:, None]
    p = z.exp_()
    p[s["lse"] == -math.inf] = 0
    at, real = _target(s)
    g = torch.where(real & torch.isfinite(s["losses"]), s["grad_losses"], torch.zeros_like(s["lse"]))
    p *= (g + s["grad_lse"])[:, None]
    p.scatter_add_(1, at, -g[:, None])
    return ((p @ s["X"].float()) / t).to(s["Q"].dtype), ((p.T @ s["Q"].float()) / t).to(s["X"].dtype)


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        import culsh_b200 as culsh

        if c["op"] == "quantize":
            rows = culsh.Int8Rows(state["X"])
            return rows.dequantize(TYPES[c["type"]]), rows.scales, rows.squares
        if c["op"] in ("product", "score"):
            rows = culsh.Int8Rows.from_parts(state["codes"], state["scales"], state["squares"], c["d"])
            if c["op"] == "product":
                return rows.product(state["Q"], metric=c["metric"], dtype=TYPES[c["type"]])
            return rows.score(state["Q"], (state["ids"], state["offsets"]), metric=c["metric"])
        if c["op"] == "loss":
            return tuple(culsh.cross_entropy(state["Q"], state["X"], state["targets"], state["bias"], temperature=c["temperature"]))[:2]
        result = culsh.CrossEntropy(state["losses"], state["lse"], state["lse_low"])
        return culsh.cross_entropy_backward(state["Q"], state["X"], state["targets"], result, state["grad_losses"], state["grad_lse"],
                                            state["bias"], temperature=c["temperature"])
    if c["op"] == "quantize":
        codes, scale = _quantize(state["X"])
        values = codes.double() * scale.double()[:, None]
        return values.to(TYPES[c["type"]]), scale, (codes.int() * codes.int()).sum(1).to(torch.int32)
    if c["op"] == "product":
        return _product(state)
    if c["op"] == "score":
        return _score(state)
    if c["op"] == "loss":
        return _loss(state)[:2]
    return _gradient(state)


def work(case):
    c, z = case, SIZE[case["type"]]
    n, d, nq = c["n"], c["d"], c["nq"]
    held = n * (16 * -(-d // 16) + 8)  # codes, a scale and a sum of squares
    if c["op"] == "quantize":
        return {"bytes": 2 * n * d * z + 8 * n, "flops": 4 * n * d}
    if c["op"] == "product":
        return {"bytes": held + 4 * nq * d + nq * n * z, "flops": 2 * nq * n * d}
    if c["op"] == "score":
        total = nq * c["mean"]
        return {"bytes": min(held, total * (held // n)) + nq * d * z + 8 * total + 8 * nq, "flops": 2 * total * d}
    both = (n + nq) * d * z + (4 * n if c["bias"] else 0)
    if c["op"] == "loss":
        return {"bytes": both + 16 * nq, "flops": 2 * nq * n * d + 4 * nq * n}
    return {"bytes": 2 * both + 32 * nq, "flops": 6 * nq * n * d + 4 * nq * n}


# ---- in 64 bits, from the definitions -------------------------------------------------------------------------------
def _held64(X):
    """What rows in 8 bits stand for: whole numbers by distance to both neighbours, and scales."""
    v = X.double()
    scale = (v.abs().amax(1) / 127).float().clamp(min=2.0 ** -126).double()
    y = v / scale[:, None]
    low = torch.floor(y)
    up = (y - low > 0.5) | ((y - low == 0.5) & (torch.remainder(low, 2) == 1))
    return torch.where(up, low + 1, low), scale


def _metric64(dot, metric, q2, x2):
    if metric == "cosine":
        return torch.nan_to_num(dot / torch.sqrt(q2) / torch.sqrt(x2), nan=0.0)
    return dot if metric == "dot" else -(q2 + x2 - 2 * dot)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    n, d, nq, t = c["n"], c["d"], c["nq"], c["temperature"]
    if c["op"] == "quantize":
        whole, scale = _held64(s["X"])
        return whole * scale[:, None], scale, (whole * whole).sum(1).to(torch.int32)
    if c["op"] in ("product", "score"):
        q, q_scale = _held64(s["Q"])
        q *= q_scale[:, None]
        x = s["codes"][:, :d].double() * s["scales"].double()[:, None]
        q2, x2 = (q * q).sum(1), (x * x).sum(1)
        if c["op"] == "product":
            if nq * n > 2_000_000_000:
                return None
            return _metric64(q @ x.T, c["metric"], q2[:, None], x2[None, :])
        out = torch.empty(s["ids"].shape[0], dtype=torch.float64, device=DEV)
        ends = s["offsets"].tolist()
        for i in range(nq):
            mine = s["ids"][ends[i]:ends[i + 1]].long()
            out[ends[i]:ends[i + 1]] = _metric64(x[mine] @ q[i], c["metric"], q2[i], x2[mine])
        return out
    Q, X = s["Q"].double(), s["X"].double()
    bias = torch.zeros(n, dtype=torch.float64, device=DEV) if s["bias"] is None else s["bias"].double()
    losses, lses = torch.zeros(nq, dtype=torch.float64, device=DEV), torch.empty(nq, dtype=torch.float64, device=DEV)
    grad_Q, grad_X = torch.zeros_like(Q), torch.zeros_like(X)
    step = max(1, 500_000_000 // n)
    for a in range(0, nq, step):
        b = min(nq, a + step)
        z = Q[a:b] @ X.T / t + bias
        lse = torch.logsumexp(z, 1)
        lses[a:b] = lse
        which = torch.nonzero((s["targets"][a:b] >= 0) & (s["targets"][a:b] < n))[:, 0]
        column = s["targets"][a:b][which]
        mine = z[which, column]
        losses[a + which] = torch.where(mine > -math.inf, lse[which] - mine, torch.full_like(mine, math.inf))
        if c["op"] == "loss":
            continue
        p = torch.nan_to_num(torch.exp(z - lse[:, None]), nan=0.0)
        g, e = s["grad_losses"][a:b].double(), s["grad_lse"][a:b].double()
        there = torch.zeros_like(g)
        there[which] = torch.where(mine > -math.inf, g[which], torch.zeros_like(mine))
        p *= (there + e)[:, None]
        p[which, column] -= there[which]
        grad_Q[a:b] = p @ X / t
        grad_X += p.T @ Q[a:b] / t
    return (losses, lses) if c["op"] == "loss" else (grad_Q, grad_X)
