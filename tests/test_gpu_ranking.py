"""Ranking operators against plain implementations in 64 bits: rows in 4 bits, products and scores, log probabilities and their
gradient.  Tolerances follow from the arithmetic: 32-bit sums of n terms err by at most n units in the last place (2^-23 for a sum that cuts off)
of the sum of magnitudes, a result rounded to a type by half a unit of it."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def culsh():
    import culsh_b200
    return culsh_b200


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- oracles --------------------------------------------------------------------------------------------------------
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def held(X):
    """The values that rows in 4 bits stand for, float64 NumPy."""
    X = np.asarray(X, dtype=np.float64)
    n, d = X.shape
    x = np.zeros((n, -(-d // 32) * 32))
    x[:, :d] = X
    x = x.reshape(n, -1, 32)
    top = np.abs(x).max(2)
    with np.errstate(all="ignore"):
        e = np.clip(np.frexp(top)[1] - 3, -127, 127)
    e = np.where(top > 0, e, -127)
    y = np.abs(x) / np.exp2(e.astype(np.float64))[:, :, None]
    far = np.abs(y[..., None] - LEVELS)
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])  # the even code of two as near
    code = order[np.argmin(far[..., order], -1)]
    v = np.copysign(LEVELS[code], x) * np.exp2(e.astype(np.float64))[:, :, None]
    v[~np.isfinite(x).all(2)] = np.nan
    return v.reshape(n, -1)[:, :d]


def metric_of(dot, q, x, metric):
    q2, x2 = (q * q).sum(1)[:, None], (x * x).sum(1)[None, :]
    if metric == "cosine":
        with np.errstate(all="ignore"):
            return np.where((q2 == 0) | (x2 == 0), 0.0, dot / np.sqrt(q2) / np.sqrt(x2))
    return dot if metric == "dot" else 2 * dot - q2 - x2


def product_bound(q, x, metric, d):
    """Of a float32 score: the sum's error, and that of the norms and of what follows."""
    size = np.abs(q) @ np.abs(x).T
    q2, x2 = (q * q).sum(1)[:, None], (x * x).sum(1)[None, :]
    if metric == "dot":
        return (d + 2) * ULP * size
    if metric == "cosine":
        with np.errstate(all="ignore"):
            return np.nan_to_num((2 * d + 10) * ULP * size / np.sqrt(q2) / np.sqrt(x2), nan=1.0)
    return (d + 4) * ULP * (2 * size + q2 + x2)


def log_probs_of(z, target):
    """(log probability, entropy, lse) of one row of float64 scores by temperature."""
    if z.size == 0 or np.all(z == -np.inf):
        return -np.inf, 0.0, -np.inf
    m = z.max()
    with np.errstate(all="ignore"):
        lse = m + np.log(np.exp(z - m).sum())
        p = np.exp(z - lse)
        h = -np.where(p == 0, 0, p * (z - lse)).sum()
    lp = -np.inf if target is None or z[target] == -np.inf else z[target] - lse
    return lp, h, lse


# ---- rows -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES + [torch.float64])
@pytest.mark.parametrize("n,d", [(1, 1), (1, 31), (3, 32), (2, 33), (130, 77), (127, 128), (129, 129), (257, 1000), (2, 4096), (1, 5000)])
def test_rows_hold_the_nearest_values(culsh, dtype, n, d):
    X = torch.randn(n, d, generator=gen(n + d), device="cuda") * torch.exp2(torch.randint(-8, 9, (n, d), generator=gen(d), device="cuda").float())
    X = X.to(dtype)
    rows = culsh.MXRows(X)
    want = held(X.double().cpu().numpy())
    for t in TYPES + [torch.float64]:
        got = rows.dequantize(t)
        assert got.shape == (n, d) and got.dtype == t
        assert np.array_equal(got.double().cpu().numpy(), torch.from_numpy(want).to(t).double().numpy())
    norms = rows.norms.double().cpu().numpy()
    assert np.all(np.abs(norms - (want ** 2).sum(1)) <= (8 + d / 16) * ULP * (want ** 2).sum(1))
    assert rows.size_bytes() == rows.codes.numel() + rows.scales.numel() + 4 * n


@pytest.mark.parametrize("dtype", TYPES + [torch.float64])
def test_rounding_of_ties_extremes_and_zeros(culsh, dtype):
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    row = [4.0] + ties + [-t for t in ties] + [7.9, -7.9, 6.0, 0.0, -0.0] + [0.24, 0.26, 0.74, 0.76, 1.2, 1.3, 4.9, 5.1, 2.4, 2.6, 3.4, 3.6]
    block = torch.tensor(row[:32], dtype=torch.float64)
    tiny, huge = torch.finfo(dtype).smallest_normal, torch.finfo(dtype).max
    X = torch.zeros(8, 64, dtype=torch.float64)
    X[0, :block.numel()] = block
    X[1, :block.numel()] = block * 2.0 ** -9
    X[2, 3] = tiny / 4
    X[3, 5] = min(huge, 2.0 ** 126)
    X[4, 40] = -1.0
    X[6] = torch.linspace(-1, 1, 64, dtype=torch.float64)
    X[7, 0], X[7, 1] = 1.0, 2.0 ** -13
    X = X.to(dtype).cuda()
    rows = culsh.MXRows(X)
    want = held(X.double().cpu().numpy())
    assert np.array_equal(rows.dequantize(torch.float64).cpu().numpy(), want)
    assert float(rows.norms[5]) == 0.0


def test_double_values_beside_a_tie_go_to_their_side(culsh):
    X = torch.zeros(1, 32, dtype=torch.float64)
    X[0, 0] = 4.0
    for i, t in enumerate([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]):
        X[0, 1 + 3 * i], X[0, 2 + 3 * i], X[0, 3 + 3 * i] = t * (1 - 2.0 ** -45), t, t * (1 + 2.0 ** -45)
    X = X.cuda()
    assert np.array_equal(culsh.MXRows(X).dequantize(torch.float64).cpu().numpy(), held(X.cpu().numpy()))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", TYPES + [torch.float64])
def test_a_block_that_is_not_finite_is_nan_and_no_other(culsh, dtype, bad):
    X = torch.ones(200, 160, dtype=dtype, device="cuda")
    X[130, 70] = bad
    rows = culsh.MXRows(X)
    got = rows.dequantize()
    assert bool(torch.isnan(got[130, 64:96]).all()) and int(torch.isnan(got).sum()) == 32
    assert math.isnan(float(rows.norms[130])) and int(torch.isnan(rows.norms).sum()) == 1
    for metric in ("dot", "cosine", "euclidean"):
        s = rows.product(X[:3], metric=metric)
        assert bool(torch.isnan(s[:, 130]).all()) and int(torch.isnan(s).sum()) == 3
        s = rows.product(X[129:132], metric=metric)  # as a query, too
        assert bool(torch.isnan(s[1]).all()) and int(torch.isnan(s).sum()) == 200 + 2
        ids = torch.tensor([129, 130, 131], dtype=torch.int32, device="cuda")
        s = rows.score(torch.ones(1, 160, device="cuda"), (ids, torch.tensor([0, 3], device="cuda")), metric=metric)
        assert torch.isnan(s).tolist() == [False, True, False]


def test_rows_of_numpy_strided_and_misaligned_arrays(culsh):
    base = torch.randn(70, 301, generator=gen(), device="cuda")
    for X in (base[:, 1:], base[3:, :200], base[::2], base.T, base[:, ::3], base.to(torch.float16)[:, 1:130], base.expand(3, 70, 301)[1]):
        assert np.array_equal(culsh.MXRows(X).dequantize().double().cpu().numpy(), held(X.double().cpu().numpy()))
    X = base.cpu().numpy()
    assert np.array_equal(culsh.MXRows(X).dequantize().double().cpu().numpy(), held(X))
    row = base[0].expand(5, 301)  # rows that overlap
    assert np.array_equal(culsh.MXRows(row).dequantize().double().cpu().numpy(), held(row.double().cpu().numpy()))


def test_parts_make_the_same_rows(culsh):
    X = torch.randn(300, 200, generator=gen(), device="cuda")
    a = culsh.MXRows(X)
    b = culsh.MXRows.from_parts(a.codes.clone(), a.scales.clone(), a.norms.clone(), 200)
    assert (b.n_rows, b.n_features) == (300, 200)
    assert torch.equal(a.dequantize(), b.dequantize())
    assert torch.equal(a.product(X[:5]), b.product(X[:5]))


# ---- products -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("metric", ["dot", "cosine", "euclidean"])
@pytest.mark.parametrize("n,nq,d", [(1, 1, 1), (128, 16, 64), (127, 17, 96), (129, 127, 128), (300, 129, 256), (1000, 300, 384), (513, 40, 1000), (260, 260, 2176)])
def test_product(culsh, n, nq, d, metric):
    g = gen(n + nq + d)
    X = torch.randn(n, d, generator=g, device="cuda") * torch.exp2(torch.randint(-6, 7, (n, 1), generator=g, device="cuda").float())
    Q = torch.randn(nq, d, generator=g, device="cuda")
    X[n // 2] = 0
    rows = culsh.MXRows(X)
    q, x = held(Q.double().cpu().numpy()), held(X.double().cpu().numpy())
    want, bound = metric_of(q @ x.T, q, x, metric), product_bound(q, x, metric, d)
    for t in TYPES:
        got = rows.product(Q, metric=metric, dtype=t)
        assert got.shape == (nq, n) and got.dtype == t
        least = 2.0 ** -25 if t == torch.float16 else 0.0  # half a step of its smallest values
        got = got.double().cpu().numpy()
        beyond = np.abs(want) >= (65520.0 if t == torch.float16 else np.inf)  # what rounds to infinity in the type
        assert np.all(got[beyond] == np.copysign(np.inf, want[beyond]))
        err = np.abs(np.where(beyond, want, got) - want)
        assert np.all(err <= bound + HALF_ULP[t] * (np.abs(want) + bound) + least), float((err - bound).max())
    assert torch.equal(rows.product(culsh.MXRows(Q), metric=metric), rows.product(Q, metric=metric))
    rows.check()


def test_product_of_scales_far_apart(culsh):
    """Blocks whose scales are up to 2^40 apart: the large ones must not take the small ones' place, in any position of a row."""
    for k in range(0, 256, 32):
        X, Q = torch.zeros(130, 256, device="cuda"), torch.zeros(20, 256, device="cuda")
        X[:, k:k + 32] = torch.exp2(torch.arange(130, device="cuda").float() - 65)[:, None]
        Q[:, k:k + 32] = torch.exp2(2 * torch.arange(20, device="cuda").float() - 20)[:, None]
        got = culsh.MXRows(X).product(Q)
        assert torch.equal(got, 32 * Q[:, k:k + 1] * X[:, k][None, :])


def test_many_units_and_queries(culsh):
    """More tiles than SMs and accumulators, in every residue of the last tile; the result is the float32 product."""
    g = gen(3)
    for n, nq, d in [(148 * 128 * 2 + 5, 257, 128), (20_000, 1, 128), (128 * 150, 385, 192), (4_000, 1_000, 1_500)]:
        X, Q = torch.randn(n, d, generator=g, device="cuda"), torch.randn(nq, d, generator=g, device="cuda")
        rows, q = culsh.MXRows(X), culsh.MXRows(Q)
        x64, q64 = rows.dequantize(torch.float64), q.dequantize(torch.float64)
        bound = (d + 2) * ULP * (q64.abs() @ x64.abs().T)
        assert bool(((rows.product(q).double() - q64 @ x64.T).abs() <= bound).all())
        assert torch.equal(rows.product(q), rows.product(q))


def test_product_of_more_than_two_to_the_31_scores(culsh):
    n, nq = 1_000_003, 2_200
    X = torch.randn(n, 32, generator=gen(), device="cuda")
    Q = torch.randn(nq, 32, generator=gen(1), device="cuda")
    rows = culsh.MXRows(X)
    got = rows.product(Q, dtype=torch.float16)
    last = rows.product(Q[-3:], dtype=torch.float16)
    assert torch.equal(got[-3:], last)
    r = culsh.log_probs(got, top_k=3)
    one = culsh.log_probs(got[-1:].clone(), top_k=3)
    assert torch.equal(r.top_ids[-1:], one.top_ids)
    assert torch.allclose(r.lse[-1:], one.lse, rtol=0, atol=1e-5)


# ---- scores of candidates -------------------------------------------------------------------------------------------
def csr(lengths, n, g):
    offsets = torch.zeros(len(lengths) + 1, dtype=torch.int64)
    offsets[1:] = torch.cumsum(torch.tensor(lengths), 0)
    ids = [torch.sort(torch.randperm(n, generator=g)[:m]).values for m in lengths]
    return torch.cat(ids).to(torch.int32).cuda() if ids else torch.zeros(0, dtype=torch.int32).cuda(), offsets.cuda()


@pytest.mark.parametrize("metric", ["dot", "cosine", "euclidean"])
@pytest.mark.parametrize("dtype", TYPES + [torch.float64])
@pytest.mark.parametrize("d", [1, 31, 64, 128, 200, 1000])
def test_score(culsh, d, dtype, metric):
    g = gen(d)
    n = 700
    X = torch.randn(n, d, generator=g, device="cuda")
    X[5] = 0
    lengths = [0, 1, 0, 0, 7, 300, 700, 2, 0, 64, 65, 63, 1, 1, 1, 0]
    Q = torch.randn(len(lengths), d, generator=g, device="cuda").to(dtype)
    Q[4] = 0
    ids, offsets = csr(lengths, n, torch.Generator().manual_seed(d))
    got = culsh.MXRows(X).score(Q, (ids, offsets), metric=metric).double().cpu().numpy()
    q, x = Q.float().double().cpu().numpy(), held(X.double().cpu().numpy())
    at, owner = ids.long().cpu().numpy(), np.repeat(np.arange(len(lengths)), lengths)
    want, bound = metric_of(q @ x.T, q, x, metric)[owner, at], product_bound(q, x, metric, d)[owner, at]
    if dtype == torch.float64:  # taken in 32 bits
        bound = bound + product_bound(q, x, metric, 2)[owner, at]
    assert np.all(np.abs(got - want) <= bound + 2.0 ** -24 * np.abs(want))


@pytest.mark.parametrize("law", ["one_term", "wide", "decades"])
def test_score_holds_small_terms_of_a_query(culsh, law):
    """Queries whose values are far apart, against rows that pick single ones out."""
    d, n = 96, 96
    X = torch.eye(n, device="cuda")
    g = gen(1)
    Q = torch.randn(3, d, generator=g, device="cuda")
    if law == "wide":
        Q *= torch.exp2(torch.randint(-30, 31, (3, d), generator=g, device="cuda").float())
    elif law == "decades":
        Q *= torch.exp2(torch.linspace(-100, 100, d, device="cuda"))[None]
    ids = torch.arange(n, dtype=torch.int32, device="cuda").repeat(3)
    got = culsh.MXRows(X).score(Q, (ids, torch.arange(4, device="cuda") * n)).view(3, n)
    assert bool(((got.double() - Q.double()).abs() <= ULP * Q.double().abs()).all())


def test_score_of_ids_that_are_no_rows(culsh):
    rows = culsh.MXRows(torch.ones(10, 40, device="cuda"))
    ids = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    s = rows.score(torch.ones(1, 40, device="cuda"), (ids, torch.tensor([0, 6], device="cuda")))
    assert torch.isnan(s).tolist() == [False, True, False, True, True, True] and float(s[0]) == 40.0


def test_score_takes_what_query_returns(culsh):
    rng = np.random.RandomState(0)
    X = rng.randn(5000, 48).astype(np.float32)
    Q = X[:200] + 0.05 * rng.randn(200, 48).astype(np.float32)
    model = culsh.RPLSH(8, 10, seed=0).fit(X)
    cand = model.query(Q)
    rows = culsh.MXRows(X)
    ids, offsets = cand.get_indices(as_torch=True), cand.get_offsets(as_torch=True)
    a, b = rows.score(Q, cand, metric="cosine"), rows.score(Q, (ids, offsets), metric="cosine")
    assert torch.equal(a, b)
    r, s = culsh.rank(rows, Q, cand, top_k=5, metric="cosine", temperature=0.1), culsh.rank(rows, Q, (ids, offsets), top_k=5, metric="cosine", temperature=0.1)
    assert all(x is y is None or torch.equal(x, y) for x, y in zip(r, s))
    assert (r.top_ids[:, 0].cpu().numpy() == np.arange(200)).mean() > 0.99  # each query's own row comes first
    # results that go at once: their memory must not be taken before it has been read
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        Qd = torch.from_numpy(Q).cuda()
        for _ in range(20):
            s = rows.score(Qd, model.query(Q), metric="cosine")
            model.query(Q[::-1].copy())
            assert torch.equal(s, a)
    empty = model.query(Q + 100 * rng.randn(*Q.shape).astype(np.float32))
    assert rows.score(Q, empty).shape[0] == empty.n_total_candidates


# ---- log probabilities ----------------------------------------------------------------------------------------------
def check_log_probs(r, scores, targets, temperature, k, rows, names=None):
    """A LogProbs against 64 bits.  rows: float64 arrays of the scores of each row."""
    for i, s in enumerate(rows):
        z = s / temperature
        t = targets[i]
        place = None
        if t is not None:
            if names is None:
                place = t if 0 <= t < len(s) else None
            else:
                hit = np.nonzero(names[i] == t)[0]
                place = int(hit[0]) if hit.size else None
        lp, h, lse = log_probs_of(z, place)
        finite = z[np.isfinite(z)]
        # the product with 1 / temperature, the sums' and the functions' errors
        tol = 4 * ULP * ((np.abs(finite).max() if finite.size else 0) + 32)
        for got, want in ((r.lse[i], lse), (r.entropy[i], h)) + (((r.log_probs[i], lp),) if r.log_probs is not None else ()):
            got = float(got)
            if not np.isfinite(want):
                assert (math.isnan(got) and math.isnan(want)) or got == want, (i, got, want)
            else:
                assert abs(got - want) <= tol, (i, got, want, tol)
        if not k:
            continue
        live = np.nonzero(~np.isnan(s) & (z != -np.inf))[0]
        order = live[np.lexsort((live, -s[live]))][:k]
        ids = r.top_ids[i].cpu().numpy()
        want_ids = order if names is None else names[i][order]
        assert np.array_equal(ids[:len(order)], want_ids), (i, ids, want_ids)
        assert np.all(ids[len(order):] == -1) and np.all(r.top_log_probs[i, len(order):].cpu().numpy() == -np.inf)
        with np.errstate(all="ignore"):
            want = z[order] - lse
        got = r.top_log_probs[i, :len(order)].double().cpu().numpy()
        assert np.all((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want))), (i, got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,temperature,pad", [
    (1, 1, 1, 1.0, 0), (3, 2, 5, 0.3, 0), (5, 511, 10, 1.0, 1), (4, 512, 1, 0.05, 0), (4, 513, 128, 1.0, 3), (3, 4099, 32, 1.0, 0),
    (2, 20_000, 10, 0.1, 7), (3, 70_001, 100, 1.0, 0), (1, 300_000, 128, 1.0, 0), (600, 20_011, 3, 1.0, 5), (2, 16_385, 0, 2.0, 0)])
def test_log_probs_of_matrices(culsh, m, n, k, temperature, pad, dtype):
    g = gen(m + n)
    wide = torch.randn(m, n + pad, generator=g, device="cuda").mul_(3 * temperature).to(dtype)
    s = wide[:, pad // 2:pad // 2 + n]  # rows and the first one begin off the boundaries
    targets = torch.randint(0, n, (m,), generator=g, device="cuda")
    targets[0] = n - 1
    if m > 2:
        targets[1], targets[2] = -1, n
    r = culsh.log_probs(s, targets, top_k=k, temperature=temperature)
    assert (r.top_ids is None) == (k == 0)
    some = sorted({0, 1, 2, m // 2, m - 1} & set(range(m)))
    sub = type(r)(*(None if x is None else x[some] for x in r))
    check_log_probs(sub, s, [int(targets[i]) for i in some], temperature, k, [s[i].double().cpu().numpy() for i in some])
    again = culsh.log_probs(s, targets, top_k=k, temperature=temperature)
    assert all(x is y is None or torch.equal(x, y) for x, y in zip(r, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [100, 3000, 40_000])
def test_log_probs_of_masks_and_values_that_are_not_finite(culsh, n, dtype):
    low = torch.finfo(dtype).min
    s = torch.randn(14, n, generator=gen(n), device="cuda").to(dtype)
    s[0] = -math.inf
    s[1] = low
    s[2, n // 3:] = -math.inf
    s[3, :n - 1] = -math.inf
    s[4, 7] = math.nan
    s[5, 9] = math.inf
    s[6, :-3] = low
    s[7] = 0.5
    s[8] = torch.linspace(-5, 5, n, device="cuda").to(dtype)
    s[9] = torch.linspace(5, -5, n, device="cuda").to(dtype)
    s[10] = -math.inf
    s[10, ::2] = low
    s[11] = -math.inf
    s[11, 3] = math.nan
    s[12] = (torch.arange(n, device="cuda") % 3).to(dtype)
    s[13, ::2] = -0.0
    s[13, 1::2] = 0.0
    targets = [0, 1, n // 2, n - 1, 3, 9, n - 1, 5, n - 1, 0, 2, 3, 2, 1]
    for t in (1.0, 0.5):
        r = culsh.log_probs(s, torch.tensor(targets, device="cuda"), top_k=20, temperature=t)
        # lowest float32 values by a temperature below 1 are beyond the type: masked
        rows = s.double().cpu().numpy()
        if dtype == torch.float32 and t < 1 or dtype == torch.bfloat16 and t < 1:
            rows = np.where(rows / t < -3.5e38, -np.inf, rows)
        check_log_probs(r, s, targets, t, 20, list(rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,k", [([0, 1, 0, 5, 512, 513, 0, 3000, 2, 0], 7), ([0, 0, 0], 2), ([70_000], 128), ([0, 40_000, 0, 90_000, 1], 10),
                                       ([3] * 1000, 5), ([600_000] + [2] * 700, 9)])
def test_log_probs_of_lists(culsh, lengths, k, dtype):
    n = max(max(lengths), 1) * 2
    ids, offsets = csr(lengths, n, torch.Generator().manual_seed(k))
    s = torch.randn(ids.shape[0], generator=gen(k), device="cuda").to(dtype)
    targets = []
    for i, m in enumerate(lengths):
        mine = ids[offsets[i]:offsets[i + 1]]
        targets.append(n + 5 if i % 4 == 3 or not m else int(mine[(i * 7) % m]))
    r = culsh.log_probs(s, torch.tensor(targets, device="cuda"), (ids, offsets), top_k=k, temperature=0.4)
    some = list(range(len(lengths))) if len(lengths) < 20 else [0, 1, 2, 3, len(lengths) - 1]
    sub = type(r)(*(x[some] for x in r))
    cut = lambda a, i: a[offsets[i]:offsets[i + 1]].cpu()  # noqa: E731
    check_log_probs(sub, s, [targets[i] for i in some], 0.4, k, [cut(s, i).double().numpy() for i in some], [cut(ids, i).numpy() for i in some])
    places = culsh.log_probs(s, None, (None, offsets), top_k=k, temperature=0.4)
    assert places.log_probs is None and torch.equal(places.lse, r.lse) and torch.equal(places.top_log_probs, r.top_log_probs)
    for i in some:
        p = places.top_ids[i]
        p = p[p >= 0].long()
        assert torch.equal(ids[offsets[i]:offsets[i + 1]][p], r.top_ids[i][r.top_ids[i] >= 0])


def test_lists_that_begin_off_a_boundary(culsh):
    for off in range(1, 9):
        for dtype in TYPES:
            s = torch.randn(2000 + off, generator=gen(off), device="cuda").to(dtype)[off:]
            offsets = torch.tensor([0, 3, 3, 700, 2000], device="cuda")
            r = culsh.log_probs(s, None, (None, offsets), top_k=4)
            check_log_probs(r, s, [None] * 4, 1.0, 4, [s[a:b].double().cpu().numpy() for a, b in ((0, 3), (3, 3), (3, 700), (700, 2000))])


def test_rows_of_nothing(culsh):
    r = culsh.log_probs(torch.empty(3, 0, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), top_k=2)
    assert r.lse.tolist() == [-math.inf] * 3 and r.entropy.tolist() == [0.0] * 3 and r.log_probs.tolist() == [-math.inf] * 3
    assert r.top_ids.tolist() == [[-1, -1]] * 3
    r = culsh.log_probs(torch.empty(0, 7, device="cuda"), top_k=2)
    assert r.lse.shape == (0,) and r.top_ids.shape == (0, 2)
    assert culsh.log_probs_backward(torch.empty(0, 7, device="cuda"), None, torch.empty(0, device="cuda"), torch.empty(0, device="cuda")).shape == (0, 7)
    rows = culsh.MXRows(torch.empty(0, 7, device="cuda"))
    assert rows.product(torch.ones(2, 7, device="cuda")).shape == (2, 0)
    assert culsh.MXRows(torch.ones(3, 7, device="cuda")).product(torch.empty(0, 7, device="cuda")).shape == (0, 3)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert rows.score(torch.ones(2, 7, device="cuda"), (none, torch.zeros(3, dtype=torch.int64, device="cuda"))).shape == (0,)


# ---- gradient -------------------------------------------------------------------------------------------------------
def gradient_of(z, target, g, h, temperature):
    lp_t, H, lse = log_probs_of(z, target)
    if lse == -np.inf:
        return np.zeros_like(z)
    with np.errstate(all="ignore"):
        lp = z - lse
        p = np.exp(lp)
        d = -h * np.where(p > 0, p * (lp + H), 0)
    if target is not None and z[target] != -np.inf:
        d = d - g * p
        d[target] += g
    return d / temperature


def gradient_bound(z, g, h, temperature):
    """log p errs by some units of the largest |z| of those that have a probability, p by as much of itself; entropy and log p of up to 100 by h p."""
    finite = z[np.isfinite(z) & (z >= z.max(initial=-np.inf) - 100)]
    big = (np.abs(finite).max() if finite.size else 0) + 32
    return 8 * ULP * big * (abs(g) + abs(h) * big) / temperature


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,temperature,pad", [(1, 1, 1.0, 0), (4, 2, 0.3, 1), (5, 511, 1.0, 0), (5, 1025, 0.2, 3), (3, 30_000, 1.0, 8), (2, 70_001, 1.0, 0)])
def test_gradient_of_matrices(culsh, m, n, temperature, pad, dtype):
    g = gen(n)
    s = torch.randn(m, n + pad, generator=g, device="cuda").mul_(2 * temperature).to(dtype)[:, pad // 2:pad // 2 + n]
    if n > 4:
        s[0, 2:5] = -math.inf
        s[m - 1, 1:] = torch.finfo(dtype).min
    targets = torch.randint(0, n, (m,), generator=g, device="cuda")
    if m > 3:
        targets[1], targets[2] = -1, n + 3
        if n > 4:
            targets[0] = 3
            s[3] = -math.inf
    gl, ge = torch.randn(m, generator=g, device="cuda"), torch.randn(m, generator=g, device="cuda")
    r = culsh.log_probs(s, targets, temperature=temperature)
    got = culsh.log_probs_backward(s, targets, r.lse, r.entropy, gl, ge, temperature=temperature)
    assert got.shape == s.shape and got.dtype == dtype and got.is_contiguous()
    only_g = culsh.log_probs_backward(s, targets, r.lse, r.entropy, grad_log_probs=gl, temperature=temperature)
    only_e = culsh.log_probs_backward(s, None, r.lse, r.entropy, grad_entropy=ge, temperature=temperature)
    for i in range(m):
        z = s[i].double().cpu().numpy() / temperature
        if dtype != torch.float16 and temperature < 1:
            z = np.where(z < -3.5e38, -np.inf, z)
        t = int(targets[i]) if 0 <= int(targets[i]) < n else None
        for out, a, b in ((got, float(gl[i]), float(ge[i])), (only_g, float(gl[i]), 0.0), (only_e, 0.0, float(ge[i]))):
            want = gradient_of(z, t, a, b, temperature)
            bound = gradient_bound(z, a, b, temperature)
            err = np.abs(out[i].double().cpu().numpy() - want)
            least = 2.0 ** -25 if dtype == torch.float16 else 0.0
            assert np.all(err <= bound + HALF_ULP[dtype] * np.abs(want) + least), (i, err.max(), bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[0, 1, 2, 0, 5, 511, 513, 0, 3000, 1, 0], [1] * 700, [50_000, 0, 3]])
def test_gradient_of_lists(culsh, lengths, dtype):
    n, temperature = 2 * max(lengths), 0.25
    ids, offsets = csr(lengths, n, torch.Generator().manual_seed(1))
    s = torch.randn(ids.shape[0] + 3, generator=gen(5), device="cuda").to(dtype)[3:]
    s[::17] = -math.inf
    m = len(lengths)
    targets = [n if i % 5 == 4 or not k else int(ids[int(offsets[i]) + (3 * i) % k]) for i, k in enumerate(lengths)]
    gl, ge = torch.randn(m, generator=gen(6), device="cuda"), torch.randn(m, generator=gen(7), device="cuda")
    t = torch.tensor(targets, device="cuda")
    r = culsh.log_probs(s, t, (ids, offsets), temperature=temperature)
    got = culsh.log_probs_backward(s, t, r.lse, r.entropy, gl, ge, (ids, offsets), temperature)
    for i in range(min(m, 50)):
        a, b = int(offsets[i]), int(offsets[i + 1])
        z = s[a:b].double().cpu().numpy() / temperature
        hit = np.nonzero(ids[a:b].cpu().numpy() == targets[i])[0]
        want = gradient_of(z, int(hit[0]) if hit.size else None, float(gl[i]), float(ge[i]), temperature)
        err = np.abs(got[a:b].double().cpu().numpy() - want)
        least = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert np.all(err <= gradient_bound(z, float(gl[i]), float(ge[i]), temperature) + HALF_ULP[dtype] * np.abs(want) + least)


def test_gradient_against_differences(culsh):
    n, temperature, target, a, b = 40, 0.5, 11, 1.3, -0.7
    s = torch.randn(1, n, generator=gen(9), device="cuda")
    t = torch.tensor([target], device="cuda")
    r = culsh.log_probs(s, t, temperature=temperature)
    got = culsh.log_probs_backward(s, t, r.lse, r.entropy, torch.tensor([a], device="cuda"), torch.tensor([b], device="cuda"), temperature=temperature)[0]
    x, step = s[0].double().cpu().numpy(), 1e-4

    def loss(v):
        lp, h, _ = log_probs_of(v / temperature, target)
        return a * lp + b * h

    for i in range(n):
        up, down = x.copy(), x.copy()
        up[i] += step
        down[i] -= step
        # second-order differences: step^2 times a third derivative of at most some tens; the kernel's own error
        assert abs(float(got[i]) - (loss(up) - loss(down)) / (2 * step)) <= 1e-6 + gradient_bound(x / temperature, a, b, temperature)


# ---- streams, refusals ----------------------------------------------------------------------------------------------
def test_work_is_queued_on_the_current_stream(culsh):
    X, Q = torch.randn(20_000, 128, generator=gen(), device="cuda"), torch.randn(64, 128, generator=gen(1), device="cuda")
    want = culsh.rank(culsh.MXRows(X), Q, top_k=5, metric="cosine", temperature=0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(6000, 6000, device="cuda")
        late = torch.zeros_like(X)
        for _ in range(5):
            big = big @ big * 1e-3  # keeps the stream busy
        late.copy_(X)
        got = culsh.rank(culsh.MXRows(late), Q, top_k=5, metric="cosine", temperature=0.1)
    side.synchronize()
    assert torch.equal(got.top_ids, want.top_ids) and torch.equal(got.lse, want.lse)


def test_operators_in_a_graph(culsh):
    X, Q = torch.randn(3000, 128, generator=gen(), device="cuda"), torch.randn(8, 128, generator=gen(1), device="cuda")
    rows = culsh.MXRows(X)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        culsh.rank(rows, Q, top_k=5)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = culsh.rank(rows, Q, top_k=5)
    Q.copy_(torch.randn(8, 128, generator=gen(2), device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    want = culsh.rank(rows, Q, top_k=5)
    assert torch.equal(r.top_ids, want.top_ids) and torch.equal(r.lse, want.lse)


def test_refusals(culsh):
    X = torch.ones(10, 40, device="cuda")
    rows = culsh.MXRows(X)
    ids, offsets = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([0, 3], device="cuda")
    s = torch.ones(2, 5, device="cuda")
    two = torch.zeros(2, device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    for error, call in [
        (ValueError, lambda: culsh.MXRows(X[0])),
        (ValueError, lambda: culsh.MXRows(torch.empty(3, 0, device="cuda"))),
        (TypeError, lambda: culsh.MXRows(X.int())),
        (TypeError, lambda: rows.dequantize(torch.int32)),
        (ValueError, lambda: culsh.MXRows.from_parts(rows.codes, rows.scales, rows.norms, 200)),
        (ValueError, lambda: culsh.MXRows.from_parts(rows.codes, rows.scales[:, :, :1], rows.norms, 40)),
        (ValueError, lambda: culsh.MXRows.from_parts(rows.codes.cpu(), rows.scales.cpu(), rows.norms.cpu(), 40)),
        (ValueError, lambda: rows.product(X[:, :39])),
        (ValueError, lambda: rows.product(X, metric="manhattan")),
        (TypeError, lambda: rows.product(X, dtype=torch.float64)),
        (TypeError, lambda: rows.product(X.int())),
        (ValueError, lambda: rows.score(X[:2], (ids, offsets))),
        (ValueError, lambda: rows.score(X[:1, :39], (ids, offsets))),
        (TypeError, lambda: rows.score(X[:1], (ids.long(), offsets))),
        (TypeError, lambda: rows.score(X[:1], (ids, offsets.int()))),
        (ValueError, lambda: rows.score(X[:1], (None, offsets))),
        (ValueError, lambda: culsh.log_probs(s, top_k=129)),
        (ValueError, lambda: culsh.log_probs(s, top_k=-1)),
        (ValueError, lambda: culsh.log_probs(s, temperature=0.0)),
        (ValueError, lambda: culsh.log_probs(s, temperature=float("nan"))),
        (ValueError, lambda: culsh.log_probs(s[0])),
        (TypeError, lambda: culsh.log_probs(s.double())),
        (ValueError, lambda: culsh.log_probs(s, t[:1])),
        (ValueError, lambda: culsh.log_probs(s, two)),
        (ValueError, lambda: culsh.log_probs(s[0], None, (ids, offsets))),
        (ValueError, lambda: culsh.log_probs(s[0, :3], t[:1], (None, offsets))),
        (ValueError, lambda: culsh.log_probs_backward(s, None, two, two, two)),
        (ValueError, lambda: culsh.log_probs_backward(s, t, two[:1], two, two)),
        (TypeError, lambda: culsh.log_probs_backward(s, t, two.double(), two, two)),
    ]:
        with pytest.raises(error):
            call()
    with pytest.raises(RuntimeError, match="16 bytes"):  # codes that TMA cannot load
        codes = torch.zeros(10 * 64 + 16, dtype=torch.uint8, device="cuda")[1:641].view(10, 64)
        culsh.MXRows.from_parts(codes, rows.scales, rows.norms, 40).dequantize()


@pytest.mark.parametrize("metric", ["dot", "cosine", "euclidean"])
@pytest.mark.parametrize("d,nq,mean", [(100, 300, 1500), (128, 3, 150_000), (256, 40, 6000), (384, 30, 5000), (512, 500, 900), (700, 20, 4000), (2300, 9, 4000)])
def test_score_of_many_candidates(culsh, d, nq, mean, metric):
    """Lists long enough for the tensor cores, of all lengths around a tile's, with ids that are no rows, against float64 on the device."""
    g, n = gen(d + nq), 200_000 if d <= 256 else 30_000
    X = torch.randn(n, d, generator=g, device="cuda")
    X[::1000] = 0
    Q = torch.randn(nq, d, generator=g, device="cuda")
    length = torch.randint(0, 2 * mean, (nq,), generator=g, device="cuda")
    length[::5] = torch.tensor([0, 1, 127, 128, 129, 256, 383], device="cuda").repeat(nq)[:length[::5].numel()]
    offsets = torch.zeros(nq + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = torch.cumsum(length, 0)
    total = int(offsets[-1])
    ids = torch.randint(0, n, (total,), generator=g, device="cuda").int()
    ids[::977] = -1
    ids[5::1013] = n
    rows = culsh.MXRows(X)
    got = rows.score(Q, (ids, offsets), metric=metric).double()
    assert torch.equal(got.isnan(), (ids < 0) | (ids >= n))
    x, q = rows.dequantize(torch.float64), Q.double()
    owner = torch.repeat_interleave(torch.arange(nq, device="cuda"), length)
    x2, q2 = (x * x).sum(1), (q * q).sum(1)
    for at in range(0, total, 200_000):
        i, o = ids[at:at + 200_000].long().clamp(0, n - 1), owner[at:at + 200_000]
        dot, size = (x[i] * q[o]).sum(1), (x[i] * q[o]).abs().sum(1)
        if metric == "dot":
            want, bound = dot, (d + 2) * ULP * size
        elif metric == "cosine":
            length2 = (x2[i] * q2[o]).sqrt()
            want = torch.where(length2 > 0, dot / length2, torch.zeros_like(dot))
            bound = torch.where(length2 > 0, (2 * d + 10) * ULP * size / length2, torch.ones_like(dot) * ULP)
        else:
            want, bound = 2 * dot - x2[i] - q2[o], (d + 4) * ULP * (2 * size + x2[i] + q2[o])
        part = got[at:at + 200_000]
        assert bool(((part - want).abs() <= bound)[~part.isnan()].all())
    assert torch.equal(rows.score(Q, (ids, offsets), metric=metric).nan_to_num(9.0), got.float().nan_to_num(9.0))


@pytest.mark.parametrize("law", ["one_term", "wide", "decades", "whole", "tiny", "huge"])
def test_score_of_many_candidates_holds_small_terms_of_a_query(culsh, law):
    d, n, times = 96, 96, 4000
    X = torch.eye(n, device="cuda")
    Q = torch.randn(3, d, generator=gen(1), device="cuda")
    if law == "wide":
        Q *= torch.exp2(torch.randint(-30, 31, (3, d), generator=gen(2), device="cuda").float())
    elif law == "decades":
        Q *= torch.exp2(torch.linspace(-50, 50, d, device="cuda"))[None]
    elif law == "whole":
        Q = torch.randint(-255, 256, (3, d), generator=gen(2), device="cuda").float()
    elif law == "tiny":
        Q *= 2.0 ** -90
    elif law == "huge":
        Q *= 2.0 ** 120
    ids = torch.arange(n, dtype=torch.int32, device="cuda").repeat(3 * times)
    got = culsh.MXRows(X).score(Q, (ids, torch.arange(4, device="cuda") * n * times)).view(3, times, n)
    assert bool((got == got[:, :1]).all())
    assert bool(((got[:, 0].double() - Q.double()).abs() <= ULP * Q.double().abs()).all())


def test_score_of_more_queries_than_the_workspace_holds(culsh):
    n, d, nq, each = 5000, 600, 4000, 130  # 2,900 of these queries are 64 MB of slices
    X, Q = torch.randn(n, d, generator=gen(), device="cuda"), torch.randn(nq, d, generator=gen(1), device="cuda")
    ids = torch.randint(0, n, (nq * each,), generator=gen(2), device="cuda").int()
    offsets = torch.arange(nq + 1, device="cuda") * each
    rows = culsh.MXRows(X)
    got = rows.score(Q, (ids, offsets)).view(nq, each).double()
    x = rows.dequantize(torch.float64)
    for q in (0, 1, 2800, 2900, 3000, nq - 1):
        r = x[ids[q * each:(q + 1) * each].long()] * Q[q].double()
        assert bool(((got[q] - r.sum(1)).abs() <= (d + 2) * ULP * r.abs().sum(1)).all())


def test_the_example_finds_and_learns():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "rank_candidates.py")
    spec = importlib.util.spec_from_file_location("rank_candidates", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    found, recall, loss = example.main(rows=20_000, queries=500, features=64, top=5, tables=16, hashes=10)
    assert found > 0.8 and recall > 0.3 and loss[1] < loss[0]


def test_calls_behind_one_another_do_not_see_what_was_there_before(culsh):
    """Kernels that are set up early read what the one in front wrote, in memory that earlier calls had used for the same: calls on changing data
    without a wait between them give what they give one at a time."""
    n, d, nq = 60_000, 128, 40
    g = gen(11)
    sets = [(torch.randn(n, d, generator=g, device="cuda"), torch.randn(nq, d, generator=g, device="cuda")) for _ in range(3)]
    ids = torch.randint(0, n, (nq * 9000,), generator=g, device="cuda").int()
    offsets = torch.arange(nq + 1, device="cuda") * 9000

    def step(X, Q):
        rows = culsh.MXRows(X)
        s = rows.score(Q, (ids, offsets), metric="cosine")
        p = rows.product(Q, metric="euclidean")
        held = rows.product(culsh.MXRows(Q), metric="cosine")
        r = culsh.log_probs(p[:3], top_k=7)  # long rows, several CTAs each
        return s, p[:, ::997].clone(), held[:, ::997].clone(), r.lse, r.entropy, r.top_ids, r.top_log_probs

    want = []
    for X, Q in sets:
        want.append([x.clone() for x in step(X, Q)])
        torch.cuda.synchronize()
    got = [(i % 3, step(*sets[i % 3])) for i in range(60)]
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_more_entries_than_places_have_bits_for_are_refused(culsh):
    from culsh_b200 import _lib
    from culsh_b200._culsh_core import get_handle
    h, x = get_handle(0), torch.zeros(64, dtype=torch.int64, device="cuda")
    at = x.data_ptr()
    for ids, total in ((None, 2 ** 31), (at, 2 ** 32)):
        status = h.lib.culsh_log_probs(h.ptr, at, 0, 1, 0, 0, at, ids, total, 1.0, None, 0, None, at, at, None, None, None, 0, None)
        assert status == -5 and b"too many" in _lib.load().culsh_last_error()
