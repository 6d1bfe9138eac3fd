"""Rows in 8-bit integers against plain implementations in 64 bits.  Codes, scales and sums of squares are equal; a score's tolerance counts its roundings: the whole number's (2^-24), the
scales' product's, the product's with it; a result rounded to a type by half a unit of it."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
ALL = [torch.float32, torch.float16, torch.bfloat16, torch.float64]
TYPES = [torch.float32, torch.float16, torch.bfloat16]
METRICS = ["dot", "cosine", "euclidean"]


@pytest.fixture(scope="module")
def culsh():
    import culsh_b200
    return culsh_b200


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def held(X):
    """(codes, scales float32, squares) of rows, NumPy."""
    x = np.asarray(X, dtype=np.float64)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(1)
        scale = np.maximum((top / 127).astype(np.float32), np.float32(2.0 ** -126))
        bad = ~np.isfinite(top) | ~np.isfinite(scale)
        code = np.rint(x / scale.astype(np.float64)[:, None])
    code[bad] = 0
    scale = np.where(bad, np.float32(np.nan), scale)
    squares = np.where(bad, -1, (code * code).sum(1)).astype(np.int64)
    return code, scale, squares


def numpy(x):
    return x.double().cpu().numpy()


def expect(Q, X, metric):
    """Scores in 64 bits and their tolerance in 32, from arrays that are held."""
    (cq, sq, nq), (cx, sx, nx) = Q, X
    a = cq @ cx.T
    s = sq.astype(np.float64)[:, None] * sx.astype(np.float64)[None, :]
    if metric == "cosine":
        with np.errstate(all="ignore"):
            v = np.where((nq[:, None] == 0) | (nx[None, :] == 0), 0.0, a / np.sqrt(nq)[:, None] / np.sqrt(nx)[None, :])
        v = np.where((nq[:, None] < 0) | (nx[None, :] < 0), np.nan, v)
        return v, 8 * U * np.abs(v)
    v = a * s
    if metric == "dot":
        return v, 4 * U * np.abs(v) + 2.0 ** -148
    q2, x2 = (sq.astype(np.float64) ** 2 * nq)[:, None], (sx.astype(np.float64) ** 2 * nx)[None, :]
    return 2 * v - q2 - x2, 8 * U * (2 * np.abs(v) + q2 + x2) + 2.0 ** -146


def close(out, want, tol, dtype=torch.float32):
    out = numpy(out)
    nan = np.isnan(want)
    assert (np.isnan(out) == nan).all()
    off = np.abs(out - want)[~nan]
    t = (tol + HALF_ULP[dtype] * (np.abs(want) + tol) + LEAST[dtype])[~nan]
    assert (off <= t).all(), (off - t).max()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,d", [(1, 1), (3, 15), (5, 16), (257, 100), (33, 129), (2, 4097), (1, 70_001), (1000, 8)])
def test_rows_hold_the_nearest_whole_numbers(culsh, dtype, n, d):
    X = torch.randn(n, d, generator=gen(n + d), device="cuda", dtype=torch.float64) * torch.exp2(torch.randint(-12, 13, (n, 1), generator=gen(1), device="cuda").double())
    X = X.to(dtype)
    rows = culsh.Int8Rows(X)
    code, scale, squares = held(numpy(X))
    assert rows.codes.shape == (n, -(-d // 16) * 16) and (numpy(rows.codes)[:, :d] == code).all() and not rows.codes[:, d:].any()
    assert (rows.scales.cpu().numpy() == scale).all() and (rows.squares.cpu().numpy() == squares).all()
    assert rows.size_bytes() == n * (rows.codes.shape[1] + 8) and (rows.n_rows, rows.n_features) == (n, d)
    for to in ALL:
        want = torch.from_numpy(code * scale.astype(np.float64)[:, None])
        got = rows.dequantize(to).cpu()
        if to == torch.float64:
            assert (got == want).all()
        else:  # 32 bits first
            assert (got == want.float().to(to)).all()


def test_ties_zeros_extremes_and_rows_that_are_not_finite(culsh):
    X = torch.zeros(8, 40, device="cuda")
    X[0, 0], X[0, 1:6] = 127.0, torch.tensor([0.5, 1.5, -2.5, 126.5, -0.5], device="cuda")  # ties: to the even number
    X[2] = 3.0e38
    X[3, 1] = 1.0e-45  # the least scale
    X[3, 2] = 2.0 ** -126
    X[4, 39] = float("nan")
    X[5, 0] = float("-inf")
    X[6, 20], X[6, 21] = -1.0e-40, 1.0e-44
    X[7] = torch.arange(40, device="cuda") * 3.3e-3
    rows = culsh.Int8Rows(X)
    code, scale, squares = held(numpy(X))
    assert (numpy(rows.codes)[:, :40] == code).all()
    assert np.array_equal(rows.scales.cpu().numpy(), scale, equal_nan=True) and (rows.squares.cpu().numpy() == squares).all()
    assert list(rows.codes[0, :6].tolist()) == [127, 0, 2, -2, 126, 0]
    assert torch.isnan(rows.dequantize()[4:6]).all() and not torch.isnan(rows.dequantize()[[0, 1, 2, 3, 6, 7]]).any()
    for m in METRICS:
        s = rows.product(X[:1], metric=m)
        assert torch.isnan(s[0, 4:6]).all() and not torch.isnan(s[0, [0, 1, 3, 6, 7]]).any()
        assert torch.isnan(culsh.Int8Rows(X[[0, 1]]).product(X[4:6], metric=m)).all()
    big = torch.tensor([[1e300, 1.0]], device="cuda", dtype=torch.float64)
    assert torch.isnan(culsh.Int8Rows(big).scales).all()


def test_float_values_beside_a_tie_go_to_their_side(culsh):
    """Quotients within 2^-20 of a half: the scale is no power of two, so few are ties."""
    top = torch.tensor([1.0 + 2.0 ** -23, 1.7, 100.3], device="cuda")
    scale = (top.double() / 127).float().double()
    k = torch.arange(-126, 126, device="cuda").double() + 0.5
    mid = (k[None, :] * scale[:, None]).float()
    X = torch.cat((top[:, None], torch.nextafter(mid, mid + 1), mid, torch.nextafter(mid, mid - 1)), 1)
    code, _, _ = held(numpy(X))
    assert (numpy(culsh.Int8Rows(X).codes)[:, :X.shape[1]] == code).all()


def test_rows_of_numpy_strided_and_misaligned_arrays(culsh):
    X = torch.randn(50, 90, generator=gen(), device="cuda")
    code, scale, _ = held(numpy(X[:, 3:72]))
    for Y in (X[:, 3:72], X[:, 3:72].cpu().numpy(), X.t().contiguous().t()[:, 3:72]):
        rows = culsh.Int8Rows(Y)
        assert (numpy(rows.codes)[:, :69] == code).all() and (rows.scales.cpu().numpy() == scale).all()


def test_parts_make_the_same_rows(culsh):
    X, Q = torch.randn(300, 70, generator=gen(), device="cuda"), torch.randn(9, 70, generator=gen(1), device="cuda")
    rows = culsh.Int8Rows(X)
    wide = torch.zeros(300, 96, dtype=torch.int8, device="cuda")
    wide[:, 7:87] = rows.codes
    again = culsh.Int8Rows.from_parts(wide[:, 7:87], rows.scales, rows.squares, 70)
    assert torch.equal(again.product(Q), rows.product(Q)) and torch.equal(again.dequantize(), rows.dequantize())
    assert torch.equal(rows.product(culsh.Int8Rows(Q)), rows.product(Q))


@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,nq,d", [(1, 1, 1), (300, 1, 128), (129, 17, 100), (1000, 65, 129), (4099, 130, 257), (257, 300, 2048)])
def test_product(culsh, n, nq, d, dtype, metric):
    X, Q = torch.randn(n, d, generator=gen(n), device="cuda"), torch.randn(nq, d, generator=gen(nq), device="cuda")
    X[n // 2] = 0
    out = culsh.Int8Rows(X).product(Q, metric=metric, dtype=dtype)
    assert out.dtype == dtype and out.shape == (nq, n)
    close(out, *expect(held(numpy(Q)), held(numpy(X)), metric), dtype)


def test_product_of_the_largest_sums(culsh):
    """All codes 127: sums beyond 2^24, exact until they are rounded."""
    for d in (1100, 131_072):
        X = torch.ones(3, d, device="cuda")
        X[1] = -1
        rows = culsh.Int8Rows(X)
        assert rows.squares.tolist() == [127 * 127 * d] * 3
        close(rows.product(X[:2]), *expect(held(numpy(X[:2])), held(numpy(X)), "dot"))
        close(rows.product(X[:2], metric="cosine"), *expect(held(numpy(X[:2])), held(numpy(X)), "cosine"))
        offsets = torch.tensor([0, 3], device="cuda")
        close(rows.score(X[:1], (torch.arange(3, dtype=torch.int32, device="cuda"), offsets)), *(v[0] for v in expect(held(numpy(X[:1])), held(numpy(X)), "dot")))


def test_product_of_more_than_two_to_the_31_scores(culsh):
    n, nq, d = 300_001, 8_000, 16
    X, Q = torch.randn(n, d, generator=gen(), device="cuda"), torch.randn(nq, d, generator=gen(1), device="cuda")
    out = culsh.Int8Rows(X).product(Q, dtype=torch.bfloat16)
    at = torch.tensor([0, 1, 4_000, 7_158, 7_159, 7_999], device="cuda")
    close(out[at], *expect(held(numpy(Q[at])), held(numpy(X)), "dot"), torch.bfloat16)


def lists_of(lengths, n, seed=0):
    rng = np.random.default_rng(seed)
    ids = np.concatenate([rng.integers(0, n, k) for k in lengths] + [np.zeros(0, int)]).astype(np.int32)
    return torch.from_numpy(ids).cuda(), torch.from_numpy(np.concatenate(([0], np.cumsum(lengths))).astype(np.int64)).cuda()


@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("d", [1, 16, 17, 100, 128, 500, 513, 1500])
def test_score(culsh, d, dtype, metric):
    n, lengths = 700, [0, 0, 1, 5, 0, 300, 33, 0, 64, 1, 1, 1, 0]
    X, Q = torch.randn(n, d, generator=gen(d), device="cuda"), torch.randn(len(lengths), d, generator=gen(1), device="cuda").to(dtype)
    X[5] = 0
    ids, offsets = lists_of(lengths, n)
    ids[2], ids[7], ids[20] = 5, -1, n
    out = culsh.Int8Rows(X).score(Q, (ids, offsets), metric=metric)
    v, t = expect(held(numpy(Q)), held(numpy(X)), metric)
    owner = np.repeat(np.arange(len(lengths)), lengths)
    at = ids.cpu().numpy()
    real = (at >= 0) & (at < n)
    safe = np.where(real, at, 0)
    close(out, np.where(real, v[owner, safe], np.nan), t[owner, safe])


def test_score_and_rank_of_what_query_returns(culsh):
    X = torch.nn.functional.normalize(torch.randn(3000, 64, generator=gen(), device="cuda"))
    Q = torch.nn.functional.normalize(X[:40] + 0.05 * torch.randn(40, 64, generator=gen(1), device="cuda"))
    rows, found = culsh.Int8Rows(X), culsh.RPLSH(8, 8, seed=1).fit(X).query(Q)
    ids, offsets = found.get_indices(as_torch=True), found.get_offsets(as_torch=True)
    scores = rows.score(Q, found, metric="cosine")
    v, t = expect(held(numpy(Q)), held(numpy(X)), "cosine")
    owner = np.repeat(np.arange(40), np.diff(offsets.cpu().numpy().astype(np.int64)))
    at = ids.cpu().numpy()
    close(scores, v[owner, at], t[owner, at])
    best = culsh.rank(rows, Q, found, top_k=3, metric="cosine", temperature=0.05)
    every = culsh.rank(rows, Q, top_k=3, metric="cosine", temperature=0.05)
    assert torch.equal(every.top_ids[:, 0].long(), torch.arange(40, device="cuda"))
    again = culsh.log_probs(scores, None, found, top_k=3, temperature=0.05)
    assert torch.equal(best.top_ids, again.top_ids) and torch.equal(best.top_log_probs, again.top_log_probs)
    few = culsh.rank(rows, Q, (ids[:0], torch.zeros(41, dtype=torch.int64, device="cuda")), top_k=2)
    assert (few.top_ids == -1).all()


def test_empty_sides(culsh):
    none, rows = culsh.Int8Rows(torch.zeros(0, 20, device="cuda")), culsh.Int8Rows(torch.ones(4, 20, device="cuda"))
    assert none.codes.shape == (0, 32) and none.dequantize().shape == (0, 20) and none.scales.shape == none.squares.shape == (0,)
    assert none.product(torch.ones(3, 20, device="cuda")).shape == (3, 0)
    assert rows.product(torch.zeros(0, 20, device="cuda")).shape == (0, 4)
    ids, offsets = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 2], device="cuda")
    assert torch.isnan(none.score(torch.ones(1, 20, device="cuda"), (ids, offsets))).all()
    assert rows.score(torch.ones(1, 20, device="cuda"), (ids[:0], offsets * 0)).shape == (0,)


def test_work_is_queued_on_the_current_stream_and_in_graphs(culsh):
    X, Q = torch.randn(5000, 100, generator=gen(), device="cuda"), torch.randn(70, 100, generator=gen(1), device="cuda")
    ids, offsets = lists_of([3] * 70, 5000)
    rows = culsh.Int8Rows(X)
    want = rows.product(Q), rows.score(Q, (ids, offsets))
    side = torch.cuda.Stream()
    q = torch.zeros_like(Q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        q.copy_(Q)
        got = rows.product(q), rows.score(q, (ids, offsets))
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = culsh.Int8Rows(X)
        p, s = r.product(q), r.score(q, (ids, offsets))
    for scale in (1.0, 3.0):
        q.copy_(Q * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, rows.product(Q * scale)) and torch.equal(s, rows.score(Q * scale, (ids, offsets)))
    rows.check()


def test_refusals(culsh):
    X = torch.ones(4, 20, device="cuda")
    rows = culsh.Int8Rows(X)
    for bad in (lambda: culsh.Int8Rows(X.int()), lambda: rows.product(X, dtype=torch.float64), lambda: rows.product(X.int()), lambda: rows.dequantize(torch.int8),
                lambda: rows.score(X, (torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda")))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: culsh.Int8Rows(X[0]), lambda: culsh.Int8Rows(X[:, :0]), lambda: rows.product(X[:, :5]), lambda: rows.product(X, metric="l1"),
                lambda: culsh.Int8Rows(torch.empty(1, 131_073, device="cuda")), lambda: rows.score(X, (None, torch.zeros(5, dtype=torch.int64, device="cuda"))),
                lambda: rows.score(X[:3], (torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda"))),
                lambda: culsh.Int8Rows.from_parts(rows.codes[:, :20], rows.scales, rows.squares, 20),
                lambda: culsh.Int8Rows.from_parts(rows.codes, rows.scales[:3], rows.squares, 20),
                lambda: culsh.Int8Rows.from_parts(rows.codes, rows.scales, rows.scales, 20),
                lambda: culsh.Int8Rows.from_parts(rows.codes.cpu(), rows.scales.cpu(), rows.squares.cpu(), 20)):
        with pytest.raises(ValueError):
            bad()
