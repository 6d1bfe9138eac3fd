"""Rows in 8 bits of any magnitude: products of two scales, and squares of one, may leave float32 where the score does not."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_ULP = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
MOST = {torch.float32: 2.0 ** 128, torch.float16: 65520.0, torch.bfloat16: 2.0 ** 128}
MAGNITUDES = [1e-42, 1e-37, 1e-30, 1e-21, 1e-20, 1e-19, 1e-17, 1e-9, 1.0, 1e9, 1e13, 1e15, 1e18, 2e21, 1e25, 1e30, 1e38]


@pytest.fixture(scope="module")
def culsh():
    import culsh_b200
    return culsh_b200


def sides(n, nq, d):
    g = torch.Generator(device="cuda").manual_seed(n + nq + d)
    X, Q = torch.rand(n, d, generator=g, device="cuda") * 2 - 1, torch.rand(nq, d, generator=g, device="cuda") * 2 - 1
    X *= torch.tensor(MAGNITUDES, device="cuda")[torch.arange(n, device="cuda") % len(MAGNITUDES)][:, None]
    Q *= torch.tensor(MAGNITUDES, device="cuda")[(7 * torch.arange(nq, device="cuda") + 14) % len(MAGNITUDES)][:, None]
    k = min(n, nq)
    Q[:k:3] = X[:k:3]             # distances of 0
    X[n // 2:n // 2 + 5, ::2] = 0    # products of 0 with these queries
    if nq > 2:
        Q[nq // 2:nq // 2 + 3, 1::2] = 0
        Q[1] = 0
    X[n // 3] = 0
    return X, Q


def expect(rows, queries, metric):
    """Scores in 64 bits of what is held, and their tolerance: the sum, the scales' product, and the product of both are rounded, distances also squares, terms and differences."""
    cq, cx = queries.codes.double(), rows.codes.double()
    sq, sx = queries.scales.double()[:, None], rows.scales.double()[None, :]
    v = (cq @ cx.T) * (sq * sx)
    if metric == "dot":
        return v, 4 * U * v.abs() + 2.0 ** -148
    q2, x2 = (cq * cq).sum(1)[:, None] * sq * sq, (cx * cx).sum(1)[None, :] * sx * sx
    return 2 * v - q2 - x2, 8 * U * (2 * v.abs() + q2 + x2) + 2.0 ** -146


def close(out, want, tol, dtype):
    tol = tol + HALF_ULP[dtype] * (want.abs() + tol) + LEAST[dtype]
    assert not torch.isnan(out).any()
    beyond = want.abs() - tol >= MOST[dtype]  # the score itself is
    assert torch.equal(out[beyond].double(), torch.sign(want[beyond]) * np.inf)
    fine = want.abs() + tol < MOST[dtype]
    off = (out.double() - want).abs()[fine] - tol[fine]
    assert float(off.max()) <= 0, (float(off.max()), float(want[fine].abs()[off.argmax()]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("metric", ["dot", "euclidean"])
@pytest.mark.parametrize("n,nq,d", [(300, 1, 100), (300, 17, 100), (300, 50, 300), (300, 90, 100), (500, 100, 300), (300, 200, 100), (600, 300, 300)])
def test_products_of_any_magnitude(culsh, n, nq, d, metric, dtype):
    X, Q = sides(n, nq, d)
    rows, queries = culsh.Int8Rows(X), culsh.Int8Rows(Q)
    close(rows.product(Q, metric=metric, dtype=dtype), *expect(rows, queries, metric), dtype)


@pytest.mark.parametrize("d", [10, 100, 300, 1_000])
@pytest.mark.parametrize("metric", ["dot", "euclidean"])
def test_scores_of_any_magnitude(culsh, metric, d):
    n, nq = 400, 70
    X, Q = sides(n, nq, d)
    rows, queries = culsh.Int8Rows(X), culsh.Int8Rows(Q)
    g = torch.Generator(device="cuda").manual_seed(d)
    ids = torch.randint(0, n, (nq * 60,), generator=g, device="cuda", dtype=torch.int32)
    ids[::60] = torch.arange(nq, device="cuda", dtype=torch.int32)
    owner = torch.arange(nq, device="cuda").repeat_interleave(60)
    want, tol = expect(rows, queries, metric)
    out = rows.score(Q, (ids, torch.arange(0, nq * 60 + 1, 60, device="cuda")), metric=metric)
    close(out, want[owner, ids.long()], tol[owner, ids.long()], torch.float32)


def test_ordinary_scores_beside_far_ones_are_the_same(culsh):
    """A row of another magnitude takes its neighbours' scores another way: dot products come out by the same roundings but for the order of powers of two."""
    g = torch.Generator(device="cuda").manual_seed(1)
    X, Q = torch.randn(256, 64, generator=g, device="cuda"), torch.randn(100, 64, generator=g, device="cuda")
    for queries in (Q[:5], Q[:40], Q):
        want = culsh.Int8Rows(X).product(queries)
        far = X.clone()
        far[::9] *= 1e-30
        got = culsh.Int8Rows(far).product(queries)
        near = torch.ones(256, dtype=torch.bool, device="cuda")
        near[::9] = False
        assert torch.equal(got[:, near], want[:, near])
