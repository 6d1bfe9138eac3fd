"""Cross entropy where a rounding in the wrong place shows: lse of tens of thousands, temperatures near either end, long rows, very many queries."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -140, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -130}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def culsh():
    import culsh_b200
    return culsh_b200


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,d", [(64, 4_891, 300), (64, 4_891, 512), (64, 4_891, 1_321), (32, 37_633, 862), (20, 30_000, 600)])
def test_losses_of_small_calls_are_as_near_as_floats(culsh, m, n, d, dtype):
    """Scores of about 8, in segments of 128 values whose 8 adds cut off half a unit of 2^-23 of a sum that is half as large on average: 8 x 2^-25 x 8 = 2e-6, of which a target's loss keeps the share
    of the other rows, and of a mean loss of 1 to 3, 1e-6 of it."""
    t = 0.05
    X = torch.nn.functional.normalize(torch.randn(n, d, generator=gen(1), device="cuda"))
    targets = torch.randint(0, n, (m,), generator=gen(2), device="cuda")
    Q = torch.nn.functional.normalize(X[targets] + torch.randn(m, d, generator=gen(3), device="cuda") * (2.5 / d ** 0.5)).to(dtype)
    X = X.to(dtype)
    r = culsh.cross_entropy(Q, X, targets, temperature=t)
    z = Q.double() @ X.double().T / t
    want = torch.logsumexp(z, 1) - z.gather(1, targets[:, None])[:, 0]
    assert float((r.losses.double() - want).norm() / want.norm()) <= 1e-6


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,d", [(16, 64), (20, 64), (20, 128), (20, 256), (20, 300), (20, 700)])
@pytest.mark.parametrize("far", [40, 256, -256])
def test_gradients_do_not_go_with_the_rounding_of_lse(culsh, far, m, d, bias, dtype):
    """Scores of whole numbers of up to 65,548, exact in every type, times log2(e) / T = c, which is a float and no power of two: lse is next to no float (its last bit is up to 2^-7).  Columns of
    the gradients are single entries of G: dX[j, 1 + i] and dQ[i, 1 + m + j].

    p is exp2 of a difference that is exact (of no bias: rounded once), off by 2^-22, by a factor that is rounded once, and lse's sum by 24 additions and exponentials of 2^-22: 2^-19 together.
    G is rounded to its type, and the result: half a unit each."""
    n, c = 24, float(np.float32(1.371))
    t = 1.4426950408889634 / c
    Q, X = torch.zeros(m, d, device="cuda"), torch.zeros(n, d, device="cuda")
    Q[:, 0], X[:, 0] = far, 256
    i, j = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    Q[:, 1 + m:1 + m + n] = torch.randint(-3, 4, (m, n), generator=gen(1), device="cuda").float()
    X[:, 1:1 + m] = torch.randint(-3, 4, (n, m), generator=gen(2), device="cuda").float()
    Q[i, 1 + i], X[j, 1 + m + j] = 1, 1
    Q, X = Q.to(dtype), X.to(dtype)
    targets = torch.randint(0, n, (m,), generator=gen(3), device="cuda")
    targets[::3] = -1
    b = 0.5 * torch.randn(n, generator=gen(4), device="cuda") if bias else None
    two = Q.double() @ X.double().T * c
    if bias:  # exponents are floats
        two = (two + (b * np.float32(1.4426950408889634)).double()).float().double()
    p = torch.softmax(two * np.log(2.0), 1)
    g, e = torch.randn(m, generator=gen(5), device="cuda"), 1 + torch.rand(m, generator=gen(6), device="cuda")
    real = targets >= 0
    gg = torch.where(real, g.double(), 0.0)
    G = p * (gg + e.double())[:, None]
    G[i[real], targets[real]] -= gg[real]
    r = culsh.cross_entropy(Q, X, targets, b, temperature=t)
    dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, g, e, b, temperature=t)
    size = p * (gg.abs() + e.double())[:, None]
    size[i[real], targets[real]] += gg.abs()[real]
    # a target's loss is rounded: its p by |loss| 2^-24
    err = 2 * HALF[dtype] + HALF[dtype] ** 2 + 2.0 ** -19 + 40 * 2.0 ** -24
    tol = (err * size + 4 * 2.0 ** -39) / t + LEAST[dtype]
    for out in (dq[i[:, None], 1 + m + j[None, :]], dx[j[None, :], 1 + i[:, None]]):
        off = (out.double() - G / t).abs() - tol
        assert float(off.max()) <= 0, (float(off.max()), float(((out.double() * t - G).abs() / size).max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [128, 300])
def test_gradients_of_16_bits_are_off_by_the_rounding_of_the_result(culsh, d, dtype):
    """G is rounded to 16 bits: what that leaves in a sum is at most half a unit of the root of its terms' squares (independent roundings), beside the result's rounding, and sums in 32 bits."""
    m, n, t = 1_000, 20_000, 0.05
    X = torch.nn.functional.normalize(torch.randn(n, d, generator=gen(), device="cuda"))
    targets = torch.randint(0, n, (m,), generator=gen(1), device="cuda")
    Q = torch.nn.functional.normalize(X[targets] + torch.randn(m, d, generator=gen(2), device="cuda") * (2.5 / d ** 0.5)).to(dtype)
    X, g, e = X.to(dtype), 1 + 0.2 * torch.randn(m, generator=gen(3), device="cuda"), 0.01 * torch.randn(m, generator=gen(4), device="cuda")
    r = culsh.cross_entropy(Q, X, targets, temperature=t)
    out = culsh.cross_entropy_backward(Q, X, targets, r, g, e, temperature=t)
    P = torch.softmax(Q.double() @ X.double().T / t, 1) * (g + e).double()[:, None]
    G = P.scatter_add(1, targets[:, None], -g.double()[:, None])
    P.scatter_(1, targets[:, None], 0.0)
    for got, want, rest in ((out[0], G @ X.double() / t, (P ** 2 @ X.double() ** 2).sqrt() / t), (out[1], G.T @ Q.double() / t, ((P ** 2).T @ Q.double() ** 2).sqrt() / t)):
        once = (want.to(dtype).double() - want).norm()
        assert float((got.double() - want).norm()) <= float(once + HALF[dtype] * rest.norm() + 2.0 ** -20 * want.norm())
    again = culsh.cross_entropy_backward(Q, X, targets, r, g, e, temperature=t)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [700, 2_048, 16_384, 65_536])
def test_p_of_long_rows_sum_up_to_1(culsh, d, dtype):
    """Scores of about 40 from positive products, of which accumulators cut off something at every step: in one sum over K a score of 65,536 products would be 3e-4 of itself smaller than in the
    losses' segments of 512, and all p with it 1e-2.  Columns of the gradients are single entries of G, as above.

    A query's G, half a unit of rounding each and half a unit of the results, sum up to the gradient of lse, as scores are taken as in the losses' pass.  Each entry: segments of 32 adds that cut off
    2^-23 and their sum's roundings, twice."""
    m, n = 20, 24
    Q, X = 0.5 + torch.rand(m, d, generator=gen(1), device="cuda"), 0.5 + torch.rand(n, d, generator=gen(2), device="cuda")
    i, j = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    Q[:, :m + n], X[:, :m + n] = 0, 0
    Q[i, i], X[j, m + j] = 16, 16
    Q, X = Q.to(dtype), X.to(dtype)
    t = float((Q.double() @ X.double().T).mean()) / 40
    e, targets = 1 + torch.rand(m, generator=gen(3), device="cuda"), torch.full((m,), -1, device="cuda")
    r = culsh.cross_entropy(Q, X, targets, temperature=t)
    dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, None, e, temperature=t)
    z = Q.double() @ X.double().T / t
    want = torch.softmax(z, 1) * e.double()[:, None]
    score = float(z.max()) * (33 * 2.0 ** -23 + d / 512 * 2.0 ** -24) + 2.0 ** -20
    assert float((r.lse.double() - torch.logsumexp(z, 1)).abs().max()) <= score + 2.0 ** -24 * float(r.lse.max())
    err = 2 * HALF[dtype] + HALF[dtype] ** 2 + 2.0 ** -18
    for out in (dq[:, m:m + n], dx[:, :m].T):
        G = out.double() * t / 16
        assert float((G.sum(1) / e.double() - 1).abs().max()) <= err
        assert float((G / want - 1).abs().max()) <= 2 * score + err


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,d", [(3, 700, 40), (20, 70, 40), (70, 1000, 100), (20, 300, 300), (140, 90, 600)])
@pytest.mark.parametrize("temperature,size", [(1e-30, 1e-15), (1e30, 1.0), (7e37, 1e30), (1e38, 1e30), (1e38, 1.0), (1.9e45, 1e30), (3e45, 1e36), (1e60, 1e36), (1e80, 1.0), (1e300, 1e36), (1e300, 1e38)])
def test_temperatures_of_any_magnitude(culsh, temperature, size, m, n, d, dtype):
    """Scores that are all next to 0: the loss is log(n).  One over the temperature, and log2(e) by it, are no floats of all their bits from 8e37 on, and none at all from 2e45 on.  `size`: of the
    rows, so that the gradient of the queries is a number of its type where it can be one."""
    if dtype == torch.float16:
        size = min(max(size, 2.0 ** -6), 2.0 ** 12)
        if temperature < 1:
            temperature = 2.0 ** -10
    Q = (torch.rand(m, d, generator=gen(1), device="cuda") - 0.5) * (size if temperature < 1 else 1.0)
    X = (torch.rand(n, d, generator=gen(2), device="cuda") - 0.5) * size
    Q, X = Q.to(dtype), X.to(dtype)
    targets = torch.randint(0, n, (m,), generator=gen(3), device="cuda")
    g, e = torch.randn(m, generator=gen(4), device="cuda"), torch.randn(m, generator=gen(5), device="cuda")
    r = culsh.cross_entropy(Q, X, targets, temperature=temperature)
    q, x = Q.double(), X.double()
    z = q @ x.T / temperature
    lse = torch.logsumexp(z, 1)
    score = float((q.abs() @ x.abs().T).max()) / temperature * (d + 8) * 2.0 ** -23 + 2.0 ** -18
    if float((q.abs() @ x.abs().T).max()) > 2.0 ** 127:  # the scores themselves, before they are divided, may be no floats: the query has no numbers then
        fine = (q.abs() @ x.abs().T).max(1).values < 2.0 ** 127
        assert not fine.any() or float((r.lse.double() - lse).abs()[fine].max()) <= score
        return
    assert float((r.lse.double() - lse).abs().max()) <= score and float((r.losses.double() - (lse - z.gather(1, targets[:, None])[:, 0])).abs().max()) <= 2 * score
    dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, g, e, temperature=temperature)
    P = torch.softmax(z, 1) * (g + e).double()[:, None]
    G = P.scatter_add(1, targets[:, None], -g.double()[:, None])
    size_of = P.abs().scatter_add(1, targets[:, None], g.double().abs()[:, None])
    err = 2 * HALF[dtype] + 4 * score + (m + n) * 2.0 ** -23
    least = LEAST[dtype] + (2.0 ** -37 * float((g + e).abs().max()) * float(x.abs().max() + q.abs().max()) * (m + n) / temperature if dtype == torch.float16 else 0)
    for out, want, tol in ((dq, G @ x / temperature, size_of @ x.abs() / temperature), (dx, G.T @ q / temperature, size_of.T @ q.abs() / temperature)):
        fine = want.abs() + tol * err < torch.finfo(dtype).max / 2
        off = (out.double() - want).abs() - (tol * err + least)
        assert not torch.isnan(out).any() and float(off[fine].max()) <= 0, (float(off[fine].max()), float(want.abs().max()))


def test_the_workspace_does_not_grow_with_both_sides(culsh):
    """Sums that are split over the other side lie there for as many queries or rows as 256 MB hold: with a copy of what the queries and rows need each, a small multiple of the inputs."""
    import ctypes as C

    from culsh_b200._culsh_core import get_handle
    h, need = get_handle(0), C.c_uint64()
    for m, n, d in ((4_096, 1_000_000, 128), (32_768, 1_000_000, 128), (1_000_000, 1_000_000, 128), (1_000_000, 10_000_000, 128), (10_000_000, 1_000_000, 256), (50_000_000, 1_000_000, 8)):
        for has_bias in (0, 1):
            assert h.lib.culsh_cross_entropy_workspace(h.ptr, 16, d, 16, d, 3, m, n, d, has_bias, 3, C.byref(need)) == 0
            # 512 MB of sums; planes of the rows, where there is a bias; sums of the targets' rows, of 32 bits; terms of queries, and up to 16 places for each row
            assert need.value <= (512 << 20) + (2 * d * n if has_bias else 0) + 4 * d * m + 16 * (m + 128) + 68 * (n + 128) + 8192, (m, n, d, need.value)


@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, False), (torch.float16, True), (torch.float16, False)])
@pytest.mark.parametrize("m,n,d", [(32_768, 20_000, 40), (32_769, 20_000, 40), (40_001, 700, 200), (300_001, 500_003, 16), (70_000, 260_001, 200)])
def test_gradients_of_very_many_queries(culsh, m, n, d, dtype, bias):
    """More queries than a sum takes, and more of both sides than the workspace holds sums of at a time: a few of the rows of each gradient against 64 bits.  Tolerances: a score errs by d + 8
    units of the sum of its magnitudes (1 / t), p by twice that; G by half a unit, sums of 32,768 entries by as many cut-off units of 2^-23 of their magnitudes; the result by half a unit."""
    t = 0.2
    X = torch.nn.functional.normalize(torch.randn(n, d, generator=gen(1), device="cuda")).to(dtype)
    Q = torch.nn.functional.normalize(torch.randn(m, d, generator=gen(2), device="cuda")).to(dtype)
    targets = torch.randint(0, n, (m,), generator=gen(3), device="cuda")
    some_rows = torch.tensor([0, 1, 127, 128, n // 2, n - 2, n - 1], device="cuda")
    some = torch.tensor([0, 5, 127, 128, 32_767, m // 2, m - 2, m - 1], device="cuda")
    targets[::7] = some_rows[torch.randint(0, 7, targets[::7].shape, generator=gen(4), device="cuda")]
    b = None
    if bias:
        b = torch.randn(n, generator=gen(5), device="cuda")
        b[5::11] = -np.inf
        b[some_rows] = 0.5
    g, e = torch.randn(m, generator=gen(6), device="cuda"), 0.1 * torch.randn(m, generator=gen(7), device="cuda")
    r = culsh.cross_entropy(Q, X, targets, b, temperature=t)
    dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, g, e, b, temperature=t)
    q, x, add = Q.double(), X.double(), 0.0 if b is None else b.double()
    masked = torch.zeros(m, dtype=torch.bool, device="cuda") if b is None else b[targets] == -np.inf
    gg = torch.where(masked, 0.0, g.double())
    f, own = gg + e.double(), torch.where(masked, 0.0, -g.double())
    # of some queries
    z = q[some] @ x.T / t + add
    lse = torch.logsumexp(z, 1)
    score = (d + 8) * 2.0 ** -23 * 1.02 / t + 6 * 2.0 ** -23 * 8
    assert float((r.lse[some].double() - lse).abs().max()) <= 2 * score + 2.0 ** -16
    p = torch.exp(z - lse[:, None])
    G = p * f[some][:, None]
    one = torch.zeros_like(G).scatter_(1, targets[some][:, None], own[some][:, None])
    err = 4 * score + 2.0 ** -16 + HALF[dtype] + 32_768 * 2.0 ** -23 + (m + n) // 32_768 * 2.0 ** -24
    low = 2.0 ** -39 * float(f.abs().max()) if dtype == torch.float16 else 0.0

    def check(out, want, size, ones):
        tol = (err * size + low * ones) / t
        off = (out.double() - want).abs() - (tol + HALF[dtype] * (want.abs() + tol) + LEAST[dtype])
        assert float(off.max()) <= 0, (float(off.max()), float(tol.max()))

    check(dq[some], (G + one) @ x / t, (G.abs() + one.abs()) @ x.abs(), torch.ones_like(G) @ x.abs())
    # of some rows
    z = q @ x[some_rows].T / t + (0.0 if b is None else b.double()[some_rows])
    G = torch.exp(z - (r.lse.double() + r.lse_low.double())[:, None]) * f[:, None]
    one = (targets[:, None] == some_rows[None, :]) * own[:, None]
    check(dx[some_rows], (G + one).T @ q / t, (G.abs() + one.abs()).T @ q.abs(), torch.ones_like(G).T @ q.abs())
    if b is not None:
        assert not dx[5::11][b[5::11] == -np.inf].any()
    only = culsh.cross_entropy_backward(Q, X, targets, r, g, e, b, temperature=t, queries=False)[1]
    assert torch.equal(only, dx)
    assert torch.equal(culsh.cross_entropy_backward(Q, X, targets, r, g, e, b, temperature=t, rows=False)[0], dq)


def test_no_wait_ran_out(culsh):
    Q, X = torch.randn(300, 100, generator=gen(), device="cuda"), torch.randn(900, 100, generator=gen(1), device="cuda")
    targets = torch.randint(0, 900, (300,), generator=gen(2), device="cuda")
    r = culsh.cross_entropy(Q, X, targets)
    culsh.cross_entropy_backward(Q, X, targets, r, torch.ones(300, device="cuda"))
    r.check()


def test_scores_of_few_queries_are_sums_of_sums(culsh):
    """Scores of 40 from 960 positive products.  A rounding is uniform within half a unit, 2^-25.2 of a sum that grows evenly: of one sum over all of them the root of the squares' mean is
    40 x 2^-25.2 x sqrt(960 / 3) = 1.9e-5, of 30 sums of 32 and their sum 40 x 2^-25.2 x sqrt(30 / 3) = 3e-6, beside the loss's own rounding and exponentials of 2^-22."""
    n, d = 300, 960
    X = 0.5 + torch.rand(n, d, generator=gen(2), device="cuda")
    off = []
    for seed in range(16):
        Q, targets = 0.5 + torch.rand(1, d, generator=gen(10 + seed), device="cuda"), torch.full((1,), 7 * seed, device="cuda")
        t = float((Q.double() @ X.double().T).mean()) / 40
        z = Q.double() @ X.double().T / t
        off.append(float(culsh.cross_entropy(Q, X, targets, temperature=t).losses.double()[0] - (torch.logsumexp(z, 1) - z[:, 7 * seed])[0]))
    assert float(np.sqrt(np.mean(np.square(off)))) <= 8e-6
