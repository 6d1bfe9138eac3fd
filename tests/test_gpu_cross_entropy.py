"""Cross entropy over every row and its gradient against plain forms in 64 bits.

Tolerances count roundings.  A score's sum of d products errs by at most d units (2^-23, the accumulators cut off) of the sum of their magnitudes S, its product with log2(e) / T, the
exponent and the exponential by 2^-23 of |z| each and 2^-22.  Sums of exponentials are of positive terms: 100 additions of 2^-24 cover the longest chain (64 pieces of 32 entries in four parts).
In the gradient p errs by twice a score's error, G is rounded to half a unit of its type, sums over K entries err by K units of the sum of magnitudes (K at most 32,768, or 1,024 in 32 bits),
the result is rounded to half a unit."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -140, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -130}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def culsh():
    import culsh_b200
    return culsh_b200


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def sides(m, n, d, dtype, seed=0, size=1.0):
    X = torch.nn.functional.normalize(torch.randn(n, d, generator=gen(seed), device="cuda")) * size
    Q = torch.nn.functional.normalize(torch.randn(m, d, generator=gen(seed + 1), device="cuda")) * size
    targets = torch.randint(0, n, (m,), generator=gen(seed + 2), device="cuda")
    return Q.to(dtype), X.to(dtype), targets


def plain(Q, X, targets, bias=None, temperature=1.0, g=None, e=None):
    """(z, losses, lse, grad_Q, grad_X, p) in 64 bits."""
    q, x = Q.double(), X.double()
    z = q @ x.T / temperature
    if bias is not None:
        z = torch.where(bias[None, :] == -np.inf, torch.full_like(z, -np.inf), z + bias.double())
    lse = torch.logsumexp(z, 1)
    real = (targets >= 0) & (targets < X.shape[0])
    at = torch.where(real, targets, 0)[:, None].long()
    mine = z.gather(1, at)[:, 0]
    losses = torch.where(real, torch.where(mine == -np.inf, torch.full_like(mine, np.inf), lse - mine), torch.zeros_like(lse))
    if g is None and e is None:
        return z, losses, lse
    p = torch.exp(z - lse[:, None])
    p = torch.where(lse[:, None] == -np.inf, torch.zeros_like(p), p)
    gg = torch.where(real & (mine > -np.inf), 0 * lse + (0 if g is None else g.double()), torch.zeros_like(lse))
    G = p * (gg + (0 if e is None else e.double()))[:, None]
    G.scatter_add_(1, at, -gg[:, None])
    if bias is not None:
        x = torch.where(bias[:, None] == -np.inf, torch.zeros_like(x), x)
    return z, losses, lse, G @ x / temperature, G.T @ q / temperature, p


def score_error(Q, X, z, temperature, bias=None):
    """Of the worst score."""
    x = X.double() if bias is None else torch.where(bias[:, None] == -np.inf, 0.0, X.double())
    s = (Q.double().abs() @ x.abs().T).max() / temperature
    top = z[torch.isfinite(z)].abs().max() if torch.isfinite(z).any() else torch.zeros((), device="cuda")
    b = 0.0 if bias is None else bias[torch.isfinite(bias)].abs().max().item() if torch.isfinite(bias).any() else 0.0
    return float((Q.shape[1] + 8) * ULP * s + 3 * ULP * (top + b))


def check_losses(r, Q, X, targets, bias=None, temperature=1.0):
    z, losses, lse = plain(Q, X, targets, bias, temperature)
    tol = 2 * score_error(Q, X, z, temperature, bias) + 100 * 2.0 ** -24 + 2.0 ** -21
    for got, want in ((r.losses, losses), (r.lse, lse)):
        fine = torch.isfinite(want)
        assert torch.equal(got.double()[~fine], want[~fine])
        off = (got.double() - want)[fine].abs() - 2.0 ** -24 * want[fine].abs()
        assert off.numel() == 0 or float(off.max()) <= tol, (float(off.max()), tol)
    assert (r.losses >= 0).all()
    assert torch.isfinite(r.lse_low).all()


def check_gradients(got, Q, X, targets, bias, temperature, g, e):
    z, _, _, dq, dx, p = plain(Q, X, targets, bias, temperature, g, e)
    m, n, dtype = Q.shape[0], X.shape[0], Q.dtype
    gg, ee = (torch.zeros(m, device="cuda", dtype=torch.float64) if v is None else v.double().abs() for v in (g, e))
    a = (gg + ee)[:, None]
    err = 4 * score_error(Q, X, z, temperature, bias) + 2.0 ** -20
    x = X.double().abs() if bias is None else torch.where(bias[:, None] == -np.inf, 0.0, X.double().abs())
    real = (targets >= 0) & (targets < n)
    at = torch.where(real, targets, 0)[:, None].long()
    own = torch.zeros_like(p).scatter_(1, at, a * real[:, None])  # what goes in apart from p's sums
    # entries of G below half precision's least, where the largest factor is 2^14 or more
    low = float(a.max()) * (2.0 ** -39 if dtype == torch.float16 else 2.0 ** -126)
    most = 1024 if dtype == torch.float32 else 32_768
    half = HALF[dtype]
    for name, out, want, left, right, k in (("dQ", got[0], dq, p * a, x, n), ("dX", got[1], dx, (p * a).T, Q.double().abs(), m)):
        if out is None:
            continue
        assert out.dtype == dtype and out.shape == want.shape
        o = own if name == "dQ" else own.T
        tol = ((err + half + min(k, most) * ULP + k // most * 2.0 ** -24) * (left @ right) + (err + (k + 4) * 2.0 ** -24) * (o @ right) + low * (torch.ones_like(left) @ right)) / temperature
        tol = tol + half * (want.abs() + tol) + 4 * 2.0 ** -24 * want.abs() + LEAST[dtype]
        off = (out.double() - want).abs() - tol
        assert float(off.max()) <= 0, (name, float(off.max()), float(tol.max()))


SHAPES = [(1, 1, 1), (1, 300, 64), (5, 3000, 33), (16, 700, 300), (16, 90_000, 5), (3, 400, 2730), (64, 1000, 100), (130, 257, 128), (129, 513, 31), (300, 70, 520), (2, 5000, 200), (700, 3, 16), (257, 1025, 1100)]


@pytest.mark.parametrize("temperature", [1.0, 0.05])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,d", SHAPES)
def test_losses_and_gradients(culsh, m, n, d, dtype, temperature):
    Q, X, targets = sides(m, n, d, dtype)
    if m > 4:
        targets[1], targets[2], targets[3] = -1, n, n - 1
    r = culsh.cross_entropy(Q, X, targets, temperature=temperature)
    check_losses(r, Q, X, targets, None, temperature)
    g, e = torch.randn(m, generator=gen(5), device="cuda"), 0.1 * torch.randn(m, generator=gen(6), device="cuda")
    grads = culsh.cross_entropy_backward(Q, X, targets, r, g, e, temperature=temperature)
    check_gradients(grads, Q, X, targets, None, temperature, g, e)
    only = culsh.cross_entropy_backward(Q, X, targets, r, g, e, temperature=temperature, rows=False)
    assert only[1] is None and torch.equal(only[0], grads[0])
    only = culsh.cross_entropy_backward(Q, X, targets, r, g, e, temperature=temperature, queries=False)
    assert only[0] is None and torch.equal(only[1], grads[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,d", [(64, 1000, 100), (130, 257, 1100), (3, 5, 7), (70, 600, 64), (200, 300, 256), (12, 2000, 640)])
def test_bias_and_masked_rows(culsh, m, n, d, dtype):
    Q, X, targets = sides(m, n, d, dtype)
    bias = torch.randn(n, generator=gen(7), device="cuda")
    bias[torch.rand(n, generator=gen(8), device="cuda") < 0.3] = -np.inf
    bias[n // 2], targets[0], targets[1] = -np.inf, n // 2, -1
    clean = X.clone()
    X[n // 2] = float("nan")  # what a masked row holds does not count
    X[bias == -np.inf, 0] = float("inf")
    clean[bias == -np.inf] = 0
    r = culsh.cross_entropy(Q, X, targets.int(), bias, temperature=0.1)
    check_losses(r, Q, clean, targets, bias, 0.1)
    assert r.losses[0] == np.inf and r.losses[1] == 0
    g, e = torch.randn(m, generator=gen(5), device="cuda"), torch.randn(m, generator=gen(6), device="cuda")
    for gg, ee in ((g, e), (g, None), (None, e)):
        grads = culsh.cross_entropy_backward(Q, X, targets, r, gg, ee, bias, temperature=0.1)
        check_gradients(grads, Q, clean, targets, bias, 0.1, gg, ee)
        assert not grads[1][bias == -np.inf].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_bias_that_leaves_no_row(culsh, dtype):
    Q, X, targets = sides(5, 300, 40, dtype)
    bias = torch.full((300,), -np.inf, device="cuda")
    targets[2] = -1
    r = culsh.cross_entropy(Q, X, targets, bias)
    assert (r.lse == -np.inf).all() and (r.lse_low == 0).all() and r.losses.tolist() == [np.inf, np.inf, 0, np.inf, np.inf]
    for grad in culsh.cross_entropy_backward(Q, X, targets, r, torch.ones(5, device="cuda"), torch.ones(5, device="cuda"), bias):
        assert not grad.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(culsh, dtype):
    Q, X, targets = sides(140, 300, 40, dtype)
    Q[3, 7], Q[135, 0] = float("nan"), float("inf")
    r = culsh.cross_entropy(Q, X, targets)
    bad = torch.zeros(140, dtype=torch.bool, device="cuda")
    bad[3] = bad[135] = True
    assert torch.isnan(r.lse[bad]).all() and torch.isnan(r.losses[bad]).all() and torch.isfinite(r.lse[~bad]).all()
    ones = torch.ones(140, device="cuda")
    dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, ones)
    assert torch.isnan(dq[bad]).all() and torch.isfinite(dq[~bad]).all() and torch.isnan(dx).all()
    X[200, 0] = float("inf")
    # 16 bits: a score of -inf, which has no part in lse, where the query's first value is negative, else of inf, or NaN.  32 bits: the planes of an infinity are NaN
    assert torch.equal(torch.isnan(culsh.cross_entropy(Q, X, targets).lse), bad | (~(Q[:, 0] < 0) if dtype != torch.float32 else True))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(culsh, dtype):
    """lse of thousands: p comes out as near as from small ones, as lse is held in two parts."""
    m, n, d = 40, 500, 32
    X = torch.randint(-4, 5, (n, d), generator=gen(), device="cuda").to(dtype)  # products and sums are whole numbers, exact in every type
    Q = torch.randint(-4, 5, (m, d), generator=gen(1), device="cuda").to(dtype)
    targets = torch.randint(0, n, (m,), generator=gen(2), device="cuda")
    bias = torch.full((n,), 65536.0, device="cuda")
    for b, t in ((None, 2.0 ** -6), (None, 2.0 ** -4), (bias, 16.0)):
        z, losses, lse = plain(Q, X, targets, b, t)
        r = culsh.cross_entropy(Q, X, targets, b, temperature=t)
        # scores are exact; their product with log2(e) / T is off by 2^-24 of it, the same for all of a row but for the rounding of what is left
        tol = float(z.abs().max()) * 2.0 ** -22 if b is None else 65536 * 2.0 ** -22
        assert float((r.losses.double() - losses).abs().max()) <= tol
        assert float((r.lse.double() + r.lse_low.double() - lse).abs().max()) <= tol
        g = torch.ones(m, device="cuda")
        dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, g, bias=b, temperature=t)
        _, _, _, want_q, want_x, p = plain(Q, X, targets, b, t, g)
        # an error of all p of a query at once would be |lse| 2^-24; what remains is the difference's from the largest score
        gap = float((lse[:, None] - z).clamp(max=60).max()) * ULP + 2.0 ** -20 + (0 if b is None else 65536 * 2.0 ** -22)
        # exponentials below 2^-126 are 0, and in half precision p below 2^-39 (G is scaled to 2^14 and more, its least is 2^-25): of at most 500 entries times 4
        least = 2000 * (2.0 ** -39 if dtype == torch.float16 else 2.0 ** -126) + LEAST[dtype]
        for out, want, size in ((dq, want_q, (p @ X.double().abs()) + X.double().abs()[targets]), (dx, want_x, p.T @ Q.double().abs() + 4.0 * m)):
            off = (out.double() - want).abs() - ((2 * HALF[dtype] + gap) * size + least) / t
            assert float(off.max()) <= 0


def test_gradients_of_targets_that_many_queries_share(culsh):
    for m, n in ((1500, 40), (600, 300), (3000, 2)):
        Q, X, targets = sides(m, n, 48, torch.float32)
        targets[:] = torch.where(torch.rand(m, generator=gen(9), device="cuda") < 0.7, 1, targets)
        r = culsh.cross_entropy(Q, X, targets, temperature=0.2)
        g = torch.randn(m, generator=gen(5), device="cuda")
        check_gradients(culsh.cross_entropy_backward(Q, X, targets, r, g, temperature=0.2), Q, X, targets, None, 0.2, g, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,d", [(33_000, 300, 24), (600, 500, 5_000), (3_000, 40, 300), (2_000, 20_000, 70)])
def test_gradients_of_many_queries_and_of_long_rows(culsh, m, n, d, dtype):
    """More queries than one accumulator takes, targets summed up for some hundred queries at a time, rows in one piece and in several."""
    Q, X, targets = sides(m, n, d, dtype)
    r = culsh.cross_entropy(Q, X, targets, temperature=0.3)
    check_losses(r, Q, X, targets, None, 0.3)
    g, e = torch.randn(m, generator=gen(5), device="cuda"), torch.randn(m, generator=gen(6), device="cuda")
    check_gradients(culsh.cross_entropy_backward(Q, X, targets, r, g, e, temperature=0.3), Q, X, targets, None, 0.3, g, e)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_loss_of_one_row_is_0(culsh, dtype):
    for m, n, d in ((3, 1, 70), (200, 1, 640), (40, 1, 64)):
        Q, X, targets = sides(m, n, d, dtype)
        assert not culsh.cross_entropy(Q, X, targets, temperature=0.3).losses.any()
        assert not culsh.cross_entropy(Q, X, targets, torch.full((1,), 0.7, device="cuda"), temperature=0.3).losses.any()
    Q, X, targets = sides(50, 900, 96, dtype)
    bias = torch.full((900,), -np.inf, device="cuda")
    bias[17] = -3.3
    r = culsh.cross_entropy(Q, X, torch.full_like(targets, 17), bias)
    assert not r.losses.any()


def test_another_thread_and_a_first_call_in_a_graph(culsh):
    """A handle of its own for each thread; a shape that is new when it is captured."""
    import threading
    Q, X, targets = sides(90, 700, 48, torch.float16)
    g = torch.ones(90, device="cuda")
    want = culsh.cross_entropy(Q, X, targets, temperature=0.2)
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            r = culsh.cross_entropy(Q, X, targets, temperature=0.2)
            got[i] = (*r, *culsh.cross_entropy_backward(Q, X, targets, r, g, temperature=0.2), culsh.Int8Rows(X).product(Q))
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4
    for out in got.values():
        assert torch.equal(out[0], want.losses) and all(torch.equal(a, b) for a, b in zip(out, got[0]))
    q, x = Q[:33, :40].float().contiguous(), X[:, :40].float().contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = culsh.cross_entropy(q, x, targets[:33], temperature=0.4)
        grads = culsh.cross_entropy_backward(q, x, targets[:33], r, g[:33], temperature=0.4)
    graph.replay()
    torch.cuda.synchronize()
    check_losses(r, q, x, targets[:33], None, 0.4)
    check_gradients(grads, q, x, targets[:33], None, 0.4, g[:33], None)


def test_nearly_certain_targets(culsh):
    """p of the target next to 1: its coefficient is a small difference, which is not rounded with it."""
    for dtype in TYPES:
        Q, X, targets = sides(60, 60, 64, dtype)
        Q, targets = X.clone(), torch.arange(60, device="cuda")
        g = torch.ones(60, device="cuda")
        r = culsh.cross_entropy(Q, X, targets, temperature=0.06)
        z, losses, lse, dq, dx, p = plain(Q, X, targets, None, 0.06, g)
        assert float(losses.max()) < 0.05
        out = culsh.cross_entropy_backward(Q, X, targets, r, g, temperature=0.06)
        # errors by what is left of p: 1 - p(target)
        left = 1 - p.diagonal()
        err = HALF[dtype] + 4 * score_error(Q, X, z, 0.06) + 2.0 ** -20
        off = (out[0].double() - dq).abs() - (3 * err * left[:, None] * 2 + 2.0 ** -21) / 0.06 - LEAST[dtype] - HALF[dtype] * dq.abs()
        assert float(off.max()) <= 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_against_differences(culsh, dtype):
    """Of the losses in 64 bits, along a few directions: central differences at h and h / 2, whose errors go with h^2."""
    m, n, d, t = 20, 70, 12, 0.5
    Q, X, targets = sides(m, n, d, dtype)
    g = torch.randn(m, generator=gen(5), device="cuda")
    r = culsh.cross_entropy(Q, X, targets, temperature=t)
    dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, g, temperature=t)

    def total(q, x):
        return float((plain(q, x, targets, None, t)[1] * g.double()).sum())

    for side, grad in ((0, dq), (1, dx)):
        for seed in range(3):
            D = torch.randn(grad.shape, generator=gen(20 + seed), device="cuda", dtype=torch.float64)
            args = [Q.double(), X.double()]

            def along(h):
                lo, hi = list(args), list(args)
                lo[side], hi[side] = args[side] - h * D, args[side] + h * D
                return (total(*hi) - total(*lo)) / (2 * h)
            a, b = along(1e-3), along(5e-4)
            exact = b + (b - a) / 3
            tol = abs(b - a) + 1e-9 + (2 * HALF[dtype] + 2.0 ** -18) * float((D.abs() * (grad.double().abs() + 2 * g.abs().double().sum() / t / (n if side else 1))).sum())
            assert abs(float((grad.double() * D).sum()) - exact) <= tol


def test_pieces_strides_and_misaligned_rows(culsh):
    """Enough queries that the rows are taken in several pieces, and rows that TMA cannot take as they are."""
    m, n, d = 20_000, 3_000, 24
    for dtype, pad in ((torch.bfloat16, 0), (torch.bfloat16, 1), (torch.float16, 8), (torch.float32, 3)):
        Q, X, targets = sides(m, n, d, dtype)
        q, x = torch.zeros(m, d + pad, dtype=dtype, device="cuda")[:, :d], torch.full((n, d + pad), float("nan"), dtype=dtype, device="cuda")[:, :d]
        q.copy_(Q), x.copy_(X)
        r = culsh.cross_entropy(q, x, targets, temperature=0.3)
        check_losses(r, Q, X, targets, None, 0.3)
        g = torch.randn(m, generator=gen(5), device="cuda") / m
        check_gradients(culsh.cross_entropy_backward(q, x, targets, r, g, temperature=0.3), Q, X, targets, None, 0.3, g, None)
        same = culsh.cross_entropy(Q, X, targets, temperature=0.3)
        assert all(torch.equal(a, b) for a, b in zip(r, same))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_same_call_gives_the_same_bits(culsh, dtype):
    Q, X, targets = sides(700, 9_000, 128, dtype)
    targets[::3] = 5
    first = None
    for _ in range(3):
        r = culsh.cross_entropy(Q, X, targets, temperature=0.1)
        out = (*r, *culsh.cross_entropy_backward(Q, X, targets, r, torch.ones(700, device="cuda"), torch.ones(700, device="cuda"), temperature=0.1))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_work_is_queued_on_the_current_stream_and_in_graphs(culsh):
    Q, X, targets = sides(200, 4_000, 100, torch.bfloat16)
    g = torch.full((200,), 0.005, device="cuda")

    def step(q, x):
        r = culsh.cross_entropy(q, x, targets, temperature=0.1)
        return (*r, *culsh.cross_entropy_backward(q, x, targets, r, g, temperature=0.1))

    want = step(Q, X)
    streams, q = [torch.cuda.Stream(), torch.cuda.Stream()], torch.zeros_like(Q)
    torch.cuda.synchronize()
    got = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            torch.cuda._sleep(10_000_000)
            mine = torch.zeros_like(Q)
            mine.copy_(Q)
            got.append(step(mine, X))
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, X)
    for scale in (1.0, 0.5):
        q.copy_(Q * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(Q * scale, X)))


def test_empty_calls(culsh):
    X = torch.randn(7, 5, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    r = culsh.cross_entropy(X[:0], X, none)
    assert all(v.shape == (0,) for v in r)
    dq, dx = culsh.cross_entropy_backward(X[:0], X, none, r, torch.zeros(0, device="cuda"))
    assert dq.shape == (0, 5) and dx.shape == (7, 5) and not dx.any()


def test_an_encoder_trained_against_every_row_and_served_from_8_bits(culsh):
    """Loss, gradients, an update of a linear encoder, rows and queries in 8 bits, ranking."""
    n, m, d = 3_000, 256, 64
    X = torch.nn.functional.normalize(torch.randn(n, d, generator=gen(), device="cuda"))
    targets = torch.randint(0, n, (m,), generator=gen(1), device="cuda")
    inputs = X[targets] + 0.05 * torch.randn(m, d, generator=gen(2), device="cuda")
    W = torch.eye(d, device="cuda") + 0.02 * torch.randn(d, d, generator=gen(3), device="cuda")
    Q = inputs @ W.T
    r = culsh.cross_entropy(Q, X, targets, temperature=0.1)
    g = torch.full((m,), 1.0 / m, device="cuda")
    dq, dx = culsh.cross_entropy_backward(Q, X, targets, r, g, temperature=0.1)
    check_gradients((dq, dx), Q, X, targets, None, 0.1, g, None)
    w = W.double().requires_grad_()
    torch.nn.functional.cross_entropy(inputs.double() @ w.T @ X.double().T / 0.1, targets).backward()
    dw = dq.T @ inputs
    assert float((dw.double() - w.grad).norm()) <= 1e-4 * float(w.grad.norm())
    rows, Q = culsh.Int8Rows(X), inputs @ (W - 0.1 * dw).T
    best = culsh.rank(rows, Q, top_k=1, targets=targets, temperature=0.1)
    assert torch.equal(best.top_ids[:, 0].long(), targets)
    z = culsh.Int8Rows(Q).dequantize(torch.float64) @ rows.dequantize(torch.float64).T / 0.1
    want = torch.log_softmax(z, 1).gather(1, targets[:, None])[:, 0]
    assert float((best.log_probs.double() - want).abs().max()) <= 2.0 ** -18


def test_refusals(culsh):
    Q, X, targets = sides(4, 9, 20, torch.float32)
    r = culsh.cross_entropy(Q, X, targets)
    one = torch.ones(4, device="cuda")
    for bad in (lambda: culsh.cross_entropy(Q.double(), X.double(), targets), lambda: culsh.cross_entropy(Q, X.half(), targets), lambda: culsh.cross_entropy(Q, X, targets, torch.zeros(9, device="cuda").half()),
                lambda: culsh.cross_entropy_backward(Q, X, targets, r, one.double())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: culsh.cross_entropy(Q[0], X, targets), lambda: culsh.cross_entropy(Q, X[:, :5], targets), lambda: culsh.cross_entropy(Q, X[:0], targets),
                lambda: culsh.cross_entropy(Q, X, targets[:3]), lambda: culsh.cross_entropy(Q, X, None), lambda: culsh.cross_entropy(Q, X, targets.float()),
                lambda: culsh.cross_entropy(Q, X, targets, torch.zeros(8, device="cuda")), lambda: culsh.cross_entropy(Q, X, targets, temperature=0.0),
                lambda: culsh.cross_entropy(Q[:, :0], X[:, :0], targets), lambda: culsh.cross_entropy_backward(Q, X, None, r, one),
                lambda: culsh.cross_entropy_backward(Q, X, targets, r, one[:3]), lambda: culsh.cross_entropy_backward(Q[:3], X, targets[:3], r, one[:3])):
        with pytest.raises(ValueError):
            bad()


def test_sizes_beyond_an_index_are_refused(culsh):
    import ctypes as C

    from culsh_b200 import _lib
    from culsh_b200._culsh_core import get_handle
    h, need = get_handle(0), C.c_uint64()
    for m, n, d in ((2 ** 31 - 1, 5, 1), (5, 2 ** 31 - 1, 1), (5, 5, 65_537), (0, 5, 5)):
        assert h.lib.culsh_cross_entropy_workspace(h.ptr, 16, 65_537, 16, 65_537, 0, m, n, d, 0, 3, C.byref(need)) == -1
    assert h.lib.culsh_cross_entropy_workspace(h.ptr, 16, 4, 16, 4, 1, 5, 5, 4, 0, 3, C.byref(need)) == -1 and b"float" in _lib.load().culsh_last_error()
