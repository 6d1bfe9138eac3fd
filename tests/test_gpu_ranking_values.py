"""Ranking operators at values, orders and sizes where sums of 32 bits, searches and range limits can go wrong, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from test_gpu_ranking import HALF_ULP, ULP, gen, gradient_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def culsh():
    import culsh_b200
    return culsh_b200


def answer_of(s, temperature):
    """(lse, entropy, log p, sum of p (log p - largest log p)^2) of float64 scores, from what they are below the largest."""
    d = (s - s.max()) / temperature
    total = np.exp(d).sum()
    lp = d - math.log(total)
    p = np.exp(lp)
    return s.max() / temperature + math.log(total), -np.where(p > 0, p * lp, 0).sum(), lp, (p * np.where(p > 0, d * d, 0)).sum()


# ---- scores of any size ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1000, 80_000])  # one CTA a row, and several
@pytest.mark.parametrize("temperature", [1.0, 0.05])
@pytest.mark.parametrize("top", [1e6, -1e6, 1e8, -1e8, 3e8, -3e8, -2.7e9, 5e9, -5e9, 1e20, -1e20])
def test_log_probs_of_large_scores(culsh, top, temperature, n, dtype):
    """Ties, near ties, sums that start far below the largest, and ones that rise step by step."""
    g = torch.Generator().manual_seed(n)
    top = float(torch.tensor(top).to(dtype))
    step = abs(top) * float(torch.finfo(dtype).eps)  # at least the distance to the next value
    s = torch.full((5, n), top, dtype=torch.float64)
    s[1] -= step * torch.randint(0, 5, (n,), generator=g)
    s[1, n // 2] = top
    s[2] = torch.where(torch.rand(n, generator=g) < 0.01, top, top - abs(top) / 2)
    s[2, n - 1] = top
    s[3] = torch.linspace(top - abs(top), top, n, dtype=torch.float64)
    s[4] = torch.linspace(top, -abs(top) * 2, n, dtype=torch.float64)
    s = s.to(dtype).cuda()
    targets = torch.tensor([n - 1, n // 2, n - 1, n - 1, 0], device="cuda")
    r = culsh.log_probs(s, targets, top_k=3, temperature=temperature)
    for i in range(5):
        z = s[i].double().cpu().numpy()
        lse, entropy, lp, square = answer_of(z, temperature)
        # a difference to the largest errs by some units of itself, so sums err by that times what it is on average, and by a unit for each of the terms that a lane adds;
        # log of the sum of exponentials by units of the largest, too
        few = ULP * (32 + 4 * math.log(n))
        assert abs(float(r.lse[i]) - lse) <= few + 4 * ULP * abs(lse), (i, float(r.lse[i]), lse)
        assert abs(float(r.entropy[i]) - entropy) <= few + 4 * ULP * square, (i, float(r.entropy[i]), entropy)
        t = int(targets[i])
        assert abs(float(r.log_probs[i]) - lp[t]) <= few + 4 * ULP * abs(lp[t]), (i, float(r.log_probs[i]), lp[t])
        order = np.lexsort((np.arange(n), -z))[:3]
        assert r.top_ids[i].tolist() == order.tolist()
        assert np.all(np.abs(r.top_log_probs[i].double().cpu().numpy() - lp[order]) <= few + 4 * ULP * np.abs(lp[order]))


# ---- lists in any order ---------------------------------------------------------------------------------------------
def mixed(lengths, n, order, seed):
    """Lists of distinct ids: ascending, ascending but for the last one, descending, or shuffled."""
    rng = np.random.RandomState(seed)
    lists = []
    for m in lengths:
        mine = np.cumsum(rng.randint(1, max(n // max(m, 1), 1) + 1, m)) - 1  # distinct and below n
        if order == "last" and m > 1:  # a positive behind ascending negatives
            at = rng.randint(m - 1)
            mine = np.append(np.delete(mine, at), mine[at])
        elif order == "down":
            mine = mine[::-1]
        elif order == "any":
            mine = rng.permutation(mine)
        lists.append(mine)
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64))
    return torch.from_numpy(np.concatenate(lists).astype(np.int32)).cuda(), offsets.cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("order", ["last", "down", "any"])
@pytest.mark.parametrize("lengths", [[31, 0, 32, 33, 64, 1, 65, 0, 2, 129, 1000, 2050, 7], [64] * 600, [50_000, 0, 3, 70_001], [300_000] + [40] * 2000, [40] * 9 + [3] * 20_000,
                                     [3000] * 200, [20_000] * 300, [100_000] + [3] * 1000, [70_000, 90_001, 80_002]])
def test_targets_of_lists_in_any_order(culsh, lengths, order, dtype):
    n, temperature = 3 * max(lengths), 0.5
    all_ids, offsets = mixed(lengths, n, order, 5)
    m, total = len(lengths), all_ids.shape[0]
    for lead in (0, 1, 3):  # ids and scores that begin off a boundary, too
        ids = torch.cat([all_ids[:lead], all_ids])[lead:]
        s = torch.randn(total + lead, generator=gen(3), device="cuda").to(dtype)[lead:]
        ends = offsets.tolist()
        if order == "last":
            at = [max(k - 1, 0) for k in lengths]
        else:
            at = [(7 * i + 3) % k if k else 0 for i, k in enumerate(lengths)]
        targets = torch.tensor([n + 1 if i % 6 == 5 or not k else int(v) for i, (k, v) in enumerate(zip(
            lengths, ids.cpu()[(offsets[:-1].cpu() + torch.tensor(at)).clamp(max=total - 1)]))], device="cuda")
        r = culsh.log_probs(s, targets, (ids, offsets), temperature=temperature)
        gl, ge = torch.randn(m, generator=gen(6), device="cuda"), torch.randn(m, generator=gen(7), device="cuda")
        got = culsh.log_probs_backward(s, targets, r.lse, r.entropy, gl, ge, (ids, offsets), temperature)
        got, z, lp = got.double().cpu().numpy(), s.double().cpu().numpy(), r.log_probs.double().cpu().numpy()
        t = targets.tolist()
        for i in sorted(set(range(min(m, 20))) | {m - 1}):
            k = lengths[i]
            if not k:
                assert lp[i] == -math.inf
                continue
            mine = z[ends[i]:ends[i + 1]]
            place = None if t[i] > n else at[i]
            _, _, want, _ = answer_of(mine, temperature)
            tol = ULP * (32 + 4 * math.log(max(k, 2)))
            assert lp[i] == -math.inf if place is None else abs(lp[i] - want[place]) <= tol + 4 * ULP * abs(want[place]), (i, lp[i])
            # p errs by what log p does, of its own size; entropy and log p of no more than 100 by h p
            a, h = float(gl[i]), float(ge[i])
            grad = gradient_of(mine / temperature, place, a, h, temperature)
            bound = 8 * ULP * 64 * (abs(a) + 64 * abs(h)) / temperature + HALF_ULP[dtype] * np.abs(grad) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
            assert np.all(np.abs(got[ends[i]:ends[i + 1]] - grad) <= bound), i


def test_rank_finds_targets_among_candidates_in_any_order(culsh):
    n, nq, mean = 5000, 50, 400
    X, Q = torch.randn(n, 64, generator=gen(), device="cuda"), torch.randn(nq, 64, generator=gen(1), device="cuda")
    rows = culsh.MXRows(X)
    up, offsets = mixed([mean] * nq, n, "up", 2)
    ids = up.view(nq, mean)[:, torch.randperm(mean, generator=gen(3), device="cuda")].reshape(-1)
    targets = ids[offsets[:-1] + 7].long()
    a = culsh.rank(rows, Q, (up, offsets), top_k=5, metric="cosine", temperature=0.1, targets=targets)
    b = culsh.rank(rows, Q, (ids, offsets), top_k=5, metric="cosine", temperature=0.1, targets=targets)
    assert bool(torch.isfinite(b.log_probs).all())
    assert torch.allclose(a.log_probs, b.log_probs, rtol=0, atol=1e-4)  # float32 scores of other lanes and sums
    assert torch.equal(a.top_ids, b.top_ids)


# ---- gradients of scores of any size --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 0.05])
@pytest.mark.parametrize("m,n,pad", [(7, 1, 0), (6, 20, 1), (9, 1000, 0), (5, 1003, 5), (3, 70_001, 0), (2000, 130, 0), (1, 300_000, 3)])
@pytest.mark.parametrize("lists", [False, True])
def test_gradient_of_large_scores(culsh, lists, m, n, pad, temperature, dtype):
    """Scores around squared distances of bytes: p comes from the scores' differences, whatever their size, and a row's gradient sums to nothing."""
    g = gen(m + n)
    near = {torch.float32: -2.0e5, torch.float16: -6.0e4, torch.bfloat16: -2.0e5}[dtype]
    if dtype == torch.float32:
        s = near + 3 * temperature * torch.randn(m, n + pad, generator=g, device="cuda")
    else:  # whole steps of the type; most of p lies at the largest few
        s = near - abs(near) * float(torch.finfo(dtype).eps) * torch.randint(0, 3, (m, n + pad), generator=g, device="cuda")
    s[::3] -= near  # rows of ordinary size among them
    if n > 4:
        s[:, 2] = -math.inf
    s = s.to(dtype)[:, pad // 2:pad // 2 + n]
    t = torch.randint(0, n, (m,), generator=g, device="cuda")
    if m > 4:
        t[4] = -1
    gl, ge = torch.randn(m, generator=g, device="cuda"), torch.randn(m, generator=g, device="cuda")
    if lists:
        lengths = torch.full((m,), n, device="cuda")
        offsets = torch.zeros(m + 1, dtype=torch.int64, device="cuda")
        offsets[1:] = torch.cumsum(lengths, 0)
        ids = (2 * torch.arange(n, device="cuda", dtype=torch.int32)).repeat(m)
        flat = torch.cat([s.new_zeros(pad), s.reshape(-1)])[pad:]
        r = culsh.log_probs(flat, 2 * t, (ids, offsets), temperature=temperature)
        got = culsh.log_probs_backward(flat, 2 * t, r.lse, r.entropy, gl, ge, (ids, offsets), temperature).view(m, n)
    else:
        r = culsh.log_probs(s, t, temperature=temperature)
        got = culsh.log_probs_backward(s, t, r.lse, r.entropy, gl, ge, temperature=temperature)
    for i in sorted(set(range(min(m, 12))) | {m - 1}):
        z = s[i].double().cpu().numpy()
        place = int(t[i]) if 0 <= int(t[i]) < n and z[int(t[i])] > -math.inf else None
        want = gradient_of((z - z.max(initial=-1e30)) / temperature if np.any(z > -math.inf) else z, place, float(gl[i]), float(ge[i]), temperature)
        a, h = abs(float(gl[i])), abs(float(ge[i]))
        mine = got[i].double().cpu().numpy()
        bound = 8 * ULP * 64 * (a + 64 * h) / temperature  # log p errs by no more than some units of 64, whatever the scores; entropy and log p below 64
        assert np.all(np.abs(mine - want) <= bound + HALF_ULP[dtype] * np.abs(want) + (2.0 ** -25 if dtype == torch.float16 else 0.0)), i
        if dtype == torch.float32:
            assert abs(mine.sum()) * temperature <= ULP * (64 + 4 * math.log(n + 1)) * 8 * (a + 64 * h), i


def test_gradient_takes_the_lse_that_it_is_given(culsh):
    """An lse that is not these scores' own, of rows that other processes hold parts of: p is what it says."""
    s = 100 + torch.randn(4, 500, generator=gen(), device="cuda")
    t, gl = torch.arange(4, device="cuda"), torch.ones(4, device="cuda")
    lse = torch.logsumexp(s, 1) + 1.0
    got = culsh.log_probs_backward(s, t, lse, torch.zeros(4, device="cuda"), gl)
    want = -torch.exp(s.double() - lse.double()[:, None])
    want[torch.arange(4), t] += 1
    assert bool(((got.double() - want).abs() <= 8 * ULP * 128).all())


@pytest.mark.parametrize("lists", [False, True])
@pytest.mark.parametrize("g,h", [(1e4, 1.0), (-3e5, 2.0), (1e-3, 1.0), (1e6, 0.5)])
def test_gradient_of_an_entry_that_is_nearly_certain(culsh, g, h, lists):
    """What the entropy's gradient adds there is small beside what goes into it and stays, however large the other gradient is."""
    n = 60
    s = torch.full((3, n), -14.0, device="cuda")
    s[:, 7] = 0.0
    s[1, 8:] = -20.0
    s[2, 8] = -3.0
    t = torch.full((3,), 7, device="cuda")
    gl, ge = torch.full((3,), g, device="cuda"), torch.full((3,), h, device="cuda")
    csr_of = (torch.arange(n, device="cuda", dtype=torch.int32).repeat(3), torch.arange(4, device="cuda") * n) if lists else None
    scores = s.reshape(-1) if lists else s
    r = culsh.log_probs(scores, t, csr_of)
    got = culsh.log_probs_backward(scores, t, r.lse, r.entropy, gl, ge, csr_of).view(3, n)
    for i in range(3):
        z, lse, entropy = s[i].double().cpu().numpy(), float(r.lse[i]), float(r.entropy[i])  # of what the call is given
        lp = z[7] - lse
        first, second = -g * math.expm1(lp), -h * math.exp(lp) * (lp + entropy)
        # each part to some units of what goes into it
        assert abs(float(got[i, 7]) - (first + second)) <= 4 * ULP * abs(first) + 8 * ULP * h * (abs(lp) + entropy), (i, float(got[i, 7]), first, second)


# ---- graphs, results that go ----------------------------------------------------------------------------------------
def test_candidates_in_a_graph(culsh):
    """The engine's stream stays out of the graph, and works on meanwhile and behind it."""
    rng = np.random.RandomState(3)
    X = rng.randn(4000, 32).astype(np.float32)
    near = X[:100] + 0.05 * rng.randn(100, 32).astype(np.float32)
    model = culsh.RPLSH(8, 8, seed=0).fit(X)
    cand = model.query(near)
    rows, Q = culsh.MXRows(X), torch.from_numpy(near).cuda()
    t = torch.arange(100, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        culsh.rank(rows, Q, cand, top_k=5, metric="cosine", targets=t)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = culsh.rank(rows, Q, cand, top_k=5, metric="cosine", targets=t)
        s = rows.score(Q, cand)
        grad = culsh.log_probs_backward(s, t, r.lse, r.entropy, torch.ones(100, device="cuda"), lists=cand)
    again = model.query(near)
    assert np.array_equal(again.get_indices(), cand.get_indices())
    for seed in (1, 2):
        Q.copy_(torch.randn(100, 32, generator=gen(seed), device="cuda"))
        graph.replay()
        want = culsh.rank(rows, Q, cand, top_k=5, metric="cosine", targets=t)
        assert torch.equal(r.top_ids, want.top_ids) and torch.equal(r.lse, want.lse) and torch.equal(r.log_probs, want.log_probs)
        one = rows.score(Q, cand)
        assert torch.equal(s, one)
        assert torch.equal(grad, culsh.log_probs_backward(one, t, want.lse, want.entropy, torch.ones(100, device="cuda"), lists=cand))


@pytest.mark.parametrize("what", ["score", "log_probs", "backward", "rank"])
def test_results_that_go_before_they_are_read(culsh, what):
    """Work that reads a result waits behind long work of its stream when the result goes and queries of the same size take its memory."""
    rng = np.random.RandomState(5)
    X = rng.randn(20_000, 64).astype(np.float32)
    Q = X[:3000] + 0.1 * rng.randn(3000, 64).astype(np.float32)
    other = Q[::-1].copy()
    model = culsh.RPLSH(8, 10, seed=0).fit(X)
    rows, Qd = culsh.MXRows(X), torch.from_numpy(Q).cuda()
    kept = model.query(Q)
    t = torch.arange(3000, device="cuda")
    scores = rows.score(Qd, kept, metric="cosine")
    r = culsh.log_probs(scores, t, kept, temperature=0.1)
    ones = torch.ones(3000, device="cuda")
    calls = {"score": lambda c: (rows.score(Qd, c, metric="cosine"),),
             "log_probs": lambda c: culsh.log_probs(scores, t, c, top_k=4, temperature=0.1),
             "backward": lambda c: (culsh.log_probs_backward(scores, t, r.lse, r.entropy, ones, ones, c, 0.1),),
             "rank": lambda c: culsh.rank(rows, Qd, c, top_k=4, metric="cosine", targets=t)}
    want = [x.clone() for x in calls[what](kept)]
    big = torch.randn(8000, 8000, device="cuda")
    torch.cuda.synchronize()
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    for _ in range(3):
        cand = model.query(Q)
        with torch.cuda.stream(side):
            x = big
            for _ in range(8):
                x = x @ big * 1e-2  # some milliseconds each in float32
            got = calls[what](cand)
            done.record(side)
        pending = not done.query()
        del cand
        again = [model.query(other) for _ in range(2)]
        side.synchronize()
        assert pending, "the work in front was done too soon to show anything"
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del again


@pytest.mark.parametrize("d,lead", [(77, 1), (33, 3), (130, 0)])
def test_calls_behind_one_another_on_changing_lists(culsh, d, lead):
    """As for whole rows: odd lengths, scores off the boundaries, ids, offsets and targets that change from call to call in the same memory, long lists."""
    n, nq, total = 30_000, 20, 20 * 60_000
    g = gen(d)
    sets = []
    for i in range(3):
        ends = torch.sort(torch.randint(0, total, (nq - 1,), generator=g, device="cuda")).values
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), ends, torch.full((1,), total, device="cuda")])
        ids = torch.randint(0, n, (total,), generator=g, device="cuda").int()
        targets = ids[(offsets[:-1] + 17 * i).clamp(max=total - 1)].long()
        sets.append((torch.randn(n, d, generator=g, device="cuda"), torch.randn(nq, d, generator=g, device="cuda"), ids, offsets, targets,
                     torch.randn(5, 100_003 + lead, generator=g, device="cuda")))
    X, Q, ids, offsets, targets, wide = (x.clone() for x in sets[0])
    held = torch.zeros(n, d + 1, device="cuda")[:, 1:]  # rows off the boundaries

    def step(given):
        for to, of in zip((X, Q, ids, offsets, targets, wide), given):
            to.copy_(of)
        held.copy_(X)
        rows = culsh.MXRows(held)
        s = rows.score(Q, (ids, offsets), metric="cosine")
        r = culsh.log_probs(s, targets, (ids, offsets), top_k=5, temperature=0.2)
        one = culsh.log_probs(wide[:, lead:], targets[:5], top_k=6)
        p = rows.product(Q[:, :], metric="euclidean")
        return s, r.lse, r.entropy, r.log_probs, r.top_ids, one.lse, one.log_probs, one.top_ids, culsh.log_probs(p[:3], top_k=3).top_ids

    want = []
    for given in sets:
        want.append([x.clone() for x in step(given)])
        torch.cuda.synchronize()
    got = [(i % 3, step(sets[i % 3])) for i in range(45)]
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


# ---- scores by few and by many candidates ---------------------------------------------------------------------------
def few_and_many(rows, Q, n, metric):
    """Scores of every row for each query, by a call of few candidates and by one of many (of which all rounds are alike)."""
    nq, times = Q.shape[0], 60_000 // n + 1
    ids = torch.arange(n, dtype=torch.int32, device="cuda")
    few = torch.stack([rows.score(Q[i:i + 1], (ids, torch.tensor([0, n], device="cuda")), metric=metric) for i in range(nq)])
    many = rows.score(Q, (ids.repeat(nq * times), torch.arange(nq + 1, device="cuda") * n * times), metric=metric).view(nq, times, n)
    assert torch.equal(many.nan_to_num(nan=7e37), many[:, :1].expand_as(many).nan_to_num(nan=7e37))
    return few, many[:, 0]


@pytest.mark.parametrize("metric", ["dot", "cosine", "euclidean"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_scores_of_queries_that_are_not_finite(culsh, dtype, metric):
    n, d = 70, 96
    X = torch.randn(n, d, generator=gen(), device="cuda")
    X[3] = 0
    X[4, :32] = 0
    Q = torch.randn(7, d, generator=gen(1), device="cuda").to(dtype)
    Q[1, 5], Q[2, 40], Q[3, 95] = math.inf, -math.inf, math.nan
    Q[4, 0], Q[4, 1] = math.inf, -math.inf
    bad = [1, 2, 3, 4]
    if dtype == torch.float64:
        Q[5, 9] = 1e300  # beyond 32 bits, which queries are taken in
        bad.append(5)
    for scores in few_and_many(culsh.MXRows(X), Q, n, metric):
        for i in range(7):
            assert bool(scores[i].isnan().all()) if i in bad else bool(scores[i].isfinite().all()), i


@pytest.mark.parametrize("metric", ["dot", "euclidean"])
def test_scores_beyond_float32(culsh, metric):
    n, d = 64, 64
    X = torch.randn(n, d, generator=gen(), device="cuda")
    X[::2] *= 2.0 ** 60
    Q = torch.randn(2, d, generator=gen(1), device="cuda") * 2.0 ** 70
    Q[1] *= 2.0 ** -70
    rows = culsh.MXRows(X)
    q, x = Q.double(), rows.dequantize(torch.float64)
    want, size = q @ x.T, q.abs() @ x.abs().T
    if metric == "euclidean":
        q2, x2 = (q * q).sum(1)[:, None], (x * x).sum(1)[None]
        want, size = 2 * want - q2 - x2, 2 * size + q2 + x2
    beyond, within = want.abs() > 2.0 ** 128, size < 2.0 ** 127  # in between a sum may pass the type before it comes back
    assert bool(beyond[0].any()) and bool(within[1].any())
    for scores in few_and_many(rows, Q, n, metric):
        assert not bool(scores.isinf().any())
        assert bool(scores[beyond].isnan().all())
        ok = ~scores.isnan()
        assert bool(ok[within].all()) and bool(((scores.double() - want).abs() <= (d + 4) * ULP * size)[ok].all())


@pytest.mark.parametrize("size", [-60, -64, -66, -90, -110, -120])
@pytest.mark.parametrize("law", ["alike", "wide"])
def test_scores_of_small_queries(culsh, size, law):
    """Queries of values around 2^size: as exact by many candidates as by few, against rows that pick single values out and rows that sum them."""
    d = n = 64
    X = torch.cat([torch.eye(32, d, device="cuda"), torch.randn(n - 32, d, generator=gen(), device="cuda")])
    X[40:] *= 2.0 ** 40
    Q = torch.randn(4, d, generator=gen(1), device="cuda")
    if law == "wide":
        Q *= torch.exp2(torch.randint(-5, 6, (4, d), generator=gen(2), device="cuda").float())
    Q *= 2.0 ** size
    Q[3] = 0
    Q[3, 5] = 3 * 2.0 ** -149  # the smallest ones there are
    rows = culsh.MXRows(X)
    x, q = rows.dequantize(torch.float64), Q.double()
    want, bound = q @ x.T, (d + 2) * ULP * (q.abs() @ x.abs().T)
    # products of the smallest numbers with 0.5 are cut to whole steps of 2^-149 before the scale
    least = 2.0 ** -149 * d * x.abs().amax(1)[None, :].clamp(min=1)
    for scores in few_and_many(rows, Q, n, "dot"):
        assert bool(((scores.double() - want).abs() <= bound + least).all())


# ---- lengths --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nq", [8, 80])  # rows or queries on the M side
@pytest.mark.parametrize("d", [96, 200, 1000, 2500])
def test_cosines_of_rows_of_any_length(culsh, d, nq):
    """Right where squares of lengths are floats, NaN where they are not, 0 for zeros."""
    sizes = [-140, -100, -80, -70, -50, -20, 0, 30, 50, 70, 100]
    g = gen(nq)
    size = lambda n: torch.exp2(torch.tensor([float(sizes[i % len(sizes)]) for i in range(n)], device="cuda"))[:, None]  # noqa: E731
    X, Q = torch.randn(66, d, generator=g, device="cuda") * size(66), torch.randn(nq, d, generator=g, device="cuda") * size(nq)
    X[5] = 0
    Q[6] = 0
    X[16, 1:] = 0  # one value of 2^0 or so
    rows = culsh.MXRows(X)
    x = rows.dequantize(torch.float64)
    x2 = (x * x).sum(1)
    assert torch.equal(rows.norms == 0, x2 == 0) and torch.equal(rows.norms.isinf(), x2 > 2.0 ** 128)

    def check(scores, q):
        q2 = (q * q).sum(1)
        dot, many = q @ x.T, q.abs() @ x.abs().T
        length = q2.sqrt()[:, None] * x2.sqrt()[None, :]
        fits = lambda v: (v >= 2.0 ** -126) & (v < 2.0 ** 128) | (v == 0)  # noqa: E731
        ok = fits(q2)[:, None] & fits(x2)[None, :]
        assert torch.equal(~scores.isnan(), ok)
        want = torch.where(length > 0, dot / length, torch.zeros_like(dot))
        bound = torch.where(length > 0, (2 * d + 10) * ULP * many / length, torch.zeros_like(dot))
        assert bool(((scores.double() - want).abs() <= bound)[ok].all())

    held = culsh.MXRows(Q)
    check(rows.product(Q, metric="cosine"), held.dequantize(torch.float64))
    check(rows.product(held, metric="cosine"), held.dequantize(torch.float64))
    for scores in few_and_many(rows, Q, 66, "cosine"):
        check(scores, Q.double())


@pytest.mark.parametrize("temperature", [1.0, 0.05])
@pytest.mark.parametrize("lengths", [[100_000] + [3] * 1000, [3] * 40 + [1] + [5000] * 30, [400_000, 7, 0, 2_000] + [30] * 900])
def test_gradient_of_large_scores_of_uneven_lists(culsh, lengths, temperature):
    """Targets in no order, in some lists not there, scores around squared distances of bytes in every other list."""
    m, n = len(lengths), 3 * max(lengths)
    ids, offsets = mixed(lengths, n, "any", 9)
    ends, total = offsets.tolist(), ids.shape[0]
    owner = torch.repeat_interleave(torch.arange(m, device="cuda"), torch.tensor(lengths, device="cuda"))
    s = 3 * temperature * torch.randn(total, generator=gen(1), device="cuda") - torch.where(owner % 2 == 0, 2.0e5, 0.0)
    at = [(7 * i + 3) % k if k else 0 for i, k in enumerate(lengths)]
    mine = ids.cpu()[(offsets[:-1].cpu() + torch.tensor(at)).clamp(max=total - 1)].tolist()
    t = torch.tensor([n + 1 if i % 5 == 4 or not lengths[i] else v for i, v in enumerate(mine)], device="cuda")
    gl, ge = torch.randn(m, generator=gen(6), device="cuda"), torch.randn(m, generator=gen(7), device="cuda")
    r = culsh.log_probs(s, t, (ids, offsets), temperature=temperature)
    got = culsh.log_probs_backward(s, t, r.lse, r.entropy, gl, ge, (ids, offsets), temperature).double().cpu().numpy()
    z = s.double().cpu().numpy()
    for i in list(range(min(m, 45))) + [m - 2, m - 1]:
        if not lengths[i]:
            continue
        one = z[ends[i]:ends[i + 1]]
        a, h = float(gl[i]), float(ge[i])
        want = gradient_of((one - one.max()) / temperature, None if int(t[i]) > n else at[i], a, h, temperature)
        bound = 8 * ULP * 64 * (abs(a) + 64 * abs(h)) / temperature + HALF_ULP[torch.float32] * np.abs(want)
        assert np.all(np.abs(got[ends[i]:ends[i + 1]] - want) <= bound), i


@pytest.mark.parametrize("lengths", [[20_000] * 50, [700] * 30, [90_000] * 3])
def test_lists_in_a_graph(culsh, lengths):
    """Kernels that begin beside the one in front of them, replayed on changing scores and targets."""
    m, total = len(lengths), sum(lengths)
    ids, offsets = mixed(lengths, 3 * max(lengths), "any", 1)
    s, t = torch.randn(total, generator=gen(1), device="cuda"), ids[offsets[:-1] + 5].long()
    gl = torch.randn(m, generator=gen(2), device="cuda")

    def step():
        r = culsh.log_probs(s, t, (ids, offsets), top_k=4, temperature=0.1)
        return r.lse, r.entropy, r.log_probs, r.top_ids, culsh.log_probs_backward(s, t, r.lse, r.entropy, gl, gl, (ids, offsets), 0.1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        s.copy_(torch.randn(total, generator=gen(seed + 5), device="cuda") - (2e5 if seed == 2 else 0))
        t.copy_(torch.where(torch.arange(m, device="cuda") % 3 == seed, 10 ** 9, ids[offsets[:-1] + 7 * seed + 1].long()))
        graph.replay()
        torch.cuda.synchronize()
        first = [x.clone() for x in got]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(first, want))
        assert bool(torch.isfinite(want[2]).any()) and bool((want[2] == -math.inf).any())
