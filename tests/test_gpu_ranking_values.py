"""Ranking operators at values, orders and sizes where sums of 32 bits, searches and range limits can go wrong, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from test_gpu_ranking import HALF_ULP, ULP, csr, gen, gradient_of, held

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
