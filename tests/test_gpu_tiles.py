"""Forms of tiles that small calls do not reach: 256 rows with a bias or with K in segments, several pieces of rows, 8-bit tiles of 256 rows for 65 to 128 queries, more tiles than CTAs; and
gradients whose rows lie apart.  Plain forms and tolerances are those of the operators' other tests."""
import ctypes as C

import numpy as np
import pytest
import torch

from test_gpu_cross_entropy import check_gradients, check_losses, gen, sides
from test_gpu_int8_rows import close, expect, held, numpy

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def culsh():
    import culsh_b200
    return culsh_b200


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,d", [(300, 9_000, 100), (100, 12_000, 100), (100, 12_003, 600), (300, 9_001, 640), (300, 9_001, 2_200), (4_099, 20_000, 300), (130, 40_000, 61)])
def test_losses_and_gradients_of_large_tiles(culsh, m, n, d, bias, dtype):
    Q, X, targets = sides(m, n, d, dtype)
    targets[1], targets[2] = -1, n - 1
    b, clean = None, X
    if bias:
        b = torch.randn(n, generator=gen(7), device="cuda")
        b[torch.rand(n, generator=gen(8), device="cuda") < 0.3] = -np.inf
        b[n // 2], b[n - 1], targets[0] = -np.inf, 0.25, n // 2
        clean = X.clone()
        clean[b == -np.inf] = 0
        X[n // 2] = float("nan")
    r = culsh.cross_entropy(Q, X, targets, b, temperature=0.1)
    check_losses(r, Q, clean, targets, b, 0.1)
    g, e = torch.randn(m, generator=gen(5), device="cuda"), torch.randn(m, generator=gen(6), device="cuda")
    grads = culsh.cross_entropy_backward(Q, X, targets, r, g, e, b, temperature=0.1)
    check_gradients(grads, Q, clean, targets, b, 0.1, g, e)
    if bias:
        assert not grads[1][b == -np.inf].any()
    r.check()


@pytest.mark.parametrize("metric", ["dot", "cosine", "euclidean"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,nq,d", [(5_000, 100, 300), (5_003, 128, 260), (60_001, 70, 300), (25_000, 300, 300), (30_000, 300, 100), (30_001, 257, 33), (100_001, 40, 130)])
def test_products_of_more_tiles_than_ctas(culsh, n, nq, d, dtype, metric):
    X, Q = torch.randn(n, d, generator=gen(n), device="cuda"), torch.randn(nq, d, generator=gen(nq), device="cuda")
    X *= torch.exp2(torch.randint(-6, 7, (n, 1), generator=gen(1), device="cuda").float())
    Q *= torch.exp2(torch.randint(-6, 7, (nq, 1), generator=gen(2), device="cuda").float())
    X[n // 2] = 0
    out = culsh.Int8Rows(X).product(Q, metric=metric, dtype=dtype)
    # held in 32 bits at least: float16 scores beyond 65,504 are infinities
    want, tol = expect(held(numpy(Q)), held(numpy(X)), metric)
    if dtype == torch.float16:
        far = np.abs(want) - tol > 65_520
        assert (np.abs(numpy(out)[far]) == np.inf).all()
        near = np.abs(want) + tol < 65_500
        close(out[torch.from_numpy(near).cuda()], want[near], tol[near], dtype)
    else:
        close(out, want, tol, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,d", [(300, 9_000, 100), (40, 500, 64), (300, 700, 304), (5, 3_000, 100), (70, 900, 33)])
@pytest.mark.parametrize("apart", [8, 13])
def test_gradients_whose_rows_lie_apart(culsh, apart, m, n, d, dtype):
    """The same numbers as in rows that do not, and nothing else is written."""
    from culsh_b200 import _lib
    from culsh_b200._culsh_core import get_handle
    Q, X, targets = sides(m, n, d, dtype)
    r = culsh.cross_entropy(Q, X, targets, temperature=0.1)
    g = torch.randn(m, generator=gen(5), device="cuda")
    want = culsh.cross_entropy_backward(Q, X, targets, r, g, temperature=0.1)
    h, need, type_ = get_handle(0), C.c_uint64(), {torch.float32: 0, torch.float16: 2, torch.bfloat16: 3}[dtype]
    _lib.check(h.lib.culsh_cross_entropy_workspace(h.ptr, Q.data_ptr(), d, X.data_ptr(), d, type_, m, n, d, 0, 3, C.byref(need)))
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    wide = [torch.full((k, d + apart), 7.0, dtype=dtype, device="cuda") for k in (m, n)]
    _lib.check(h.lib.culsh_cross_entropy_backward(h.ptr, Q.data_ptr(), d, X.data_ptr(), d, type_, m, n, d, targets.data_ptr(), None, 0.1, *(v.data_ptr() for v in r), g.data_ptr(), None,
                                                  wide[0].data_ptr(), d + apart, wide[1].data_ptr(), d + apart, work.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream))
    for got, same in zip(wide, want):
        assert torch.equal(got[:, :d], same) and (got[:, d:] == 7).all()
