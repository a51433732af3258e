"""f32 products whose 128 x 64 tiles take several rounds of blocks, in all transpose forms, with and without a remainder of K."""
import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from ferrox_amd import capi
    with capi.Context(0) as c:
        yield c


@pytest.mark.parametrize("m,k,n", [(3000, 192, 3000), (3000, 260, 3000), (2999, 132, 2997), (5000, 128, 2000)])
def test_products_of_several_rounds(ctx, m, k, n):
    rng = np.random.default_rng(m + k)
    A, B = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    y, _, bound, _ = ref.linear_fwd(A, B, None, "none", None)
    for ta, tb in ((False, True), (False, False), (True, False), (True, True)):
        got = ctx.gemm(ctx.upload(A.T if ta else A), ctx.upload(B.T if tb else B), ta, tb).numpy()
        assert (np.abs(got - y) <= bound).all(), (ta, tb)


@pytest.mark.parametrize("m,k,n", [(4092, 192, 1020), (4090, 260, 1021), (4095, 132, 1023), (8192, 128, 900)])
def test_epilogue_in_128_x_64_tiles(ctx, m, k, n):
    rng = np.random.default_rng(m + k)
    A, B = rng.standard_normal((m, k)).astype(np.float32), (rng.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32)
    bias, res = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n)).astype(np.float32)
    for (ta, tb), act in zip(((False, True), (False, False), (True, False), (True, True)), ("gelu", "none", "silu", "relu")):
        pre = ctx.empty((m, n))
        got = ctx.gemm_bias_act_residual(ctx.upload(A.T if ta else A), ctx.upload(B.T if tb else B), ta, tb, bias=ctx.upload(bias), act=act,
                                         residual=ctx.upload(res), pre=pre).numpy()
        y, p, by, bp = ref.linear_fwd(A, B, bias, act, res)
        assert (np.abs(got - y) <= by).all() and (np.abs(pre.numpy() - p) <= bp).all(), (ta, tb, act)
