"""RMS norm of rows whose squares leave the type's range at either end, forward and backward, beside ordinary rows.  The plain form is in
long double (15 bits of exponent)."""
import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from ferrox_amd import capi
    with capi.Context(0) as c:
        yield c


SCALES = {np.float32: [1e18, 1e20, 1e30, 1e37, 1e-18, 1e-20, 1e-25, 1e-30, 1.0], np.float64: [1e150, 1e160, 1e250, 1e306, 1e-150, 1e-160, 1e-200, 1e-290, 1.0]}


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("eps", [0.0, 1e-6, "tiny"])
@pytest.mark.parametrize("dim", [5, 256, 1001, 3000, 9001, 17000])
def test_rows_of_all_sizes(ctx, dim, eps, dtype):
    rng = np.random.default_rng(dim)
    eps = float(dtype(1e-37 if dtype == np.float32 else 1e-300)) if eps == "tiny" else eps
    scales = np.array(SCALES[dtype])[:, None]
    x = (rng.uniform(0.5, 1, (len(scales), dim)) * rng.choice([-1, 1], (len(scales), dim)) * scales).astype(dtype)
    w = (1 + 0.1 * rng.standard_normal(dim)).astype(dtype)
    _, y, r = ctx.rmsnorm_fwd(ctx.upload(x), ctx.upload(w), eps)
    wide = x.astype(np.longdouble)
    want_r = 1 / np.sqrt((wide * wide).mean(1) + np.longdouble(eps))
    want = wide * want_r[:, None] * w
    rel = ref.rmsnorm_rel(dim, dtype)
    low = float(np.finfo(dtype).smallest_subnormal)
    assert (np.abs(r.numpy() - want_r) <= rel * want_r + low).all()
    assert (np.abs(y.numpy() - want) <= np.abs(want) * (rel + 3 * ref.u(dtype)) + low).all()
    # with the residual in front: the same numbers from halves
    h, y2, _ = ctx.rmsnorm_fwd(ctx.upload(x / 2), ctx.upload(w), eps, res=ctx.upload(x / 2))
    assert np.array_equal(h.numpy(), x / 2 + x / 2) and (np.abs(y2.numpy() - want) <= np.abs(want) * (rel + 3 * ref.u(dtype)) + low).all()
    # backward from what the forward pass saved; gradients of the size that such rows get, so that dx is of size 1
    r = r.numpy()
    dy = (rng.standard_normal(x.shape) * np.minimum(scales, 1e3)).astype(dtype)
    dx, _ = ctx.rmsnorm_bwd(ctx.upload(dy), ctx.upload(x), ctx.upload(w), ctx.upload(r))
    g, rr = dy.astype(np.longdouble) * w, r.astype(np.longdouble)[:, None]
    q, size = (g * wide).mean(1, keepdims=True) * rr * rr, np.abs(g * wide).mean(1, keepdims=True) * rr * rr
    # as ref.rmsnorm_bwd counts them, and each product's own subnormal step carried to dx
    bound = ref.u(dtype) * rr * (4 * np.abs(g) + np.abs(wide) * size * (ref.sum_depth(dim) + 8)) + low * (4 + 4 * rr + 4 * np.abs(wide) * rr * rr * (1 + rr))
    assert (np.abs(dx.numpy() - rr * (g - wide * q)) <= 1.01 * bound).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("dim", [7, 700, 5000, 17000])
def test_rows_without_a_norm(ctx, dim, dtype):
    """An infinite element: rstd 0, NaN there and zeros elsewhere; a NaN: NaN throughout; zeros: zeros, or NaN without eps."""
    x = np.ones((4, dim), dtype)
    x[0, 3], x[1, 2], x[2] = np.inf, np.nan, 0
    w = np.full(dim, 2, dtype)
    for eps in (0.0, 1e-6):
        _, y, r = ctx.rmsnorm_fwd(ctx.upload(x), ctx.upload(w), eps)
        y, r = y.numpy(), r.numpy()
        assert r[0] == 0 and np.isnan(y[0, 3]) and (np.delete(y[0], 3) == 0).all()
        assert np.isnan(r[1]) and np.isnan(y[1]).all()
        assert (np.isnan(y[2]).all() and r[2] == np.inf) if eps == 0 else (y[2] == 0).all()
        assert np.isfinite(y[3]).all()
