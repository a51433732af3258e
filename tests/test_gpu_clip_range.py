"""The gradient norm and clipping over the whole range of both types: squares that pass f64's range at either end, norms that pass the
tensors' type, factors below its smallest normal number.  The plain form is in long double (15 bits of exponent)."""
import numpy as np
import pytest

import lm_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]


@pytest.fixture(scope="module")
def ctx():
    from ferrox_amd import capi
    with capi.Context(0) as c:
        yield c


def plain(gs, max_norm):
    wide = [g.astype(np.longdouble) for g in gs]
    norm = np.sqrt(sum((g * g).sum() for g in wide))
    factor = np.longdouble(max_norm) / norm if norm > max_norm else np.longdouble(1)
    return [g * factor for g in wide], norm


def mixed(n, dtype, *values):
    """The values in turn with changing signs, the rest zeros."""
    g = np.zeros(n, dtype)
    g[::7] = np.resize(np.array(values, dtype), g[::7].size)
    g[::14] *= -1
    return g


top, low = {t: np.finfo(t).max for t in DTYPES}, {t: np.finfo(t).smallest_subnormal for t in DTYPES}
CASES = [  # type, values, max_norm
    (np.float64, (1e200,), 1.0), (np.float64, (1e160, 3.0, 1e-200), 10.0), (np.float64, (1e-200, 2e-190), 1e-201), (np.float64, (1e-200, 0.0), 1.0),
    (np.float64, (top[np.float64],), 1.0), (np.float64, (top[np.float64], 1.0), 1e300), (np.float64, (low[np.float64], 3e-322), 1e-323),
    (np.float64, (1e150, 1e-170), 1e-300), (np.float64, (1e-154, 1e-155), 1e-156), (np.float64, (3e153, 1e154, 1e146), 2.0),
    (np.float64, (1e300,), 1e-300), (np.float64, (1e308,), np.inf), (np.float64, (1e-300, 1e-160), 0.0),
    (np.float32, (top[np.float32],), 1.0), (np.float32, (1e30,), 1e-12), (np.float32, (low[np.float32], 1e-40), 1e-42), (np.float32, (1e25, 1e-25), 1e-20),
    (np.float32, (top[np.float32],), 1e30), (np.float32, (1.0,), 1e-39)]


@pytest.mark.parametrize("n", [3, 5000, 300001])
@pytest.mark.parametrize("dtype,values,max_norm", CASES)
def test_clipping_over_the_range(ctx, dtype, values, max_norm, n):
    gs = [mixed(n, dtype, *values), mixed(n // 2 + 1, dtype, *reversed(values)), np.zeros(9000, dtype)]
    want, norm = plain(gs, max_norm)
    count = sum(g.size for g in gs)
    rel = ref.norm_rel(count, dtype) + 4 * ref.u(np.float64)  # the partial sums' rescaling rounds a few times more
    tiny = float(low[dtype])

    def holds(got):
        if norm > np.longdouble(top[dtype]) * (1 + rel):
            assert got == np.inf
        else:  # a subnormal norm is rounded to a step of its own
            assert abs(np.longdouble(got) - norm) <= rel * norm + tiny
    dev = [ctx.upload(g) for g in gs]
    holds(ctx.grad_norm(dev).numpy()[0])
    outs = [ctx.empty(g.shape, dtype) for g in gs]
    holds(ctx.clip_grad_norm(dev, max_norm, outs=outs).numpy()[0])
    for o, w, g in zip(outs, want, gs):
        o = o.numpy()
        if not norm > max_norm:
            assert np.array_equal(o, g)
        else:  # the norm, the quotient, its rounding to the type, the product; a subnormal result is rounded to its step
            assert (np.abs(o.astype(np.longdouble) - w) <= np.abs(w) * (rel + 4 * ref.u(dtype)) + tiny).all()
    ctx.clip_grad_norm(dev, max_norm)
    assert all(np.array_equal(d.numpy(), o.numpy()) for d, o in zip(dev, outs))


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_infinite_gradients_among_large_and_small_ones(ctx, bad):
    g = mixed(20000, np.float64, 1e200, 1e-200, 1.0)
    g[12345] = bad
    dev = ctx.upload(g)
    got = ctx.clip_grad_norm([dev], 1.0).numpy()[0]
    assert np.isnan(got) if np.isnan(bad) else got == np.inf
    assert np.array_equal(dev.numpy(), g, equal_nan=True)
