"""What the pieces of a long recurrence hand on to one another: infinite states against the definition step by step, states carried over
dozens of pieces."""
import numpy as np
import pytest

import lm_reference as ref
import recurrence_chains as rc

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]


@pytest.fixture(scope="module")
def ctx():
    from ferrox_amd import capi
    with capi.Context(0) as c:
        yield c


def as_defined(got, want, bound, what):
    """Equal where the definition gives an infinity or NaN, within the bound elsewhere."""
    got = np.asarray(got, np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    end = np.isinf(want)
    assert np.array_equal(got[end], want[end]) and np.array_equal(np.isinf(got), end), what
    fine = np.isfinite(want)
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all(), what


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", [(2, 7, 20), (2, 30, 20), (2, 100, 33), (1, 700, 70), (1, 5000, 20)])
def test_infinite_states(ctx, B, T, D, dtype):
    """Small gates: the product of a piece's gates underflows, none of them is 0 except where z is -inf."""
    rng = np.random.default_rng(T + D)
    z = rng.uniform(*((-6, 2) if dtype == np.float32 else (-20, -4)), (B, T, D)).astype(dtype)
    x, dh = rng.standard_normal((B, T, D)).astype(dtype), rng.standard_normal((B, T, D)).astype(dtype)
    h0, nxt = rng.standard_normal((B, D)).astype(dtype), rng.standard_normal((B, D)).astype(dtype)
    h = rng.standard_normal((B, T, D)).astype(dtype)
    h0[:, 0], h0[:, 1], nxt[:, 0], nxt[:, 1] = np.inf, -np.inf, np.inf, -np.inf
    x[:, T // 3, 2], x[:, T // 2, 3], x[:, 0, 4] = np.inf, -np.inf, np.inf
    dh[:, T // 3, 2], dh[:, T // 2, 3], dh[:, T - 1, 4] = np.inf, -np.inf, np.inf
    x[:, T // 3, 5], x[:, T // 2, 5] = np.inf, -np.inf      # NaN from the second on
    dh[:, T // 3, 5], dh[:, T // 2, 5] = -np.inf, np.inf
    h0[:, 6], nxt[:, 6], z[:, T // 2, 6] = np.inf, np.inf, -np.inf  # a gate of 0: NaN from there on
    z[:, T // 2, 7] = -np.inf                               # a finite state starts anew
    h0[:, 8], nxt[:, 8] = np.finfo(dtype).max, np.finfo(dtype).max / 4  # large but finite: dies away
    h0[:, 9], z[:, T // 4, 9] = np.inf, np.nan
    tame = np.where(np.isfinite(x), x, 0).astype(dtype)
    with np.errstate(all="ignore"):
        want, bound = ref.recurrence_fwd(z, x, h0)
        back, bounds = ref.recurrence_bwd(dh, z, tame, h, None, nxt)
    got = ctx.gated_recurrence_fwd(ctx.upload(z), ctx.upload(x), ctx.upload(h0)).numpy()
    as_defined(got, want, bound, "h")
    outs = ctx.gated_recurrence_bwd(ctx.upload(dh), ctx.upload(z), ctx.upload(tame), ctx.upload(h), None, ctx.upload(nxt), want_dh0=True)
    for o, w, b, name in zip(outs, back, bounds, ("dz", "dx", "dh0")):
        as_defined(o.numpy(), w, b, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", rc.SHAPES)
def test_states_carried_over_many_pieces(ctx, B, T, D, dtype):
    z, x, h0, dh, nxt = rc.inputs(B, T, D, dtype)
    up = {name: ctx.upload(a) for name, a in (("z", z), ("x", x), ("h0", h0), ("dh", dh), ("nxt", nxt))}
    h = ctx.gated_recurrence_fwd(up["z"], up["x"], up["h0"])
    rc.check_forward(h.numpy().astype(np.float64), z, x, h0)
    dz, dx, dh0 = ctx.gated_recurrence_bwd(up["dh"], up["z"], up["x"], h, up["h0"], up["nxt"])
    rc.check_backward(*(a.numpy().astype(np.float64) for a in (dz, dx, dh0)), dh, z, x, h.numpy(), h0, nxt)
