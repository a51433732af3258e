"""The plain forms that the language-model operators are tested against, themselves checked on the CPU: gradients against central
differences of the forward forms, and the refusals that need no device."""
import ctypes as C

import numpy as np
import pytest

import lm_reference as ref


def directional(f, args, at, rng, step=1e-6):
    d = rng.standard_normal(args[at].shape)
    up, down = list(args), list(args)
    up[at], down[at] = args[at] + step * d, args[at] - step * d
    return (f(*up) - f(*down)) / (2 * step), d


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
def test_linear_gradients(name):
    rng = np.random.default_rng(0)
    x, w, b, g = rng.standard_normal((5, 7)), rng.standard_normal((6, 7)), rng.standard_normal(6), rng.standard_normal((5, 6))

    def f(x, w, b):
        return float((ref.linear_fwd(x, w.T, b, name, None)[0] * g).sum())
    pre = ref.linear_fwd(x, w.T, b, name, None)[1]
    (dx, dw, db, _), _ = ref.linear_bwd(g, w, x, pre, name)
    for at, got in ((0, dx), (1, dw), (2, db)):
        want, d = directional(f, [x, w, b], at, rng)
        assert abs(want - (got * d).sum()) < 1e-6 * max(1, abs(want))


@pytest.mark.parametrize("with_res", [False, True])
def test_rmsnorm_gradients(with_res):
    rng = np.random.default_rng(1)
    x, w, g, gh = rng.standard_normal((4, 9)), rng.standard_normal(9), rng.standard_normal((4, 9)), rng.standard_normal((4, 9))
    r = rng.standard_normal((4, 9)) if with_res else None

    def f(x, w):
        h, y, _ = ref.rmsnorm_fwd(x, w, 1e-5, r)
        return float((y * g).sum() + (h * gh).sum())
    h, _, rstd = ref.rmsnorm_fwd(x, w, 1e-5, r)
    dx, dw, _, _ = ref.rmsnorm_bwd(g, h, w, rstd, gh)
    for at, got in ((0, dx), (1, dw)):
        want, d = directional(f, [x, w], at, rng)
        assert abs(want - (got * d).sum()) < 1e-6 * max(1, abs(want))


def test_recurrence_gradients():
    rng = np.random.default_rng(2)
    z, x, h0 = rng.standard_normal((2, 11, 3)), rng.standard_normal((2, 11, 3)), rng.standard_normal((2, 3))
    g, gn = rng.standard_normal((2, 11, 3)), rng.standard_normal((2, 3))

    def f(z, x, h0):
        h = ref.recurrence_fwd(z, x, h0)[0]
        return float((h * g).sum() + (h[:, -1] * gn).sum())
    h = ref.recurrence_fwd(z, x, h0)[0]
    (dz, dx, dh0), _ = ref.recurrence_bwd(g, z, x, h, h0, gn)
    for at, got in ((0, dz), (1, dx), (2, dh0)):
        want, d = directional(f, [z, x, h0], at, rng)
        assert abs(want - (got * d).sum()) < 1e-6 * max(1, abs(want))


def test_embedding_gradient():
    rng = np.random.default_rng(3)
    w, ids, g = rng.standard_normal((5, 4)), np.array([3, 0, 3, -1, 7, 3, 5, 4]), rng.standard_normal((8, 4))
    dw, _ = ref.embedding_bwd(g, ids, 5, 1.5)
    want, d = directional(lambda w: float((ref.embedding_fwd(w, ids, 1.5) * g).sum()), [w], 0, rng)
    assert abs(want - (dw * d).sum()) < 1e-6


def test_entry_points_refuse_a_null_context():
    from ferrox_amd import capi
    lib = capi.lib
    n = C.c_int64(1)
    for s in ("f32", "f64"):
        calls = [("embedding_fwd", (None,) * 4 + (1, 1, 1, 1.0)), ("embedding_bwd", (None,) * 4 + (1, 1, 1, 1.0)),
                 ("rmsnorm_fwd", (None,) * 4 + (1e-6,) + (None,) * 3 + (1, 1)), ("rmsnorm_bwd", (None,) * 8 + (1, 1)),
                 ("gemm_bias_act_residual", (None, 0, 0, 1, 1, 1) + (None,) * 6 + (0,)),
                 ("linear_act_bwd", (None, 1, 1, 1) + (None,) * 4 + (0,) + (None,) * 4),
                 ("gated_recurrence_fwd", (None,) * 5 + (1, 1, 1)), ("gated_recurrence_bwd", (None,) * 10 + (1, 1, 1)),
                 ("grad_norm_multi", (None, 0, None, C.byref(n), None)), ("clip_grad_norm_multi", (None, 0, None, None, C.byref(n), 1.0, None))]
        for name, args in calls:
            assert getattr(lib, f"fx_{name}_{s}")(*args) == 1, name
            assert b"null context" in lib.fx_last_error(), name
