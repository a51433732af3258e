"""The operators of a language model's training step (embedding, RMS norm with residual, Linear with activation and residual, gated
recurrence, gradient clipping) against their plain float64 forms, with bounds that count roundings (lm_reference.py)."""
import ctypes as C

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


def within(got, want, bound, what):
    got = np.asarray(got, np.float64)
    assert got.shape == np.shape(want), what
    off = np.abs(got - want)
    assert np.isfinite(got).all() and (off <= bound).all(), (what, float(off.max()), float((off / np.maximum(bound, 1e-300)).max()))


def shifted(ctx, a, by=1):
    """A copy of `a` on the device that starts `by` elements into a block: a pointer that is not 16-byte aligned."""
    from ferrox_amd import capi
    a = np.ascontiguousarray(a)
    base = ctx.upload(np.concatenate([np.zeros(by, a.dtype), a.ravel()]))
    v = capi.DeviceArray(ctx, a.shape, a.dtype, base.ptr + by * a.dtype.itemsize, 0, None)
    v._base = base
    return v


def _view(ctx, ptr, shape, dtype=np.float32):
    from ferrox_amd import capi
    return capi.DeviceArray(ctx, shape, dtype, ptr, 0, None)


def filled(ctx, shape, dtype, by=0):
    """An output full of NaN between guard elements, and a check that the guards are untouched."""
    n = int(np.prod(shape))
    host = np.full(n + 64, np.nan, dtype)
    host[:by], host[by + n:] = 7.0, 7.0
    from ferrox_amd import capi
    base = ctx.upload(host)
    v = capi.DeviceArray(ctx, shape, dtype, base.ptr + by * np.dtype(dtype).itemsize, 0, None)
    v._base = base

    def intact():
        h = base.numpy()
        return (h[:by] == 7.0).all() and (h[by + n:] == 7.0).all()
    return v, intact


# ---- embedding -------------------------------------------------------------------------------------------------------------------
def token_ids(rng, n, vocab, kind):
    if kind == "one":
        return np.full(n, vocab - 1, np.int64)
    if kind == "each":
        return rng.permutation(np.arange(n, dtype=np.int64) % vocab)
    if kind == "padding":
        return np.full(n, -1, np.int64)
    ids = np.minimum(np.floor(np.exp(rng.random(n) * np.log(vocab + 1.0))).astype(np.int64) - 1, vocab - 1)  # P(id) ~ 1 / (id + 1)
    if kind == "outside":
        ids[rng.random(n) < 0.3] = -1
        ids[rng.random(n) < 0.1] = vocab
        ids[rng.random(n) < 0.05] = np.iinfo(np.int64).max
        ids[rng.random(n) < 0.05] = np.iinfo(np.int64).min
    return ids


EMBED = [(1, 1, 1, "zipf"), (1, 300, 8, "zipf"), (5, 7, 3, "outside"), (16, 2, 64, "one"), (17, 1, 12, "one"), (31, 5, 1024, "zipf"),
         (33, 1000, 260, "each"), (64, 255, 16, "each"), (65, 256, 16, "each"), (700, 257, 36, "outside"), (1024, 65536, 4, "zipf"),
         (1025, 70, 1001, "zipf"), (2048, 3, 128, "zipf"), (4097, 40, 20, "padding"), (4096, 500, 40, "one"), (5000, 65535, 7, "outside"),
         (16384, 5000, 24, "zipf"), (16385, 5000, 24, "zipf"), (20000, 300, 33, "outside"), (40001, 70000, 8, "zipf"), (70000, 1, 5, "one"),
         (100, 50, 5000, "zipf"), (300, 2200000, 2, "zipf"), (2000, 600000, 3, "outside"), (32768, 300, 4, "zipf"), (32768, 200, 3, "one"), (66000, 17000000, 1, "zipf")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,dim,kind", EMBED)
def test_embedding(ctx, n, vocab, dim, kind, dtype):
    rng = np.random.default_rng(n + vocab)
    ids = token_ids(rng, n, vocab, kind)
    w = rng.standard_normal((vocab, dim)).astype(dtype)
    scale = float(np.sqrt(dim))
    di = ctx.upload_ids(ids)
    out, intact = filled(ctx, (n, dim), dtype)
    ctx.embedding_fwd(ctx.upload(w), di, scale, out=out)
    assert np.array_equal(out.numpy(), ref.embedding_fwd(w, ids, scale)) and intact()
    g = rng.standard_normal((n, dim)).astype(dtype)
    g[(ids < 0) | (ids >= vocab)] = np.nan  # what belongs to padding is not looked at
    want, bound = ref.embedding_bwd(g, ids, vocab, scale)
    dw, intact = filled(ctx, (vocab, dim), dtype)
    dg = ctx.upload(g)
    ctx.embedding_bwd(dg, di, vocab, scale, out=dw)
    first = dw.numpy()
    within(first, want, bound, "dW")
    assert intact()
    ctx.embedding_bwd(dg, di, vocab, scale, out=dw)
    assert np.array_equal(first, dw.numpy())  # one order of summation


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_unaligned_and_empty(ctx, dtype):
    rng = np.random.default_rng(4)
    w, ids = rng.standard_normal((50, 32)).astype(dtype), rng.integers(-1, 50, (6, 35))
    out, intact = filled(ctx, (6, 35, 32), dtype, by=1)
    ctx.embedding_fwd(shifted(ctx, w), ctx.upload_ids(ids), 0.5, out=out)
    assert np.array_equal(out.numpy(), ref.embedding_fwd(w, ids, 0.5)) and intact()
    g = rng.standard_normal((6, 35, 32)).astype(dtype)
    dw, intact = filled(ctx, (50, 32), dtype, by=3)
    ctx.embedding_bwd(shifted(ctx, g), ctx.upload_ids(ids), 50, 0.5, out=dw)
    want, bound = ref.embedding_bwd(g, ids, 50, 0.5)
    within(dw.numpy(), want, bound, "dW")
    assert intact()
    # no tokens at all: nothing is looked up, the gradient is zero
    from ferrox_amd.capi import check, lib
    s = "f32" if dtype == np.float32 else "f64"
    check(getattr(lib, f"fx_embedding_fwd_{s}")(ctx.h, None, None, None, 0, 50, 32, 1.0))
    check(getattr(lib, f"fx_embedding_bwd_{s}")(ctx.h, None, None, dw.ptr, 0, 50, 32, 1.0))
    assert (dw.numpy() == 0).all() and intact()


def test_embedding_rows_beyond_32_bit_offsets(ctx):
    """A table of 4.4 GB: rows past byte 2^32 and element 2^30."""
    vocab, dim = 1100000, 1000
    w = ctx.uniform((vocab, dim), 7, -1.0, 1.0)
    ids = np.array([0, vocab - 1, 1073742, 1099999, 536871, -1], np.int64)
    got = ctx.embedding_fwd(w, ctx.upload_ids(ids), 2.0).numpy()
    for k, i in enumerate(ids.tolist()):
        assert np.array_equal(got[k], w.rows(i, i + 1).numpy()[0] * np.float32(2.0) if i >= 0 else np.zeros(dim, np.float32)), i
    g = np.arange(6 * dim, dtype=np.float32).reshape(6, dim)
    ctx.embedding_bwd(ctx.upload(g), ctx.upload_ids(ids), vocab, 1.0, out=w)
    assert np.array_equal(w.rows(vocab - 1, vocab).numpy()[0], g[1] + g[3])
    for k in (0, 2, 4):
        assert np.array_equal(w.rows(int(ids[k]), int(ids[k]) + 1).numpy()[0], g[k])
    for v in (1, 1073741, 1073743, vocab - 2):
        assert (w.rows(v, v + 1).numpy() == 0).all()
    assert ctx.reduce("max", w.reshape(vocab * dim), 0).numpy().item() == (g[1] + g[3]).max()


# ---- RMS norm ------------------------------------------------------------------------------------------------------------------------
NORM = [(1, 1), (1, 8), (3, 5), (7, 255), (9, 256), (5, 257), (4, 512), (130, 516), (6, 1000), (5, 1001), (3, 1024), (1030, 1024), (3, 1025),
        (2, 2048), (5, 2052), (3, 4096), (3, 4097), (2, 8192), (3, 16384), (2, 16385), (3, 20000), (5000, 12), (2100, 2056)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("rows,dim", NORM)
def test_rmsnorm(ctx, rows, dim, with_res, dtype):
    rng = np.random.default_rng(rows * 7 + dim)
    x, w = rng.standard_normal((rows, dim)).astype(dtype), (1 + 0.1 * rng.standard_normal(dim)).astype(dtype)
    res = (2 * rng.standard_normal((rows, dim))).astype(dtype) if with_res else None
    x[rows // 2] = 0  # a row of zeros: rstd = 1 / sqrt(eps)
    if with_res:
        res[rows // 2] = 0
    eps = 1e-6
    (h, hi), (y, yi), (r, ri) = filled(ctx, (rows, dim), dtype), filled(ctx, (rows, dim), dtype), filled(ctx, (rows,), dtype)
    ctx.rmsnorm_fwd(ctx.upload(x), ctx.upload(w), eps, ctx.upload(res) if with_res else None, out=(h if with_res else None, y, r))
    want_h, want_y, want_r = ref.rmsnorm_fwd(x, w, eps, res)
    rel = ref.rmsnorm_rel(dim, dtype)
    if with_res:
        assert np.array_equal(h.numpy(), want_h)
    within(r.numpy(), want_r, want_r * rel, "rstd")
    within(y.numpy(), want_y, np.abs(want_y) * (rel + 3 * ref.u(dtype)), "y")
    assert hi() and yi() and ri()
    # backward, from the values the forward pass saved
    dy, dh = rng.standard_normal((rows, dim)).astype(dtype), rng.standard_normal((rows, dim)).astype(dtype) if with_res else None
    saved = r.numpy()
    (dx, xi), (dw, wi) = filled(ctx, (rows, dim), dtype), filled(ctx, (dim,), dtype)
    ins = [ctx.upload(dy), ctx.upload(want_h), ctx.upload(w), ctx.upload(saved)]
    ctx.rmsnorm_bwd(*ins, dh=ctx.upload(dh) if with_res else None, out=(dx, dw))
    ex, ew, bx, bw = ref.rmsnorm_bwd(dy, want_h, w, saved, dh)
    within(dx.numpy(), ex, bx, "dx")
    within(dw.numpy(), ew, bw, "dw")
    assert xi() and wi()
    kept = dx.numpy(), dw.numpy()
    again = ctx.rmsnorm_bwd(*ins, dh=ctx.upload(dh) if with_res else None, want_dw=False)
    assert again[1] is None and np.array_equal(kept[0], again[0].numpy())
    ctx.rmsnorm_bwd(*ins, dh=ctx.upload(dh) if with_res else None, out=(dx, dw))
    assert np.array_equal(kept[0], dx.numpy()) and np.array_equal(kept[1], dw.numpy())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(70, 256), (9, 1002), (3, 3000), (2, 16400)])
def test_rmsnorm_in_place_and_unaligned(ctx, rows, dim, dtype):
    rng = np.random.default_rng(dim)
    x, r, w = (rng.standard_normal(s).astype(dtype) for s in ((rows, dim), (rows, dim), (dim,)))
    plain = [a.numpy() for a in ctx.rmsnorm_fwd(ctx.upload(x), ctx.upload(w), 1e-5, ctx.upload(r))]
    dx, dr = ctx.upload(x), ctx.upload(r)
    ctx.rmsnorm_fwd(dx, ctx.upload(w), 1e-5, dr, out=(dr, dx, None))  # the residual stream in place, y over x, rstd not wanted
    assert np.array_equal(dr.numpy(), plain[0]) and np.array_equal(dx.numpy(), plain[1])
    dy, dh = rng.standard_normal((rows, dim)).astype(dtype), rng.standard_normal((rows, dim)).astype(dtype)
    h, y, s = ctx.rmsnorm_fwd(shifted(ctx, x), shifted(ctx, w), 1e-5, shifted(ctx, r, 3))
    assert np.array_equal(h.numpy(), plain[0])
    within(y.numpy(), *[(a, np.abs(a) * (ref.rmsnorm_rel(dim, dtype) + 3 * ref.u(dtype))) for a in [ref.rmsnorm_fwd(x, w, 1e-5, r)[1]]][0], "y")
    gx, gw = (a.numpy() for a in ctx.rmsnorm_bwd(ctx.upload(dy), h, ctx.upload(w), s, ctx.upload(dh)))
    for over in ("dy", "dh"):
        a, b = ctx.upload(dy), ctx.upload(dh)
        _, dw = ctx.rmsnorm_bwd(a, h, ctx.upload(w), s, b, out=((a if over == "dy" else b), ctx.empty((dim,), dtype)))
        assert np.array_equal((a if over == "dy" else b).numpy(), gx) and np.array_equal(dw.numpy(), gw)
    ux, uw = ctx.rmsnorm_bwd(shifted(ctx, dy), shifted(ctx, h.numpy(), 2), shifted(ctx, w), s, shifted(ctx, dh))
    ex, ew, bx, bw = ref.rmsnorm_bwd(dy, h.numpy(), w, s.numpy(), dh)
    within(ux.numpy(), ex, bx, "dx")
    within(uw.numpy(), ew, bw, "dw")


# ---- Linear with activation and residual -------------------------------------------------------------------------------------------------
LINEAR = [(1, 1, 1), (1, 32, 8), (5, 7, 3), (33, 31, 65), (64, 64, 64), (100, 64, 100), (256, 784, 256), (256, 256, 10), (10, 2048, 300), (128, 132, 128),
          (130, 192, 260), (16, 4096, 40), (300, 1000, 129), (512, 128, 1024), (1024, 512, 512), (2, 20000, 6), (256, 16384, 10), (32, 64, 9000),
          (1030, 260, 1028), (2100, 40, 2100), (1, 4097, 130), (2, 513, 31), (3, 1001, 257), (4, 512, 64), (4, 2600, 5)]
ACTS = ["none", "relu", "gelu", "silu"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_gemm_bias_act_residual(ctx, m, k, n, dtype):
    rng = np.random.default_rng(m * 3 + k + n)
    A, B = rng.standard_normal((m, k)).astype(dtype), (rng.standard_normal((k, n)) / np.sqrt(k)).astype(dtype)
    bias, res = rng.standard_normal(n).astype(dtype), (2 * rng.standard_normal((m, n))).astype(dtype)
    dbias, dres = ctx.upload(bias), ctx.upload(res)
    turn = 0
    for ta in (False, True):
        for tb in (False, True):
            a, b = ctx.upload(A.T if ta else A), ctx.upload(B.T if tb else B)
            # every transpose form with every activation over the four of them, bias / residual / pre in all combinations
            for act in ACTS:
                use = [(True, True, True), (False, True, False), (True, False, True), (False, False, False), (True, True, False),
                       (False, False, True), (True, False, False), (False, True, True)][turn % 8]
                turn += 3
                out, oi = filled(ctx, (m, n), dtype)
                pre, pi = filled(ctx, (m, n), dtype)
                ctx.gemm_bias_act_residual(a, b, ta, tb, bias=dbias if use[0] else None, act=act, residual=dres if use[1] else None,
                                           pre=pre if use[2] else None, out=out)
                y, p, by, bp = ref.linear_fwd(A, B, bias if use[0] else None, act, res if use[1] else None)
                within(out.numpy(), y, by, (ta, tb, act, use))
                if use[2]:
                    within(pre.numpy(), p, bp, (ta, tb, act, use, "pre"))
                assert oi() and pi()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gemm_epilogue_unaligned_empty_and_plain(ctx, dtype):
    rng = np.random.default_rng(5)
    A, B = rng.standard_normal((70, 132)).astype(dtype), rng.standard_normal((132, 96)).astype(dtype)
    bias, res = rng.standard_normal(96).astype(dtype), rng.standard_normal((70, 96)).astype(dtype)
    out, oi = filled(ctx, (70, 96), dtype, by=1)
    pre, pi = filled(ctx, (70, 96), dtype, by=3)
    ctx.gemm_bias_act_residual(shifted(ctx, A), shifted(ctx, B), bias=shifted(ctx, bias), act="gelu", residual=shifted(ctx, res), pre=pre, out=out)
    y, p, by, bp = ref.linear_fwd(A, B, bias, "gelu", res)
    within(out.numpy(), y, by, "C")
    within(pre.numpy(), p, bp, "pre")
    assert oi() and pi()
    # the bits of fx_gemm_bias_act where that call does the same
    from ferrox_amd.capi import check, lib
    s = "f32" if dtype == np.float32 else "f64"
    for act, name in ((0, "none"), (1, "relu")):
        for (m, k, n) in ((70, 132, 96), (256, 784, 256), (512, 256, 512), (256, 4096, 10)):
            a, b, v = (ctx.upload(rng.standard_normal(q).astype(dtype)) for q in ((m, k), (k, n), (n,)))
            there = ctx.empty((m, n), dtype)
            check(getattr(lib, f"fx_gemm_bias_act_{s}")(ctx.h, 0, 0, m, n, k, a.ptr, b.ptr, v.ptr, there.ptr, act))
            assert np.array_equal(ctx.gemm_bias_act_residual(a, b, bias=v, act=name).numpy(), there.numpy())
    # K = 0: the empty product, still with its epilogue
    check(getattr(lib, f"fx_gemm_bias_act_residual_{s}")(ctx.h, 0, 0, 70, 96, 0, None, None, ctx.upload(bias).ptr, None, None, out.ptr, 1))
    assert np.array_equal(out.numpy(), np.broadcast_to(np.maximum(bias, 0), (70, 96))) and oi()


@pytest.mark.parametrize("m,k,n", [(2052, 192, 2048), (2560, 128, 2564), (2049, 132, 2053), (1024, 256, 512), (1025, 260, 511)])
def test_gemm_epilogue_of_the_large_tiles(ctx, m, k, n):
    """f32 products of the 128- and 64-row tiles, with and without a remainder of K, rows of C at any alignment."""
    rng = np.random.default_rng(m)
    A, B = rng.standard_normal((m, k)).astype(np.float32), (rng.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32)
    bias, res = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n)).astype(np.float32)
    dbias, dres = shifted(ctx, bias), shifted(ctx, res, 3)
    for (ta, tb), act, use in zip(((False, True), (False, False), (True, False), (True, True)), ("gelu", "silu", "relu", "none"),
                                  ((True, True), (False, True), (True, True), (True, False))):
        out, oi = filled(ctx, (m, n), np.float32)
        pre, pi = filled(ctx, (m, n), np.float32, by=1)
        ctx.gemm_bias_act_residual(ctx.upload(A.T if ta else A), ctx.upload(B.T if tb else B), ta, tb, bias=dbias if use[0] else None, act=act,
                                   residual=dres if use[1] else None, pre=pre, out=out)
        y, p, by, bp = ref.linear_fwd(A, B, bias if use[0] else None, act, res if use[1] else None)
        within(out.numpy(), y, by, (ta, tb, act))
        within(pre.numpy(), p, bp, (ta, tb, act, "pre"))
        assert oi() and pi()


@pytest.mark.parametrize("dtype", DTYPES)
def test_activations_at_their_ends(ctx, dtype):
    """Through a product with the identity: saturation, signed zeros, infinities, NaN."""
    v = np.array([0.0, -0.0, 1e-30, -1e-30, 5, -5, 13, -13, 20, -20, 90, -90, 800, -800, np.inf, -np.inf, np.nan, 3e38, -3e38], dtype)
    K = v.size
    eye = np.eye(K, dtype=dtype)
    for act in ACTS:
        # one value per product row would mix the others' infinities in: add it as the bias of a zero product
        got = ctx.gemm_bias_act_residual(ctx.upload(eye[:1] * 0), ctx.upload(eye), bias=ctx.upload(v), act=act).numpy()[0]
        with np.errstate(all="ignore"):
            want = ref.act(v.astype(np.float64), act)
        if act in ("gelu", "silu"):
            want[v == -np.inf] = 0.0
            want[v == np.inf] = np.inf
        if act == "relu":
            want[np.isnan(v)] = 0.0  # v > 0 ? v : 0, as every ReLU of the library
        assert np.array_equal(np.isnan(got), np.isnan(want)), act
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)].astype(dtype)), act
        within(got[fine], want[fine], 3 * ref.u(dtype) * np.abs(np.where(np.isfinite(v), v, 0)[fine].astype(np.float64)) + 24 * ref.u(dtype) * np.abs(want[fine]) + np.finfo(dtype).tiny, act)
        # derivatives
        vv, one = ctx.upload(v[:, None]), ctx.upload(np.ones((K, 1), dtype))
        d = ctx.linear_act_bwd(one, ctx.upload(np.ones((1, 1), dtype)), ctx.upload(np.zeros((K, 1), dtype)), vv, act)[3].numpy()[:, 0]
        with np.errstate(all="ignore"):
            slope = ref.act_grad(v.astype(np.float64), act)
        slope[v == np.inf], slope[v == -np.inf] = 1.0, 0.0 if act != "none" else 1.0
        big = np.abs(v) > 1e30
        slope[big & (v > 0)], slope[big & (v < 0)] = 1.0, 0.0 if act != "none" else 1.0
        if act in ("gelu", "silu"):
            assert np.isnan(d[np.isnan(v)]).all()
        ok = ~np.isnan(v)
        within(d[ok], slope[ok], 36 * ref.u(dtype), act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("b,i,o", [(1, 1, 1), (3, 5, 7), (64, 33, 40), (256, 784, 256), (300, 64, 1030), (1000, 129, 5), (512, 256, 512), (2050, 20, 12)])
def test_linear_act_bwd(ctx, b, i, o, act, dtype):
    rng = np.random.default_rng(b + i + o)
    dy, w, x = rng.standard_normal((b, o)).astype(dtype), (rng.standard_normal((o, i)) / np.sqrt(i)).astype(dtype), rng.standard_normal((b, i)).astype(dtype)
    pre = (2 * rng.standard_normal((b, o))).astype(dtype)
    shapes = [(b, i), (o, i), (o,), (b, o)]
    outs = [filled(ctx, s, dtype) for s in shapes]
    ddy, dw_, dx_, dpre = ctx.upload(dy), ctx.upload(w), ctx.upload(x), ctx.upload(pre)
    ctx.linear_act_bwd(ddy, dw_, dx_, dpre, act, out=[v for v, _ in outs])
    want, bounds = ref.linear_bwd(dy, w, x, pre, act)
    kept = [v.numpy() for v, _ in outs]
    for got, e, bd, name in zip(kept, want, bounds, ("dx", "dw", "db", "dpre")):
        within(got, e, bd, name)
    assert all(intact() for _, intact in outs)
    # without the bias gradient, and with dpre over dY and over pre: the same bits
    for over in (ddy, dpre):
        got = ctx.linear_act_bwd(ctx.upload(dy) if over is dpre else ddy, dw_, dx_, ctx.upload(pre) if over is ddy else dpre, act,
                                 out=(ctx.empty((b, i), dtype), ctx.empty((o, i), dtype), None, over))
        for q in (0, 1, 3):
            assert np.array_equal(got[q].numpy(), kept[q])


# ---- gated recurrence ---------------------------------------------------------------------------------------------------------------------
SCAN = [(1, 1, 1), (1, 1, 8), (64, 1, 96), (3, 2, 5), (2, 7, 64), (1, 8, 65), (2, 9, 33), (5, 31, 12), (1, 32, 130), (2, 33, 16), (1, 127, 3), (2, 128, 7),
        (1, 129, 64), (3, 300, 70), (1, 513, 64), (1, 1024, 20), (2, 1025, 5), (1, 2047, 65), (1, 5000, 3), (40, 140, 1), (300, 20, 70), (1, 3, 20000)]


def scan_inputs(rng, B, T, D, dtype):
    z = (2 + 2 * rng.standard_normal((B, T, D))).astype(dtype)
    x = rng.standard_normal((B, T, D)).astype(dtype)
    z.reshape(-1)[rng.random(z.size) < 0.02] = -np.inf  # the state starts anew
    z.reshape(-1)[rng.random(z.size) < 0.02] = np.inf   # the state is kept
    z.reshape(-1)[rng.random(z.size) < 0.01] = np.finfo(dtype).min
    return z, x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", SCAN)
def test_gated_recurrence(ctx, B, T, D, dtype):
    rng = np.random.default_rng(B * 11 + T + D)
    z, x = scan_inputs(rng, B, T, D, dtype)
    dz_, dx_ = ctx.upload(z), ctx.upload(x)
    for with_h0 in (False, True):
        h0 = rng.standard_normal((B, D)).astype(dtype) if with_h0 else None
        d0 = ctx.upload(h0) if with_h0 else None
        h, hi = filled(ctx, (B, T, D), dtype)
        ctx.gated_recurrence_fwd(dz_, dx_, d0, out=h)
        want, bound = ref.recurrence_fwd(z, x, h0)
        got = h.numpy()
        within(got, want, bound, ("h", with_h0))
        assert hi()
        dh, nxt = rng.standard_normal((B, T, D)).astype(dtype), rng.standard_normal((B, D)).astype(dtype) if with_h0 else None
        outs = [filled(ctx, (B, T, D), dtype), filled(ctx, (B, T, D), dtype), filled(ctx, (B, D), dtype)]
        ctx.gated_recurrence_bwd(ctx.upload(dh), dz_, dx_, h, d0, ctx.upload(nxt) if with_h0 else None, out=[v for v, _ in outs])
        want, bounds = ref.recurrence_bwd(dh, z, x, got, h0, nxt)
        for (v, intact), e, b, name in zip(outs, want, bounds, ("dz", "dx", "dh0")):
            within(v.numpy(), e, b, (name, with_h0))
            assert intact()
        two = ctx.gated_recurrence_bwd(ctx.upload(dh), dz_, dx_, h, d0, ctx.upload(nxt) if with_h0 else None, want_dh0=False)
        assert two[2] is None and np.array_equal(two[0].numpy(), outs[0][0].numpy()) and np.array_equal(two[1].numpy(), outs[1][0].numpy())


@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_segments_and_single_steps(ctx, dtype):
    """A sequence cut into segments, each from the last state of the one before, and token by token; and backwards the same."""
    rng = np.random.default_rng(12)
    B, T, D = 3, 200, 40
    z, x = scan_inputs(rng, B, T, D, dtype)
    want, bound = ref.recurrence_fwd(z, x, None)
    state, parts, cuts = None, [], [0, 1, 2, 70, 199, 200]
    for a, b in zip(cuts[:-1], cuts[1:]):
        h = ctx.gated_recurrence_fwd(ctx.upload(z[:, a:b]), ctx.upload(x[:, a:b]), state).numpy()
        parts.append(h)
        state = ctx.upload(h[:, -1])
    whole = np.concatenate(parts, 1)
    within(whole, want, bound, "segments")
    dh = rng.standard_normal((B, T, D)).astype(dtype)
    (ez, ex, _), (bz, bx, _) = ref.recurrence_bwd(dh, z, x, whole, None, None)
    nxt = None
    for a, b in reversed(list(zip(cuts[:-1], cuts[1:]))):
        h0 = ctx.upload(whole[:, a - 1]) if a else None
        dz, dx, nxt = ctx.gated_recurrence_bwd(ctx.upload(dh[:, a:b]), ctx.upload(z[:, a:b]), ctx.upload(x[:, a:b]), ctx.upload(whole[:, a:b]), h0, nxt,
                                               want_dh0=True)
        within(dz.numpy(), ez[:, a:b], bz[:, a:b], ("dz", a))
        within(dx.numpy(), ex[:, a:b], bx[:, a:b], ("dx", a))


@pytest.mark.parametrize("dtype", DTYPES)
def test_recurrence_unaligned(ctx, dtype):
    rng = np.random.default_rng(13)
    z, x = scan_inputs(rng, 2, 50, 36, dtype)
    h, hi = filled(ctx, (2, 50, 36), dtype, by=1)
    ctx.gated_recurrence_fwd(shifted(ctx, z), shifted(ctx, x, 3), out=h)
    within(h.numpy(), *ref.recurrence_fwd(z, x, None), "h")
    assert hi()


# ---- clipping -----------------------------------------------------------------------------------------------------------------------------
CLIP = [[1], [0], [0, 5, 0], [3, 4095, 4096, 4097, 1], [10] * 97, [1 << 20, 7], [33] * 200 + [100003], [9000000]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", CLIP, ids=lambda s: f"{len(s)}x{s[0]}")
def test_clip_grad_norm(ctx, sizes, dtype):
    from ferrox_amd import capi
    rng = np.random.default_rng(len(sizes))
    gs = [rng.standard_normal(n).astype(dtype) for n in sizes]
    empty = capi.DeviceArray(ctx, (0,), dtype, None, 0, None)
    # every second tensor starts off a 16-byte border
    dev = [empty if g.size == 0 else shifted(ctx, g) if k % 2 else ctx.upload(g) for k, g in enumerate(gs)]
    _, norm = ref.clip(gs, 1.0)
    rel = ref.norm_rel(sum(sizes), dtype)
    assert abs(ctx.grad_norm(dev).numpy()[0] - norm) <= rel * norm
    for max_norm in (0.5 * norm, 2.0 * norm + 1e-3, 0.0):
        want, _ = ref.clip(gs, max_norm)
        scaled = norm > max_norm
        outs = [(empty, lambda: True) if g.size == 0 else filled(ctx, g.shape, dtype, by=k % 3) for k, g in enumerate(gs)]
        got = ctx.clip_grad_norm(dev, max_norm, outs=[o for o, _ in outs])
        assert abs(got.numpy()[0] - norm) <= rel * norm
        for k, (o, intact) in enumerate(outs):
            # the factor: the norm before its rounding, one quotient, one rounding to the type; then the product
            within(o.numpy(), want[k], np.abs(want[k]) * (rel + 3 * ref.u(dtype)) if scaled else 0.0, (k, max_norm))
            assert intact()
        same = [empty if g.size == 0 else ctx.upload(g) for g in gs]
        ctx.clip_grad_norm(same, max_norm)
        for k, g in enumerate(same):
            assert np.array_equal(g.numpy(), outs[k][0].numpy()), "in place"


@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_extremes(ctx, dtype):
    # no tensors at all
    from ferrox_amd.capi import check, lib
    s = "f32" if dtype == np.float32 else "f64"
    norm = ctx.fill((1,), 3.0, dtype)
    check(getattr(lib, f"fx_grad_norm_multi_{s}")(ctx.h, 0, None, None, norm.ptr))
    assert norm.numpy()[0] == 0
    check(getattr(lib, f"fx_clip_grad_norm_multi_{s}")(ctx.h, 0, None, None, None, 1.0, norm.ptr))
    assert norm.numpy()[0] == 0
    # squares that pass f32's range, and ones that vanish in it
    if dtype == np.float32:
        for v in (1e30, 1e-30):
            g = ctx.fill((1000,), v, dtype)
            want = np.float64(np.float32(v)) * np.sqrt(1000.0)
            got = ctx.clip_grad_norm([g], 0.5 * float(want)).numpy()[0]
            assert abs(got - want) <= ref.norm_rel(1000, dtype) * want
            assert np.allclose(g.numpy(), np.float32(v) * np.float32(0.5), rtol=4 * ref.u(dtype) * 2, atol=0)
    # a norm that is no number scales nothing and says so
    for bad in (np.nan, np.inf, -np.inf):
        host = np.ones(5000, dtype)
        host[4321] = bad
        a, b = ctx.upload(host), ctx.upload(np.full(10, 2.0, dtype))
        got = ctx.clip_grad_norm([a, b], 1.0).numpy()[0]
        assert np.isnan(got) if np.isnan(bad) else got == np.inf
        assert np.array_equal(a.numpy(), host, equal_nan=True) and (b.numpy() == 2.0).all()


# ---- sizes past 2^32 threads of one launch, rows of nearly 2^31 ----------------------------------------------------------------------------------
def test_rmsnorm_of_many_short_rows(ctx):
    rows = (1 << 26) + 5
    x, w = ctx.uniform((rows, 1), 3, -2.0, 2.0), ctx.fill((1,), 0.5)
    h, y, rstd = ctx.rmsnorm_fwd(x, w, 1e-6, res=x)
    x, h, y, rstd = (a.numpy().ravel() for a in (x, h, y, rstd))
    assert np.array_equal(h, x + x)
    h = h.astype(np.float64)
    r = 1.0 / np.sqrt(h * h + 1e-6)
    # the square, the addition and eps each at most u (the root halves them), root, reciprocal: 3.5 u, with room for the division by the row's
    # length; then two products
    assert (np.abs(rstd - r) <= 6 * ref.u(np.float32) * r).all()
    assert (np.abs(y - h * r * 0.5) <= 8 * ref.u(np.float32) * np.abs(h * r * 0.5)).all()


def test_one_row_times_many_columns(ctx):
    n = (1 << 26) + 5
    a, b, bias = ctx.fill((1, 2), 3.0), ctx.uniform((n, 2), 4, -1.0, 1.0), ctx.uniform((n,), 5, -1.0, 1.0)
    got = ctx.gemm_bias_act_residual(a, b, tb=True, bias=bias, act="relu", residual=bias.reshape(1, n)).numpy()[0].astype(np.float64)
    b, bias = b.numpy().astype(np.float64), bias.numpy().astype(np.float64)
    pre = 3.0 * b[:, 0] + 3.0 * b[:, 1] + bias
    size = 3.0 * np.abs(b).sum(1) + np.abs(bias)
    # two products, two additions (the largest chain: four roundings of a term), then the residual's addition
    assert (np.abs(got - (np.maximum(pre, 0) + bias)) <= 6 * ref.u(np.float32) * (size + np.abs(bias))).all()


def test_embedding_of_indices_found_on_the_device(ctx):
    """The arg-max of a product's rows as the next token ids, without a copy to the host; ids of another type are refused."""
    from ferrox_amd.capi import FerroxHipError
    rng = np.random.default_rng(5)
    logits, w = rng.standard_normal((6, 50)).astype(np.float32), rng.standard_normal((50, 8)).astype(np.float32)
    best = ctx.upload_ids(np.full(6, -1))
    ctx.reduce_max_noalloc(ctx.upload(logits), 1, ctx.empty((6,)), best)
    assert np.array_equal(ctx.embedding_fwd(ctx.upload(w), best).numpy(), w[logits.argmax(1)])
    for call in (lambda: ctx.embedding_fwd(ctx.upload(w), ctx.fill((6,), 1.0)), lambda: ctx.embedding_bwd(ctx.upload(w[:6]), ctx.fill((6,), 1.0), 50)):
        with pytest.raises(FerroxHipError, match="int64"):
            call()


# ---- refusals: the host's checks, before any launch ------------------------------------------------------------------------------------------
def test_refusals(ctx):
    from ferrox_amd.capi import FerroxHipError, lib
    f = np.float32
    a, b, v, row = ctx.fill((8, 8), 1.0), ctx.fill((8, 8), 2.0), ctx.fill((8,), 1.0), ctx.fill((8,), 1.0)
    ids = ctx.upload_ids(np.zeros(8, np.int64))
    big = ctx.fill((16, 8), 3.0)
    lo, hi = big.rows(0, 8), big.rows(4, 12)  # overlapping halves

    def refused(match, call, *args, **kw):
        with pytest.raises(FerroxHipError, match=match):
            call(*args, **kw)
    refused("overlaps", ctx.embedding_fwd, lo, ids, out=hi)
    refused("overlaps", ctx.embedding_bwd, lo, ids, 8, out=hi)
    refused("not", ctx.embedding_fwd, a, ids, out=ctx.empty((8, 9)))
    refused("not", ctx.embedding_bwd, v, ids, 8)
    assert lib.fx_embedding_fwd_f32(ctx.h, a.ptr, ids.ptr, None, 8, 8, 8, 1.0) == 1
    assert lib.fx_embedding_fwd_f32(ctx.h, a.ptr, ids.ptr, b.ptr, -1, 8, 8, 1.0) == 1
    assert lib.fx_embedding_fwd_f32(ctx.h, a.ptr, ids.ptr, b.ptr, 8, 0, 8, 1.0) == 1
    assert lib.fx_embedding_bwd_f32(ctx.h, a.ptr, ids.ptr, b.ptr, 8, 1 << 31, 8, 1.0) == 1
    refused("negative", ctx.rmsnorm_fwd, a, v, -1.0)
    refused("residual", ctx.rmsnorm_fwd, a, v, 1e-6, out=(b, ctx.empty((8, 8)), None))
    refused("overlap", ctx.rmsnorm_fwd, a, v, 1e-6, b, out=(a, a, None))
    refused("overlap", ctx.rmsnorm_fwd, lo, v, 1e-6, out=(None, hi, None))
    refused("not", ctx.rmsnorm_fwd, a, ctx.fill((7,), 1.0), 1e-6)
    refused("not", ctx.rmsnorm_fwd, a, ctx.fill((8,), 1.0, np.float64), 1e-6)
    refused("overlaps", ctx.rmsnorm_bwd, a, b, v, row, out=(b, None))
    refused("overlaps", ctx.rmsnorm_bwd, a, b, v, row, out=(ctx.empty((8, 8)), v))
    refused("shape mismatch", ctx.gemm_bias_act_residual, a, ctx.fill((7, 8), 1.0))
    refused("overlaps", ctx.gemm_bias_act_residual, a, b, residual=lo, out=hi)
    refused("overlaps", ctx.gemm_bias_act_residual, a, b, residual=lo, out=lo)
    refused("overlaps", ctx.gemm_bias_act_residual, a, b, pre=lo, out=hi)
    assert lib.fx_gemm_bias_act_residual_f32(ctx.h, 0, 0, 8, 8, 8, a.ptr, b.ptr, None, None, None, lo.ptr, 4) == 1
    assert lib.fx_gemm_bias_act_residual_f32(ctx.h, 0, 0, 8, 8, 8, a.ptr, None, None, None, None, lo.ptr, 0) == 1
    e = lambda *s: ctx.empty(s)  # noqa: E731
    refused("overlap", ctx.linear_act_bwd, a, b, e(8, 8), lo, "gelu", out=(e(8, 8), e(8, 8), None, hi))
    refused("overlap", ctx.linear_act_bwd, a, b, e(8, 8), lo, "gelu", out=(lo, e(8, 8), None, e(8, 8)))
    assert lib.fx_linear_act_bwd_f32(ctx.h, 0, 8, 8, a.ptr, b.ptr, a.ptr, a.ptr, 0, lo.ptr, lo.ptr, lo.ptr, None) == 1
    z = ctx.fill((2, 4, 8), 1.0)
    refused("not", ctx.gated_recurrence_fwd, z, ctx.fill((2, 8, 4), 1.0))
    refused("overlaps", ctx.gated_recurrence_fwd, z, ctx.fill((2, 4, 8), 1.0), out=z)
    refused("overlap", ctx.gated_recurrence_bwd, z, ctx.fill((2, 4, 8), 1.0), ctx.fill((2, 4, 8), 1.0), ctx.fill((2, 4, 8), 1.0),
            out=(big.reshape(4, 4, 8).rows(0, 2), big.reshape(4, 4, 8).rows(1, 3), None))
    assert lib.fx_gated_recurrence_bwd_f32(ctx.h, *([z.ptr] * 4), None, None, lo.ptr, hi.ptr, None, 2, 0, 8) == 1
    refused("overlaps", ctx.clip_grad_norm, [lo, hi], 1.0)
    refused("overlaps", ctx.clip_grad_norm, [a, b], 1.0, outs=[e(8, 8), a])
    refused("overlaps", ctx.clip_grad_norm, [a, a], 1.0)
    refused("overlaps", ctx.grad_norm, [a], norm=a.reshape(64).rows(5, 6))
    refused("overlaps", ctx.clip_grad_norm, [a], 1.0, norm=a.reshape(64).rows(63, 64))
    refused("overlaps", ctx.embedding_fwd, a, ids, out=_view(ctx, ids.ptr, (8, 8)))
    refused("negative", ctx.clip_grad_norm, [a], -1.0)
    refused("negative", ctx.clip_grad_norm, [a], float("nan"))
    refused("in a call of", ctx.clip_grad_norm, [a, ctx.fill((8,), 1.0, np.float64)], 1.0)
    n = (C.c_int64 * 1)(-1)
    t = (C.c_void_p * 1)(a.ptr)
    assert lib.fx_grad_norm_multi_f32(ctx.h, 1, t, n, v.ptr) == 1 and lib.fx_grad_norm_multi_f32(ctx.h, -1, t, n, v.ptr) == 1
    assert (a.numpy() == 1).all() and (b.numpy() == 2).all() and (v.numpy() == 1).all()


# ---- recorded into graphs ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
def test_recorded_calls_replay_bit_exact(ctx, dtype):
    """Every operator in one graph, replayed over new inputs with eager calls of other sizes in between, against eager calls."""
    from ferrox_amd.capi import check, lib
    rng = np.random.default_rng(20)
    n, vocab, d, B, T = 600, 90, 48, 4, 150

    def make():
        return [rng.standard_normal(s).astype(dtype) for s in ((vocab, d), (n, d), (n, d), (d,), (4 * d, d), (4 * d,), (n, 4 * d))]
    host = make()
    ids_host = rng.integers(-1, vocab, n)
    dev, ids = [ctx.upload(a) for a in host], ctx.upload_ids(ids_host)

    def outputs():
        shapes = [(n, d), (vocab, d), (n, d), (n, d), (n,), (n, d), (d,), (n, 4 * d), (n, 4 * d), (n, d), (4 * d, d), (4 * d,), (n, 4 * d), (B, T, d), (B, T, d),
                  (B, T, d), (1,)]
        return [ctx.empty(s, dtype) for s in shapes]

    def step(o):
        W, x, g, w, U, b, g4 = dev
        ctx.embedding_fwd(W, ids, 3.0, out=o[0])
        ctx.embedding_bwd(g, ids, vocab, 3.0, out=o[1])
        ctx.rmsnorm_fwd(x, w, 1e-6, o[0], out=(o[2], o[3], o[4]))
        ctx.rmsnorm_bwd(g, o[2], w, o[4], x, out=(o[5], o[6]))
        ctx.gemm_bias_act_residual(o[3], U, tb=True, bias=b, act="gelu", residual=g4, pre=o[8], out=o[7])
        ctx.linear_act_bwd(g4, U, o[3], o[8], "gelu", out=(o[9], o[10], o[11], o[12]))
        z, xx, gg = (a.reshape(B, T, d) for a in (x, g, o[3]))
        ctx.gated_recurrence_fwd(z, xx, out=o[13])
        ctx.gated_recurrence_bwd(gg, z, xx, o[13], out=(o[14], o[15], None))
        ctx.clip_grad_norm([o[1], o[6], o[10], o[11]], 0.5, norm=o[16])
    kept, eager = outputs(), outputs()
    step(kept)
    ctx.graph_begin()
    step(kept)
    graph = ctx.graph_end()
    for rep in range(4):
        for a, new in zip(dev, make()):
            check(lib.fx_h2d(ctx.h, a.ptr, new.ctypes.data, new.nbytes))
        new_ids = rng.integers(-1, vocab, n)
        check(lib.fx_h2d(ctx.h, ids.ptr, new_ids.ctypes.data, new_ids.nbytes))
        step(eager)
        want = [a.numpy() for a in eager]
        # other work of another size: the library's scratch grows and is used in between
        many = rng.integers(0, 50, 20000 * (rep + 1))
        ctx.embedding_bwd(ctx.fill((many.size, 4), 1.0, dtype), ctx.upload_ids(many), 50)
        ctx.graph_launch(graph)
        for k, (a, b) in enumerate(zip(kept, want)):
            assert np.array_equal(a.numpy(), b), (rep, k)
    ctx.graph_destroy(graph)


# ---- together: a training step of a small recurrent language model ------------------------------------------------------------------------------
class Model:
    """embedding -> RMS norm -> gates and values (Linear, Linear + SiLU) -> gated recurrence -> Linear + residual -> RMS norm -> logits, with the
    loss sum(logits * G) for a fixed G; every gradient by the library's calls, in place of autograd."""

    def __init__(self, ctx, rng, vocab, d, B, T, dtype):
        self.ctx, self.shape, self.dtype = ctx, (vocab, d, B, T), dtype
        n = lambda *s: (rng.standard_normal(s) / np.sqrt(s[-1])).astype(dtype)  # noqa: E731
        self.p = {"E": rng.standard_normal((vocab, d)).astype(dtype), "w1": (1 + 0.1 * rng.standard_normal(d)).astype(dtype), "Z": n(d, d),
                  "bz": np.full(d, 1.5, dtype), "X": n(d, d), "bx": n(d), "O": n(d, d), "w2": (1 + 0.1 * rng.standard_normal(d)).astype(dtype),
                  "L": n(vocab, d)}
        self.ids = rng.integers(0, vocab, (B, T))
        self.ids[0, :3] = -1
        self.G = rng.standard_normal((B * T, vocab)).astype(dtype)

    def device(self, params=None):
        return {k: self.ctx.upload(v) for k, v in (params or self.p).items()}

    def forward(self, p):
        c, (vocab, d, B, T) = self.ctx, self.shape
        s = {"ids": c.upload_ids(self.ids.ravel())}
        s["h"] = c.embedding_fwd(p["E"], s["ids"], 2.0)
        _, s["y1"], s["r1"] = c.rmsnorm_fwd(s["h"], p["w1"], 1e-6)
        s["z"] = c.gemm_bias_act_residual(s["y1"], p["Z"], tb=True, bias=p["bz"])
        s["xpre"] = c.empty((B * T, d), self.dtype)
        s["x"] = c.gemm_bias_act_residual(s["y1"], p["X"], tb=True, bias=p["bx"], act="silu", pre=s["xpre"])
        s["s"] = c.gated_recurrence_fwd(s["z"].reshape(B, T, d), s["x"].reshape(B, T, d))
        s["o"] = c.gemm(s["s"].reshape(B * T, d), p["O"], tb=True)
        s["h2"], s["y2"], s["r2"] = c.rmsnorm_fwd(s["o"], p["w2"], 1e-6, res=s["h"])
        s["logits"] = c.gemm(s["y2"], p["L"], tb=True)
        return s

    def loss(self, params):
        return float((self.forward(self.device(params))["logits"].numpy().astype(np.float64) * self.G).sum())

    def backward(self, p, s):
        c, (vocab, d, B, T) = self.ctx, self.shape
        n, g = B * T, {}
        dy2, g["L"], _ = c.linear_bwd(c.upload(self.G), p["L"], s["y2"], want_db=False)
        dh2, g["w2"] = c.rmsnorm_bwd(dy2, s["h2"], p["w2"], s["r2"])           # of h2 = o + h: the gradient of both
        ds, g["O"], _ = c.linear_bwd(dh2, p["O"], s["s"].reshape(n, d), want_db=False)
        dz, dx, _ = c.gated_recurrence_bwd(ds.reshape(B, T, d), s["z"].reshape(B, T, d), s["x"].reshape(B, T, d), s["s"])
        dy1, g["X"], g["bx"], _ = c.linear_act_bwd(dx.reshape(n, d), p["X"], s["y1"], s["xpre"], "silu")
        dy1z, g["Z"], g["bz"] = c.linear_bwd(dz.reshape(n, d), p["Z"], s["y1"])
        dy = c.binary("add", dy1, dy1z)
        dh, g["w1"] = c.rmsnorm_bwd(dy, s["h"], p["w1"], s["r1"], dh=dh2)
        g["E"] = c.embedding_bwd(dh, s["ids"], vocab, 2.0)
        return g


def test_training_step_of_a_recurrent_language_model(ctx):
    rng = np.random.default_rng(30)
    m = Model(ctx, rng, 37, 24, 3, 50, np.float64)
    p = m.device()
    s = m.forward(p)
    grads = m.backward(p, s)
    for name in m.p:
        direction = rng.standard_normal(m.p[name].shape)
        step = 1e-6
        up, down = dict(m.p), dict(m.p)
        up[name], down[name] = m.p[name] + step * direction, m.p[name] - step * direction
        want = (m.loss(up) - m.loss(down)) / (2 * step)
        got = float((grads[name].numpy() * direction).sum())
        # central differences: third derivative times step^2 / 6, and the loss' rounding (below 1e-10 of its terms) over 2 step
        assert abs(got - want) <= 2e-5 * max(1.0, abs(want), float(np.linalg.norm(grads[name].numpy()))), (name, got, want)
    # clipping and the optimizer's update on the same tables
    names = list(m.p)
    gs, ps = [grads[k] for k in names], [p[k] for k in names]
    host = [g.numpy() for g in gs]
    want, norm = ref.clip(host, 1.0)
    got = ctx.clip_grad_norm(gs, 1.0)
    assert abs(got.numpy()[0] - norm) <= ref.norm_rel(sum(g.size for g in host), np.float64) * norm and norm > 1.0
    ctx.sgd_step_multi(ps, gs, 0.1)
    for k, w in zip(names, want):
        assert np.allclose(p[k].numpy(), m.p[k] - 0.1 * w, rtol=0, atol=1e-14 * max(1.0, np.abs(m.p[k]).max()))


def test_training_step_f32_against_f64(ctx):
    """The same step in f32: every gradient within 2000 roundings of the f64 step's norm (the chain is some ten operators of at most 50
    to 200 additions per sum, on values of one size)."""
    m64 = Model(ctx, np.random.default_rng(31), 61, 40, 4, 130, np.float64)
    m32 = Model(ctx, np.random.default_rng(31), 61, 40, 4, 130, np.float32)
    for k in m64.p:
        m64.p[k] = m32.p[k].astype(np.float64)
    m64.G = m32.G.astype(np.float64)
    out = []
    for m in (m64, m32):
        p = m.device()
        out.append({k: v.numpy().astype(np.float64) for k, v in m.backward(p, m.forward(p)).items()})
    for k in out[0]:
        assert np.linalg.norm(out[0][k] - out[1][k]) <= 2000 * ref.u(np.float32) * np.linalg.norm(out[0][k]), k


def test_concurrent_contexts(ctx):
    """A second context on the same device: its own stream and scratch, results as alone."""
    from ferrox_amd import capi
    rng = np.random.default_rng(40)
    ids = rng.integers(0, 200, 5000)
    g = rng.standard_normal((5000, 64)).astype(np.float32)
    alone = ctx.embedding_bwd(ctx.upload(g), ctx.upload_ids(ids), 200).numpy()
    with capi.Context(0) as other:
        sides = [(c, c.upload(g), c.upload_ids(ids)) for c in (ctx, other)]
        outs = [c.embedding_bwd(dg, di, 200) for _ in range(3) for c, dg, di in sides]  # enqueued on both streams, nothing waits between
        for o in outs:
            assert np.array_equal(o.numpy(), alone)
        del outs, sides, o
