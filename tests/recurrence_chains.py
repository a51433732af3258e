"""Long recurrences whose pieces matter to one another: gates near 1 over dozens of pieces, first and last states well above the inputs,
and a model of how pieces hand their maps on, with the mistakes that such inputs have to show."""
import numpy as np

import lm_reference as ref

GROUP = 32


def piece_steps(dtype, back):
    return 128 if dtype == np.float32 else (32 if back else 64)


# B, T, D: more than one group of pieces in both directions and types, a partial last tile of chains, chains of two sequences in one tile
SHAPES = [(1, 4500, 70), (2, 8300, 3), (1, 4097, 64), (3, 9000, 33)]


def inputs(B, T, D, dtype):
    """z near 8 (a product over 128 gates is about 0.95), every fifth chain with open gates throughout (what enters it arrives as it is)."""
    rng = np.random.default_rng(T + D)
    z = (8 + rng.standard_normal((B, T, D))).astype(dtype)
    z[:, :, ::5] = np.inf
    x, dh = rng.standard_normal((B, T, D)).astype(dtype), (0.001 * rng.standard_normal((B, T, D))).astype(dtype)
    h0, nxt = ((10 + rng.random((B, D))) * np.where(rng.random((B, D)) < 0.5, -1, 1)).astype(dtype), (10 + rng.random((B, D))).astype(dtype)
    return z, x, h0, dh, nxt


def states(A, H, start, steps, mistake=None):
    """v_t = A_t v_(t-1) + H_t along axis 1 from `start`, by pieces of `steps`: the state in front of a piece comes from the maps of the
    pieces since the last multiple of GROUP and the state that was published there.  mistake: what the hand-over does wrong."""
    B, T, D = A.shape
    out, maps, published = np.zeros((B, T, D)), [], []
    for p in range(-(-T // steps)):
        part = range(p * steps, min(T, (p + 1) * steps))
        g0 = p // GROUP * GROUP
        v = start if g0 == 0 or mistake == "no group state" else published[g0 // GROUP - 1]
        if mistake == "no first state" and p > 0:
            v = 0 * start
        for a, h in (maps[g0:p - 1] if mistake == "a map short" else maps[g0:p]):
            v = (0 if mistake == "no A" else a) * v + (0 if mistake == "no H" else h)
        a, h = np.ones((B, D)), np.zeros((B, D))
        for t in part:
            v = A[:, t] * v + H[:, t]
            out[:, t] = v
            a, h = A[:, t] * a, A[:, t] * h + H[:, t]
        maps.append((a, h))
        if p % GROUP == GROUP - 1:
            published.append(v)
    return out


MISTAKES = ["no A", "no H", "no first state", "no group state", "a map short"]


def check_forward(got, z, x, h0):
    want, bound = ref.recurrence_fwd(z, x, h0)
    assert (np.abs(got - want) <= bound).all()
    open_ = np.isposinf(z).all(1)  # [B, D]: kept bit for bit
    assert (got == np.where(open_, h0, 0)[:, None])[np.broadcast_to(open_[:, None], got.shape)].all()


def check_backward(dz, dx, dh0, dh, z, x, h, h0, nxt):
    want, bounds = ref.recurrence_bwd(dh, z, x, h, h0, nxt)
    for g, w, b in zip((dz, dx, dh0), want, bounds):
        if g is not None:
            assert (np.abs(g - w) <= b).all()
