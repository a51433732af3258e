"""The inputs of the long recurrences' GPU tests, on the CPU: the step-by-step definition cut into pieces holds the bounds, and every
mistake in what one piece hands to the next breaks them."""
import numpy as np
import pytest

import lm_reference as ref
import recurrence_chains as rc


@pytest.mark.parametrize("dtype", [np.float32, np.float64])
@pytest.mark.parametrize("B,T,D", rc.SHAPES)
def test_mistakes_between_pieces_show(B, T, D, dtype):
    z, x, h0, dh, nxt = rc.inputs(B, T, D, dtype)
    f, k = ref.sigmoid(z.astype(np.float64)), ref.sigmoid(-z.astype(np.float64))
    steps, back = rc.piece_steps(dtype, False), rc.piece_steps(dtype, True)
    assert T > rc.GROUP * steps and T > rc.GROUP * back
    h = rc.states(f, k * x, h0.astype(np.float64), steps)
    rc.check_forward(h, z, x, h0)
    for m in rc.MISTAKES:
        with pytest.raises(AssertionError):
            rc.check_forward(rc.states(f, k * x, h0.astype(np.float64), steps, m), z, x, h0)

    def gradients(mistake=None):  # C_q = f (dh + C_(q-1)) against time; S = dh + C
        rev = slice(None, None, -1)
        C = rc.states(f[:, rev], (f * dh)[:, rev], nxt.astype(np.float64), back, mistake)[:, rev]
        S = dh + np.concatenate([C[:, 1:], nxt[:, None]], 1)
        before = np.concatenate([h0[:, None], h[:, :-1]], 1)
        return S * (before - x) * f * k, k * S, C[:, 0]
    rc.check_backward(*gradients(), dh, z, x, h, h0, nxt)
    for m in rc.MISTAKES:
        with pytest.raises(AssertionError):
            rc.check_backward(*gradients(m), dh, z, x, h, h0, nxt)
