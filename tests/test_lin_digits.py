"""That the limits for linear attention in pieces (lin_pieces.py) tell its arithmetic from the same with a part less, in numpy."""
import numpy as np
import pytest

import lin_pieces as ref
import lm_reference as lm


def inputs(n, dk, dv, dt):
    g = np.random.default_rng(91)
    return [lm.from_bits(lm.to_bits(g.standard_normal((n, d)), dt), dt) for d in (dk, dk, dv)]


def exact(q, k, v, decay):
    s, out = np.zeros((q.shape[1], v.shape[1])), np.zeros(v.shape)
    for t in range(len(q)):
        s = np.exp(-np.float64(decay)) * s + np.outer(k[t].astype(np.float64), v[t])
        out[t] = q[t].astype(np.float64) @ s * q.shape[1] ** -0.5
    return out, s


@pytest.mark.parametrize("dt", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("n,dk,dv", [(40, 64, 32), (300, 128, 32), (700, 96, 16), (100, 256, 32)])
def test_a_part_less_is_seen(n, dk, dv, dt):
    q, k, v = inputs(n, dk, dv, dt)
    most = ref.FULL if dt == "F32" else ref.HELD
    for decay in ref.DECAYS:
        want = exact(q, k, v, decay)
        out, s = (ref.error(x, w) for x, w in zip(ref.pieces(q, k, v, decay, dt), want))
        assert out <= most / 1.5 and s <= ref.FULL / 1.5, (out, s)
        out, _ = (ref.error(x, w) for x, w in zip(ref.pieces(q, k, v, decay, dt, held=2 if dt == "F32" else 1), want))
        assert out > 2 * most, out
        _, s = (ref.error(x, w) for x, w in zip(ref.pieces(q, k, v, decay, dt, taken=2), want))
        assert s > 2 * ref.FULL, s
        if dt != "BF16":
            out, s = (ref.error(x, w) for x, w in zip(ref.pieces(q, k, v, decay, dt, inputs=ref.PARTS[dt] - 1), want))
            assert s > 2 * ref.FULL and out > 2 * most, (out, s)
