"""The 8-bit key/value cache and the attention over it at scores far from zero."""
import numpy as np
import pytest

import lm_reference as ref
from test_gpu_lm import attn_case, run_attn

pytestmark = pytest.mark.gpu

BLOCK = ref.BLOCK


# ---- scores far from zero ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("seqs", [[(1, 300), (1, 2000)], [(40, 300)], [(40, 1700)]])
@pytest.mark.parametrize("dt", ["BF16", "F32"])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_scores_past_the_steps_of_float32(dev, seqs, dt, sign):
    """One key far ahead of the others, at scores of both signs up to 2^80, where neighbouring float32 numbers are more than 1 apart: its
    probability is 1, so the row is its value and the log sum its score."""
    heads, group, dim, win = 1, 4, 64, 70
    cache, table, starts, lengths, bits, q, rows, stride, _ = attn_case(dev, seqs, heads, group, dim, dt, {}, seed=81)
    g = np.random.default_rng(82)
    # all of q's features are one positive number, so a score is that number times the sum of the key's codes
    if sign > 0:
        cache.k[:] = g.integers(-50, 51, cache.k.shape)
        best = 127
    else:
        cache.k[:] = g.integers(-127, -99, cache.k.shape)
        best = -20
    cache.s[0] = 0.02 * (1 + 0.1 * g.random(cache.s[0].shape))
    for b in range(len(seqs)):
        cache.k[table[b, win // BLOCK], :, win % BLOCK] = best
    rate = np.abs(dim * best * 0.02 * dim ** -0.5)                              # about a score at q = 1
    power = np.linspace(18, 80, rows * group).reshape(rows, group)
    q1 = ref.from_bits(ref.to_bits((2.0 ** power * (1 + g.random(power.shape)) / rate).astype(np.float32), dt), dt)
    val = np.zeros((rows, stride), np.float32)
    val[:, 8:8 + group * dim] = np.repeat(q1, dim, 1)
    out, lse = run_attn(dev, cache, table, starts, lengths, ref.to_bits(val, dt), None, rows, stride, None, group, dt, "F32", {"lse": True})
    for b in range(len(seqs)):
        page, at = table[b, win // BLOCK], slice(starts[b], starts[b + 1])
        want = cache.v[page, 0, :, win % BLOCK].astype(np.float64) * cache.s[1, page, 0]
        score = q1[at].astype(np.float64) * dim * best * np.float64(cache.s[0, page, 0]) * dim ** -0.5
        # the other keys are at least a tenth of 2^18 behind; a probability of 16-bit queries is off by half a step of half
        rel = (2.0 ** -11 if dt != "F32" else 2.0 ** -22) + 2.0 ** -21
        assert (np.abs(out[at] - want) <= rel * np.abs(want)).all(), np.abs(out[at] - want).max()
        # float32 queries as two halves (2^-22) and some six roundings of the score (2^-24 each)
        assert (np.abs(lse[at] - score) <= 2.0 ** -20 * np.abs(score)).all()
