"""The 8-bit key/value cache and the attention over it at scores far from zero and for batches of one long sequence among many short ones."""
import numpy as np
import pytest

import lm_reference as ref
from helpers import up
from test_gpu_lm import attn_case, compare_cache, i32, run_attn, tables, upload

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import ops  # noqa: E402

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


# ---- one long sequence among many short ones ------------------------------------------------------------------------------------

def ragged(news, pasts, seed):
    """The block table, the blocks of the pool and the starts of sequences with so many new tokens behind so many cached ones."""
    g = np.random.default_rng(seed)
    table, blocks = tables([(p + n + BLOCK - 1) // BLOCK for p, n in zip(pasts, news)], seed=seed)
    starts = np.concatenate([[0], np.cumsum(news)])
    return g, table, blocks, starts


@pytest.mark.parametrize("heads,dim,seqs,long", [
    (32, 8, 1024, 16400),        # 1024 times the longest would be more than a launch takes
    (2, 64, 3, 700),
    (1, 100, 64, 300),
    (2, 192, 65, 300),           # more sequences than a wavefront has lanes
    (1, 256, 130, 500),
    (1, 16, 4100, 200),          # more than 64 times as many
])
def test_write_and_read_of_one_long_sequence_among_many(dev, heads, dim, seqs, long):
    """The work is that of the rows there are, whichever sequences have them. Rows before the first sequence and behind the last stay."""
    news, pasts = np.ones(seqs, int), np.arange(seqs) % 67
    news[seqs // 2], news[seqs - 1] = long, 130
    if seqs > 8:
        news[3], news[4], news[6] = 0, 64, 65
    g, table, blocks, starts = ragged(news, pasts, 83)
    starts = starts + 200
    cache = ref.Cache(blocks, heads, dim, 83)
    rows = int(starts[-1]) + 2
    val = g.standard_normal((rows, 2 * heads * dim)).astype(np.float32)
    x = up(dev, val, "F32", [rows, 2 * heads * dim])
    r = [ops.Rows(x, i * heads * dim, 2 * heads * dim, rows, heads, dim) for i in (0, 1)]
    c, t, st = upload(dev, cache), i32(dev, table), i32(dev, starts)
    ops.kv_write(c, t, r[0], r[1], st, i32(dev, pasts), long)
    cache.write(table, starts, pasts, [val[:, i * heads * dim:(i + 1) * heads * dim].reshape(rows, heads, dim) for i in (0, 1)])
    compare_cache(c, cache)
    y = up(dev, np.full((rows, 2 * heads * dim), 77.0, np.float32), "F32", [rows, 2 * heads * dim])
    o = [ops.Rows(y, i * heads * dim, 2 * heads * dim, rows, heads, dim) for i in (0, 1)]
    ops.kv_read(c, t, st, i32(dev, pasts), long, o[0], o[1])
    want = np.full((rows, 2 * heads * dim), 77.0, np.float32)
    for b in range(seqs):
        for i in (0, 1):
            v, _ = cache.values(i, table[b], pasts[b] + np.arange(news[b]))
            want[starts[b]:starts[b + 1], i * heads * dim:(i + 1) * heads * dim] = v.transpose(1, 0, 2).reshape(-1, heads * dim)
    assert np.array_equal(y.to_numpy(), want)
