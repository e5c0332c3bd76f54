"""The 8-bit key/value cache and the attention over it at scores far from zero and for batches of one long sequence among many short ones."""
import numpy as np
import pytest

import lm_reference as ref
from helpers import launches, new, up
from test_gpu_lm import Recorded, attn_case, check_attn, compare_cache, i32, run_attn, tables, upload

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import Error, Tensor, ops  # noqa: E402

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


def parts_of(table, starts, lengths, picks):
    """The rows [j, j + n) of sequence b, for each (b, j, n), as sequences of their own: their tables, the rows and their lengths."""
    at = np.concatenate([np.arange(starts[b] + j, starts[b] + j + n) for b, j, n in picks])
    lens = [lengths[b] - (starts[b + 1] - starts[b]) + j + n for b, j, n in picks]
    return table[[b for b, _, _ in picks]], at, np.concatenate([[0], np.cumsum([n for _, _, n in picks])]), np.array(lens)


@pytest.mark.parametrize("heads,group,dim,seqs,long,dt", [
    (32, 8, 8, 1024, 8192, "BF16"),        # more tiles than a launch takes, were every sequence as long
    (2, 8, 64, 3, 500, "BF16"),
    (2, 8, 128, 70, 300, "F32"),           # more sequences than a wavefront has lanes
    (1, 4, 80, 130, 200, "F16"),
    (1, 12, 192, 5, 90, "BF16"),
    (1, 1, 64, 4200, 100, "BF16"),         # more than 64 times as many
])
def test_attention_of_one_long_sequence_among_many(dev, heads, group, dim, seqs, long, dt):
    """Prompts beside sequences that answer with a token, some of them over long caches, and sequences without a row."""
    news, pasts = np.ones(seqs, int), np.arange(seqs) * 29 % 190
    at = seqs // 2
    news[at], pasts[at] = long, 40
    news[0], pasts[0] = 1, 1900
    news[seqs - 1], pasts[seqs - 1] = 0, 100
    if seqs > 8:
        news[1], news[2] = 33, 5
        pasts[3] = 2500
    g, table, blocks, starts = ragged(news, pasts, 84)
    cache = ref.Cache(blocks, heads, dim, 84)
    starts = starts + 40                                                          # (rows before the first sequence)
    rows, stride = int(starts[-1]) + 3, heads * group * dim + 24
    bits = ref.to_bits(g.standard_normal((rows, stride)), dt)
    q = ref.from_bits(bits, dt)[:, 8:8 + heads * group * dim].reshape(rows, heads * group, dim)
    lengths = pasts + news
    got, lse = run_attn(dev, cache, table, starts, lengths, bits, q, rows, stride, None, group, dt, "F32", {"lse": True})
    picks = [(0, 0, 1), (at, 0, 2), (at, long // 2, 2), (at, long - 2, 2)] + [(b, 0, 1) for b in {1, 2, 3, seqs // 3, seqs - 2} if 0 < b < seqs - 1 and b != at]
    if heads * group > 64:
        picks = picks[:1] + [(at, 10, 1), (at, 400, 1), (seqs - 2, 0, 1)]        # (a row of the reference takes its time)
    tb, rw, st, ln = parts_of(table, starts, lengths, picks)
    want = ref.attention(cache, tb, st, ln, q[rw], group, dt, "F32")
    check_attn(got[rw], lse[rw], want, len(rw), str(picks))
    own = slice(int(starts[0]), int(starts[-1]))
    none = np.r_[0:own.start, own.stop:rows]
    assert (got[none] == 55.0).all() and (lse[none] == 44.0).all()
    assert np.isfinite(got[own]).all() and not (got[own] == 55.0).all(-1).any() and not (lse[own] == 44.0).any()


def test_attention_past_a_launch_is_refused(dev):
    """More blocks of threads than a launch takes are an error, not a part of the work."""
    seqs, heads, dim = 1 << 22, 8, 1
    c = ops.KvCache.new(dev, 1, heads, dim)
    table, starts, lengths = (new(dev, "I32", s) for s in ([seqs, 1], [seqs + 1], [seqs]))
    q, out = new(dev, "F32", [8, heads]), new(dev, "F32", [8, heads])
    with pytest.raises(Error, match="too many blocks of work"):
        ops.kv_attention(c, table, ops.Rows(q, 0, heads, 8, heads, dim), starts, lengths, 1, out)

def test_attention_of_prompts_beside_answers_recorded(dev):
    """A prompt beside sequences that answer with one token over long caches: two launches, the answers' caches split among more blocks of
    threads. Recorded with a workspace of the size that is asked for, and replayed when other sequences have the rows."""
    heads, group, dim, dt, seqs = 2, 8, 64, "BF16", 4
    g = np.random.default_rng(85)
    table, blocks = tables([60] * seqs, seed=85)
    cache = ref.Cache(blocks, heads, dim, 85)
    rows, width = 503, heads * group * dim
    bits = ref.to_bits(g.standard_normal((rows, width + 24)), dt)
    q = ref.from_bits(bits, dt)[:, 8:8 + width].reshape(rows, heads * group, dim)
    c, t, x = upload(dev, cache), i32(dev, table), up(dev, bits, dt, [rows, width + 24])
    starts, lengths = i32(dev, [0, 500, 501, 502, 503]), i32(dev, [500, 3800, 100, 1])
    rq, out = ops.Rows(x, 8, width + 24, rows, heads * group, dim), up(dev, np.zeros((rows, width), np.float32), "F32", [rows, width])
    size = ops.kv_attention_work(c, t, rq, starts, 500)
    whole = up(dev, np.full(size + 64, 0xA5, np.uint8), "U8", [size + 64])
    work = Tensor(whole.dtype, [size], whole.ptr(), whole, dev)

    def call():
        ops.kv_attention(c, t, rq, starts, lengths, 500, out, work=work)

    ran = [name.split("<")[0] for name, _, _ in launches(dev, call)]
    assert ran == ["kv_attn_rows_kernel", "kv_merge_kernel", "kv_attn_kernel", "kv_merge_kernel"], ran
    graph = Recorded(dev, call)
    for st, ln in (([0, 500, 501, 502, 503], [500, 3800, 100, 1]), ([0, 1, 2, 502, 503], [3800, 90, 3000, 2000]), ([0, 2, 5, 5, 405], [3000, 3, 64, 3700])):
        starts._owner.write(np.array(st, np.int32))
        lengths._owner.write(np.array(ln, np.int32))
        out._owner.write(np.full((rows, width), 55.0, np.float32))
        graph.replay()
        got = out.to_numpy().reshape(rows, heads * group, dim)
        call()                                                                    # (eager work of the context between the replays)
        assert np.array_equal(out.to_numpy().reshape(got.shape), got)
        long = int(np.argmax(np.diff(st)))
        picks = [(b, 0, st[b + 1] - st[b]) for b in range(seqs) if b != long and st[b + 1] > st[b]] + [(long, j, 1) for j in (0, 60, 399)]
        tb, rw, s2, l2 = parts_of(table, st, np.array(ln), picks)
        check_attn(got[rw], None, ref.attention(cache, tb, s2, l2, q[rw], group, dt, "F32"), len(rw), str(st))
        assert (got[st[-1]:] == 55.0).all()
        assert (whole.to_numpy()[size:] == 0xA5).all()
    graph.close()
    # (four sequences of 100 rows cannot have one of few)
    r400 = ops.Rows(x, 8, width + 24, 400, heads * group, dim)
    out, work = new(dev, "F32", [400, width]), new(dev, "U8", [ops.kv_attention_work(c, t, r400, starts, 100)])
    even = launches(dev, lambda: ops.kv_attention(c, t, r400, starts, lengths, 100, out, work=work))
    assert [name.split("<")[0] for name, _, _ in even] == ["kv_attn_rows_kernel", "kv_merge_kernel"], even


# ---- digits of answered tokens -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["BF16", "F16"])
@pytest.mark.parametrize("seqs,heads,group,dim,opts", [
    ([(1, 500), (1, 64), (2, 3)], 2, 4, 128, {}),
    ([(1, 5000)], 1, 8, 64, {}),
    ([(4, 900), (3, 200)], 2, 8, 128, {"mask": 0.7}),
    ([(1, 700)], 1, 3, 200, {"window": 300}),
    ([(1, 300), (1, 1300)], 1, 8, 160, {}),
])
def test_attention_probabilities_of_answered_tokens_in_full(dev, seqs, heads, group, dim, dt, opts):
    """16-bit queries of few rows: probabilities have float32's bits but two, as those of float32 queries."""
    case = attn_case(dev, seqs, heads, group, dim, dt, opts, seed=86)
    cache, table, starts, lengths, bits, q, rows, stride, mask = case
    got, lse = run_attn(dev, *case, group, dt, "F32", {**opts, "lse": True})
    want = ref.attention(cache, table, starts, lengths, q, group, "F32", "F32", None, opts.get("window", 0), mask)
    check_attn(got, lse, want, int(starts[-1]), str(seqs))
