"""Attention over the key/value cache (include/h3lm.h, kv_attention and kv_attention_spans), against its restatement in numpy
(spans_reference.py): to how many bits sequences of few rows have their results beside longer ones, and the launches that shared tokens take
where sequences have many rows."""
import numpy as np
import pytest

import lm_reference as lm
import spans_reference as ref
from helpers import launches, new, up
from test_gpu_lm import Recorded, check_attn
from test_gpu_spans import Case, context

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import Tensor, ops  # noqa: E402


@pytest.fixture(scope="module")
def cus():
    """Contexts that size their grids for so many compute units."""
    made = {}
    yield lambda n: made.setdefault(n, None) or made.update({n: context(n)}) or made[n]
    for d in made.values():
        d.close()


@pytest.fixture(scope="module")
def dev2(cus):
    return cus(2)


def kernels(case, out_dt="F32", **kw):
    """The launches of a call, by the kernels' names with their template arguments."""
    args, shared, mask = case.upload()
    wide = case.heads * case.group
    out = new(case.dev, out_dt, [case.rows, wide * case.dim])
    n = ops.kv_attention_work(*args[:4], case.most, shared=shared, **kw)
    work = new(case.dev, "U8", [max(n, 16)])
    return [k for k, _, _ in launches(case.dev, lambda: ops.kv_attention(*args, out, shared=shared, mask=mask, work=work, **kw))]


DIGITS = [
    # sequences, heads, group, dim, groups, window, first tokens, on two compute units
    ([(1, 1500 + b) for b in range(7)] + [(8, 1400)], 1, 8, 128, (), 1024, 4, False),
    ([(1, 1500 + b) for b in range(7)] + [(8, 1400)], 1, 8, 128, (), 0, 0, False),
    ([(4, 300), (3, 200), (70, 320), (2, 250), (1, 200)], 2, 8, 128, (), 0, 0, False),
    ([(8, 300), (70, 320), (1, 200)], 2, 4, 64, (), 100, 3, True),
    ([(1, 300), (90, 320), (1, 200)], 1, 30, 64, (), 0, 0, False),
    ([(1, 300), (90, 320), (2, 200)], 1, 8, 256, (), 0, 0, True),
    ([(40, 300), (30, 320), (2, 200), (30, 330), (3, 280)], 2, 4, 96, (), 90, 70, False),
    ([(1, 900), (20, 920), (2, 930), (1, 960)] * 3, 1, 8, 128, [(0, 12, 832)], 0, 0, True),
    ([(1, 900), (20, 920), (2, 930), (1, 960)] * 3, 1, 8, 128, [(0, 12, 832)], 700, 30, True),
]


@pytest.mark.parametrize("dt", ["BF16", "F16"])
@pytest.mark.parametrize("seqs,heads,group,dim,groups,window,sinks,two", DIGITS)
def test_digits_of_few_rows_beside_many(dev, dev2, seqs, heads, group, dim, groups, window, sinks, two, dt):
    """Float32 results of 16-bit queries, of sequences with up to 32 rows times heads of a group (16 of more than 128 features), are float32's
    beside any others: a term's error is that of its score, below 2^3, in float32 (2^-20 of the term; probabilities as two halves add 2^-22),
    and terms and errors add up alike. Eight times that is allowed. (Probabilities as one half are off by up to 2^-11 each.)"""
    case = Case(dev2 if two else dev, seqs, heads, group, dim, dt, groups, seed=41)
    few = [r for b, (n, _) in enumerate(seqs) if n * group <= (32 if dim <= 128 else 16) for r in range(case.starts[b], case.starts[b] + n)]
    got = case.run(window=window, sinks=sinks, scale=0.02)[0][few]
    want = ref.attention(case.cache, case.table, case.starts, case.lengths, case.q, group, dt, "F32", np.float32(0.02), window, sinks, None,
                         case.first, case.tokens, rows=set(few))[0][few]
    assert np.sqrt(((got - want) ** 2).mean()) <= 2.0 ** -17 * np.sqrt((want ** 2).mean())


@pytest.mark.parametrize("dt,out_dt", [("BF16", "F32"), ("F16", "F16")])
@pytest.mark.parametrize("units", [256, 2])
def test_few_rows_beside_many_by_launches(cus, dt, out_dt, units):
    """Sequences of up to 32 rows beside a long one are a launch of tiles of 16 (most have no more) or 32; where none is long all are a launch of the
    rows' kernel with probabilities as two halves. With a window, first tokens and a mask too."""
    for seqs, few in (([(4, 300), (1, 200), (70, 320), (2, 250), (0, 9), (1, 200), (1, 4)], 1),
                      ([(4, 300), (3, 200), (70, 320), (4, 250), (0, 9), (1, 200), (4, 4)], 2),
                      ([(4, 2500), (1, 3000), (5, 700)], 0), ([(40, 300), (2, 280), (0, 7), (1, 200)], 0)):
        for mask in (None, 0.6):
            case = Case(cus(units), seqs, 2, 8, 128, dt, seed=45, mask=mask)
            for window, sinks in ((0, 0), (100, 0), (100, 30)):
                mode = 1 if sinks else 0
                ran = kernels(case, out_dt, window=window, sinks=sinks)
                if few:
                    assert any(r.startswith(f"kv_attn_kernel<2, {few}, false, {mode}>") for r in ran) and ", false>" in ran[0], ran
                else:
                    assert ran[0].startswith(f"kv_attn_rows_kernel<2, 1, false, {mode}, true>"), ran
                rows = some_rows(case, 60) if case.rows < 50 else [r for r in range(case.starts[-1]) if r < 8 or r > 72]
                check_rows(case, case.run(out_dt, window=window, sinks=sinks), rows, out_dt, str((seqs, window, mask)), window=window, sinks=sinks)


def batch(most, mixed, seqs, tokens, own, groups):
    """Sequences of about `most` rows (every third of one, if mixed) and `own` tokens behind the `tokens` that their group shares."""
    rows = [1 if mixed and i % 3 == 0 else max(most - i % 3, 1) for i in range(seqs)]
    edge = [i * seqs // groups for i in range(groups + 1)]
    return [(n, tokens + own + i) for i, n in enumerate(rows)], [(a, e, tokens) for a, e in zip(edge, edge[1:])]


APART = [
    # (rows, mixed, sequences, shared tokens, own tokens, groups), heads, group, dim, type, result, window, compute units, the launches: of the shared
    # tokens, of the sequences' own, whether those have parts, and of the sequences with few rows
    ((9, 0, 12, 960, 40, 1), 1, 8, 128, "BF16", "BF16", 0, 2, "rows2 rows2"),
    ((9, 0, 12, 960, 40, 1), 1, 8, 128, "BF16", "BF16", 700, 2, "rows2 rows2"),
    ((9, 0, 12, 960, 40, 1), 1, 8, 128, "F32", "F32", 0, 2, "rows1 rows1"),
    ((9, 0, 12, 960, 40, 1), 1, 8, 128, "F32", "BF16", 0, 2, "rows1 rows1"),
    ((60, 1, 4, 640, 40, 3), 1, 2, 160, "BF16", "BF16", 1000, 2, "rows1 rows2"),
    ((20, 0, 8, 448, 40, 3), 1, 4, 64, "BF16", "BF16", 0, 2, "rows2 rows2"),
    ((17, 1, 4, 640, 300, 2), 1, 7, 96, "BF16", "BF16", 1000, 2, "rows2 rows2"),
    ((5, 0, 6, 256, 40, 2), 1, 4, 256, "BF16", "BF16", 0, 4, "rows1 rows1"),
    ((30, 1, 20, 960, 700, 3), 1, 4, 80, "BF16", "BF16", 0, 8, "rows2 rows2 join"),
    ((3, 0, 6, 960, 700, 1), 2, 8, 160, "BF16", "BF16", 0, 8, "rows2 rows1 join"),
    ((9, 0, 20, 448, 700, 3), 1, 2, 160, "BF16", "BF16", 0, 16, "rows1 rows1 join"),
    ((3, 1, 6, 448, 700, 2), 1, 16, 160, "F32", "F32", 0, 4, "rows1 rows1 join"),
    ((9, 0, 6, 448, 700, 1), 1, 2, 160, "F32", "F32", 1000, 4, "rows1 rows1 join"),
    ((9, 1, 20, 256, 700, 1), 1, 4, 256, "F32", "F32", 1000, 8, "rows1 rows1 join"),
    ((20, 1, 4, 960, 40, 2), 1, 2, 64, "BF16", "F32", 0, 2, "rows1h rows1h"),
    ((12, 1, 6, 256, 40, 2), 1, 2, 160, "F16", "F32", 300, 1, "rows1h rows1h"),
    ((20, 0, 6, 640, 700, 1), 1, 1, 160, "BF16", "F32", 0, 4, "rows1h rows1h join"),
    ((20, 1, 4, 1280, 700, 3), 1, 1, 160, "BF16", "F32", 0, 8, "few1 rows1h join"),
    ((12, 1, 4, 640, 3000, 4), 1, 2, 256, "F16", "F16", 0, 4, "few1 rows1h few1 join"),
    ((9, 0, 4, 1280, 3000, 1), 1, 2, 256, "BF16", "F32", 0, 4, "rows1h rows1h few1 join"),
    ((20, 1, 4, 1280, 3000, 1), 1, 1, 160, "F32", "F32", 0, 4, "rows1 rows1 few1 join"),
    ((17, 0, 20, 4096, 37, 20), 1, 4, 64, "F16", "F16", 4096, 16, "rows1h rows1 few2"),
    ((5, 0, 20, 4096, 25, 2), 1, 16, 80, "BF16", "F32", 0, 1, "rows1h rows2 few2"),
    ((20, 1, 4, 640, 300, 3), 1, 1, 160, "BF16", "BF16", 1000, 4, "few1 rows1"),
    ((20, 1, 4, 1280, 40, 3), 2, 2, 80, "F32", "F32", 0, 4, "few2 rows1"),
    ((20, 1, 4, 640, 100, 3), 1, 2, 80, "F16", "F32", 1000, 1, "few2 rows1h"),
    ((20, 0, 4, 448, 100, 1), 1, 1, 80, "F32", "F32", 0, 2, "rows1 few2"),
    ((12, 1, 4, 448, 40, 1), 1, 2, 96, "F16", "F32", 700, 2, "rows1h few2"),
]


def named(want, dim, dt):
    """The kernels that a line of APART means (h: probabilities as two halves, as those of float32 queries are)."""
    wide, two, seen, tile = (dim + 63) // 64, "true" if dt == "F32" else "false", [], 0
    for word in want.split():
        mode, tiles = 1 if seen else 2, word.strip("rowsfewjoinh")
        if word == "join":
            seen.append(f"kv_join_kernel<{wide}, {tile}>")
        elif word.startswith("few"):
            seen.append(f"kv_attn_kernel<{wide}, {tiles}, {two}, {mode}>")
        else:
            seen.append(f"kv_attn_rows_kernel<{wide}, {tiles}, {two}, {mode}, {'true' if word[-1] == 'h' else two}>")
        tile = (64 if word[0] == "r" else 16) * int(tiles or 0)
    return seen


def some_rows(case, count=36):
    """Rows to look at: the first and last of the first and last sequences, others anywhere."""
    used = int(case.starts[-1])
    ends = {0, used - 1, int(case.starts[1]) - 1, int(case.starts[-2])}
    return sorted(ends | set(np.random.default_rng(93).permutation(used)[:count].tolist()))


def check_rows(case, got, rows, out_dt, what="", **kw):
    want = ref.attention(case.cache, case.table, case.starts, case.lengths, case.q, case.group, case.dt, out_dt, kw.get("scale"), kw.get("window", 0),
                         kw.get("sinks", 0), case.mask, case.first, case.tokens, rows=set(rows))
    used = int(case.starts[-1])
    check_attn(got[0][rows], got[1][rows], [w[rows] for w in want], len(rows), what)
    assert (got[0][used:] == 55.0).all() and (got[1][used:] == 44.0).all(), what


@pytest.mark.parametrize("shape,heads,group,dim,dt,out_dt,window,units,want", APART)
def test_shared_tokens_apart_from_many_rows(cus, shape, heads, group, dim, dt, out_dt, window, units, want):
    """A launch of the shared tokens and one of the sequences' own of many rows, which takes up its sums or leaves parts to join; with a mask too."""
    dev, kw = cus(units), dict(window=window, sinks=20 if window else 0)
    seqs, groups = batch(*shape)
    for mask in (None, 0.5):
        case = Case(dev, seqs, heads, group, dim, dt, groups, seed=42, mask=mask)
        ran = kernels(case, out_dt, **kw)
        names = named(want, dim, dt)
        assert [r[:len(n)] for r, n in zip(ran, names)] == names and len(ran) == len(names), (ran, names)
        check_rows(case, case.run(out_dt, **kw), some_rows(case), out_dt, f"mask {mask}", **kw)


MANY = [0, 1, 4, 6, 8, 12, 14, 17, 18, 20]   # of APART: each kind of launch


@pytest.mark.parametrize("i", MANY)
def test_shared_blocks_that_are_not_there_or_not_finite(cus, i):
    """Shared blocks that are not in the table, all of them too, and one whose scales are NaN and that the mask hides."""
    shape, heads, group, dim, dt, out_dt, window, units, _ = APART[i]
    kw = dict(window=window, sinks=20 if window else 0)
    seqs, groups = batch(*shape)
    case = Case(cus(units), seqs, heads, group, dim, dt, groups, seed=43)
    for a, _, _ in groups:
        case.table[a, [0, 3]] = [-1, 1 << 29]
    rows = some_rows(case, 12)
    check_rows(case, case.run(out_dt, **kw), rows, out_dt, "some", **kw)
    for a, _, n in groups:
        case.table[a, :n // 64] = -1
    check_rows(case, case.run(out_dt, **kw), rows, out_dt, "none", **kw)
    case = Case(cus(units), seqs, heads, group, dim, dt, groups, seed=43)
    for a, _, n in groups:
        case.cache.s[:, case.table[a, n // 64 - 1]] = np.nan                        # (the last shared one, which every row sees)
    case.mask = np.ones((len(seqs), int(case.lengths.max())), np.uint8)
    case.mask[:, shape[3] - 64:shape[3]] = 0
    check_rows(case, case.run(out_dt, **kw), rows, out_dt, "hidden", **kw)
    case.mask = None
    assert np.isnan(case.run(out_dt, **kw)[0][:int(case.starts[-1])]).all()


@pytest.mark.parametrize("i", MANY)
def test_apart_recorded(cus, i):
    """Recorded with a workspace of the size that is asked for, full of NaN, and replayed on other lengths and shared tokens: what an eager call
    gives, bit for bit, and nothing behind the workspace is written."""
    shape, heads, group, dim, dt, out_dt, window, units, _ = APART[i]
    dev, kw = cus(units), dict(window=window, sinks=20 if window else 0)
    seqs, groups = batch(*shape)
    case = Case(dev, seqs, heads, group, dim, dt, groups, seed=44)
    args, shared, _ = case.upload()
    wide, used = heads * group, int(case.starts[-1])
    size = ops.kv_attention_work(*args[:4], case.most, shared=shared, **kw)
    whole = up(dev, np.full(size + 64, 0xFF, np.uint8), "U8", [size + 64])
    work = Tensor(whole.dtype, [size], whole.ptr(), whole, dev)
    out = up(dev, lm.to_bits(np.full((case.rows, wide * dim), 55.0), out_dt), out_dt, [case.rows, wide * dim])
    lse = up(dev, np.full((case.rows, wide), 44.0, np.float32), "F32", [case.rows, wide])
    graph = Recorded(dev, lambda: ops.kv_attention(*args, out, shared=shared, work=work, lse=lse, **kw))
    rows, lengths, tokens = some_rows(case, 6), case.lengths.copy(), list(case.tokens)
    for step in range(3):
        case.lengths = np.maximum(lengths - 41 * step, 1)
        case.tokens = [max(n - 128 * step + step, 0) for n in tokens]
        args[4]._owner.write(case.lengths.astype(np.int32))
        shared.tokens._owner.write(np.array(case.tokens, np.int32))
        whole._owner.write(np.full(size + 64, 0xFF, np.uint8))
        graph.replay()
        got = out.to_numpy(), lse.to_numpy()
        assert (whole.to_numpy()[size:] == 0xFF).all()
        ops.kv_attention(*args, out, shared=shared, lse=lse, **kw)
        assert np.array_equal(got[0], out.to_numpy()) and np.array_equal(got[1], lse.to_numpy()), step
        # (the entries behind a group's fewer shared tokens name blocks that are not there)
        check_rows(case, (lm.from_bits(got[0], out_dt).reshape(case.rows, wide, dim), got[1]), rows, out_dt, str(step), **kw)
        assert used < case.rows
    graph.close()
