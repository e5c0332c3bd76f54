"""The 8-bit key/value cache, the attention over it and the 4-bit linear layer (include/h3lm.h) against their restatement in
numpy: the cache bit for bit, the others within bounds derived from the types (lm_reference.py)."""
import numpy as np
import pytest

import lm_reference as ref
from helpers import launches, new, up

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import Device, Error, Tensor, ops  # noqa: E402

BLOCK = ref.BLOCK


def upload(dev, c: ref.Cache):
    w = ref.width(c.dim)
    return ops.KvCache(up(dev, c.k, "I8", [c.blocks, c.heads, BLOCK, w]), up(dev, c.v, "I8", [c.blocks, c.heads, w, BLOCK]),
                       up(dev, c.s[0], "F32", [c.blocks, c.heads]), up(dev, c.s[1], "F32", [c.blocks, c.heads]), c.dim)


def i32(dev, a):
    a = np.ascontiguousarray(a, np.int32)
    return up(dev, a, "I32", list(a.shape))


def tables(seqs_blocks, spare=2, seed=1):
    """Block tables of sequences of so many blocks, in a shuffled pool; unused entries -1. Returns (table, blocks of the pool)."""
    g = np.random.default_rng(seed)
    total = sum(seqs_blocks) + spare
    order = g.permutation(total)
    t = np.full((len(seqs_blocks), max(max(seqs_blocks), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(seqs_blocks):
        t[b, :n] = order[at:at + n]
        at += n
    return t, total


def compare_cache(got: ops.KvCache, want: ref.Cache, finite=None):
    k, v = got.k.to_numpy(), got.v.to_numpy()
    s = np.stack([got.k_scale.to_numpy(), got.v_scale.to_numpy()]).reshape(want.s.shape)
    assert np.array_equal(s, want.s, equal_nan=True), f"scales: {np.argwhere(~((s == want.s) | (np.isnan(s) & np.isnan(want.s))))[:5]}"
    good = np.isfinite(want.s)
    for name, a, b, ok in (("k", k, want.k, good[0]), ("v", v, want.v, good[1])):
        bad = np.argwhere((a != b) & ok[:, :, None, None])
        assert len(bad) == 0, f"{name}: {len(bad)} codes differ, first {bad[:3]}: {a[tuple(bad[0])]} for {b[tuple(bad[0])]}"


# ---- kv_write, kv_read ------------------------------------------------------------------------------------------------------

WRITES = [
    # heads, dim, type, (past, new) of each sequence
    (8, 128, "BF16", [(299, 1)]),
    (2, 128, "F16", [(0, 1), (63, 1), (64, 1), (127, 2), (5, 0)]),
    (1, 64, "BF16", [(0, 64), (0, 65), (1, 63), (1, 64), (30, 200)]),
    (3, 80, "F32", [(17, 40), (0, 0), (100, 30)]),
    (2, 100, "BF16", [(10, 70), (64, 5)]),
    (4, 96, "F16", [(0, 300)]),
    (2, 192, "BF16", [(50, 30), (0, 3)]),
    (2, 256, "F32", [(13, 77), (64, 64)]),
    (1, 1, "F32", [(0, 70)]),
    (2, 7, "F16", [(3, 130)]),
]


def write_case(heads, dim, dt, seqs, seed, tail=3, stride=None, offset=0):
    g = np.random.default_rng(seed)
    table, blocks = tables([(p + n + BLOCK - 1) // BLOCK for p, n in seqs], seed=seed)
    cache = ref.Cache(blocks, heads, dim, seed)
    starts = np.concatenate([[0], np.cumsum([n for _, n in seqs])])
    rows = int(starts[-1]) + tail
    stride = stride or 2 * heads * dim
    bits = ref.to_bits(g.standard_normal((rows, stride)) * np.exp(g.normal(0, 1, (rows, 1))), dt)
    val = ref.from_bits(bits, dt)
    at = (offset, offset + heads * dim)
    kv = [val[:, a:a + heads * dim].reshape(rows, heads, dim) for a in at]
    return table, cache, starts, bits, kv, at, rows, stride


@pytest.mark.parametrize("heads,dim,dt,seqs", WRITES)
def test_write_and_read(dev, heads, dim, dt, seqs):
    table, cache, starts, bits, kv, at, rows, stride = write_case(heads, dim, dt, seqs, 7 + heads * dim)
    past = np.array([p for p, _ in seqs])
    most = max(n for _, n in seqs)
    c, t = upload(dev, cache), i32(dev, table)
    x = up(dev, bits, dt, [rows, stride])
    r = [ops.Rows(x, a, stride, rows, heads, dim) for a in at]
    ops.kv_write(c, t, r[0], r[1], i32(dev, starts), i32(dev, past), most)
    cache.write(table, starts, past, kv)
    compare_cache(c, cache)
    # the sequences from some token on as values, in each type, into rows wider than they need; rows behind the last stay
    first = np.maximum(past - 3, 0)
    counts = [p + n - f if n else 0 for (p, n), f in zip(seqs, first)]
    s2 = np.concatenate([[0], np.cumsum(counts)])
    n2, wide = int(s2[-1]) + 2, heads * dim + 8
    for out in ("F32", "BF16", "F16"):
        mark = ref.to_bits(np.full((n2, 2 * wide), 77.0), out)
        y = up(dev, mark, out, [n2, 2 * wide])
        ko, vo = (ops.Rows(y, i * wide, 2 * wide, n2, heads, dim) for i in (0, 1))
        ops.kv_read(c, t, i32(dev, s2), i32(dev, first), max(max(counts), 1), ko, vo)
        want = mark.copy()
        for b in range(len(seqs)):
            for i in (0, 1):
                val, _ = cache.values(i, table[b], first[b] + np.arange(counts[b]))
                want[s2[b]:s2[b + 1], i * wide:i * wide + heads * dim] = ref.to_bits(val.transpose(1, 0, 2).reshape(-1, heads * dim), out)
        assert np.array_equal(y.to_numpy(), want), out


def test_tokens_one_by_one(dev):
    """A sequence grows token by token over three blocks; the scales rise on the way, and every step is the restatement's."""
    heads, dim = 2, 128
    g = np.random.default_rng(3)
    table, blocks = tables([3])
    cache = ref.Cache(blocks, heads, dim, 5)
    c, t, starts = upload(dev, cache), i32(dev, table), i32(dev, [0, 1])
    for p in range(0, 150, 1):
        val = (g.standard_normal((1, 2 * heads * dim)) * (1 + 0.05 * p)).astype(np.float32)
        x = up(dev, val, "F32", [1, 2 * heads * dim])
        r = [ops.Rows(x, i * heads * dim, 2 * heads * dim, 1, heads, dim) for i in (0, 1)]
        ops.kv_write(c, t, r[0], r[1], starts, i32(dev, [p]), 1)
        cache.write(table, [0, 1], [p], [val[:, i * heads * dim:(i + 1) * heads * dim].reshape(1, heads, dim) for i in (0, 1)])
        if p % 25 == 24 or p in (0, 63, 64):
            compare_cache(c, cache)


def test_write_odd_values_and_pages(dev):
    """Zeros, denormals, infinities and NaN in new tokens; a NaN scale in a block that is used afresh; pages that are not there;
    tokens past the table's end; sequences whose starts run past the rows."""
    heads, dim = 2, 64
    seqs = [(0, 5), (10, 4), (0, 64), (70, 8), (60, 10), (120, 20), (0, 3)]
    table, blocks = tables([2] * 7)
    table[3, 1], table[4, 0] = blocks + 5, -7                              # not there: 3 writes nothing, 4 only its second block
    cache = ref.Cache(blocks, heads, dim, 9)
    cache.s[:, table[2, 0]] = np.nan                                       # (no token was there: not looked at)
    starts = np.concatenate([[0], np.cumsum([n for _, n in seqs])])
    rows = int(starts[-1])
    g = np.random.default_rng(4)
    val = g.standard_normal((rows, 2 * heads * dim)).astype(np.float32)
    val[starts[0]:starts[1]] = 0
    val[starts[1], 3], val[starts[1] + 1, heads * dim + 70] = np.inf, np.nan
    val[starts[6]:starts[7]] = 1e-39
    x = up(dev, val, "F32", [rows, 2 * heads * dim])
    kv = [val[:, i * heads * dim:(i + 1) * heads * dim].reshape(rows, heads, dim) for i in (0, 1)]
    c, t = upload(dev, cache), i32(dev, table)
    past = np.array([p for p, _ in seqs])
    r = [ops.Rows(x, i * heads * dim, 2 * heads * dim, rows, heads, dim) for i in (0, 1)]
    ops.kv_write(c, t, r[0], r[1], i32(dev, starts), i32(dev, past), 64)
    cache.write(table, starts, past, kv)
    compare_cache(c, cache)
    # starts out of order and out of range: cut to the rows, nothing outside is touched
    wild = np.array([0, 4, 2, -9, 1 << 30, rows, rows + 1000, 3])
    ops.kv_write(c, t, r[0], r[1], i32(dev, wild), i32(dev, past), 8)
    dev.wait()


# ---- kv_attention ------------------------------------------------------------------------------------------------------------

ATTN = [
    # (new, length) of each sequence, heads, group, dim, type, out type, options
    ([(1, 300)], 8, 8, 128, "BF16", "BF16", {}),
    ([(1, 1), (1, 64), (1, 65), (1, 200), (0, 50), (1, 0)], 2, 4, 128, "F16", "F16", {"lse": True}),
    ([(1, 700)], 1, 1, 64, "BF16", "F32", {"lse": True}),
    ([(1, 2100), (1, 90)], 1, 16, 128, "BF16", "BF16", {"lse": True}),          # split, sequences of other lengths
    ([(2, 130), (3, 3), (1, 500)], 2, 8, 96, "F16", "BF16", {}),               # 24 rows: two tiles of 16
    ([(7, 71), (5, 400)], 2, 8, 80, "BF16", "BF16", {"window": 33}),           # 56 rows: two tiles of 32
    ([(40, 40), (13, 200)], 2, 4, 128, "BF16", "BF16", {"lse": True}),         # rows of their own for each wavefront
    ([(100, 163)], 1, 7, 64, "F16", "F16", {"window": 50, "mask": 0.7}),
    ([(130, 1000)], 1, 1, 128, "BF16", "BF16", {"lse": True}),                 # few tiles: split
    ([(33, 80)], 2, 3, 100, "BF16", "BF16", {}),                               # rows that are no 16-byte pieces
    ([(5, 77), (1, 130)], 2, 2, 7, "F16", "F32", {"mask": 0.5, "lse": True}),
    ([(1, 400), (2, 64)], 2, 4, 192, "BF16", "BF16", {"lse": True}),
    ([(30, 150)], 2, 4, 256, "BF16", "F16", {}),
    ([(1, 333)], 2, 12, 256, "F32", "F32", {"lse": True}),
    ([(1, 900)], 1, 20, 80, "F32", "F32", {"lse": True, "mask": 0.8}),         # 20 rows
    ([(45, 110), (3, 9)], 2, 2, 80, "F32", "F32", {"lse": True, "window": 64}),
    ([(20, 64)], 1, 8, 128, "F32", "BF16", {"scale": 0.37}),
    ([(9, 4)], 1, 2, 64, "BF16", "BF16", {"lse": True}),                       # fewer tokens than rows: the first see nothing
]
# the number of rows on both sides of each kernel's
ATTN_ROWS = [
    ([(4, 300), (1, 90)], 2, 8, 64, "BF16", "BF16", {"lse": True}),            # 32 rows
    ([(11, 250)], 2, 3, 128, "F16", "F16", {"mask": 0.6}),                     # 33
    ([(2, 600), (2, 2)], 1, 16, 128, "F32", "F32", {"window": 100}),           # 32
    ([(3, 200)], 2, 6, 250, "BF16", "F32", {"lse": True}),                     # 18 wide rows
    ([(16, 400), (5, 5)], 1, 1, 200, "F32", "BF16", {"lse": True}),            # 16 wide rows
    ([(97, 300), (20, 500)], 3, 1, 64, "BF16", "BF16", {"lse": True}),
    ([(96, 96)], 3, 1, 64, "F16", "BF16", {"window": 40}),
    ([(150, 190), (1, 70)], 2, 2, 128, "F32", "F32", {"lse": True, "mask": 0.9}),
    # short caches beside none
    ([(1, 1000), (2, 321), (0, 9), (1, 0)], 2, 8, 128, "BF16", "BF16", {"lse": True}),
    ([(1, 700), (1, 1)], 3, 12, 64, "F32", "F32", {"lse": True, "mask": 0.5}),
    ([(3, 500)], 2, 5, 75, "F16", "F16", {"window": 130}),
    ([(1, 900)], 1, 1, 128, "F32", "F32", {"max_len": 300}),                    # longer than said
]


def attn_case(dev, seqs, heads, group, dim, dt, opts, seed=11, spread=1.0):
    g = np.random.default_rng(seed)
    table, blocks = tables([(l + BLOCK - 1) // BLOCK for _, l in seqs], seed=seed)
    cache = ref.Cache(blocks, heads, dim, seed)
    starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])])
    rows = int(starts[-1]) + 2
    stride = heads * group * dim + 24
    bits = ref.to_bits(g.standard_normal((rows, stride)) * spread, dt)
    q = ref.from_bits(bits, dt)[:, 8:8 + heads * group * dim].reshape(rows, heads * group, dim)
    mask = None
    if opts.get("mask"):
        mask = (g.random((len(seqs), max(l for _, l in seqs))) < opts["mask"]).astype(np.uint8) * 3
    return cache, table, starts, np.array([l for _, l in seqs]), bits, q, rows, stride, mask


def run_attn(dev, cache, table, starts, lengths, bits, q, rows, stride, mask, group, dt, out_dt, opts, most=None, c=None, work=None):
    heads, dim = cache.heads * group, cache.dim
    c = c or upload(dev, cache)
    x = up(dev, bits, dt, [rows, stride])
    mark = ref.to_bits(np.full((rows, heads * dim), 55.0), out_dt)
    out = up(dev, mark, out_dt, [rows, heads * dim])
    lse = up(dev, np.full((rows, heads), 44.0, np.float32), "F32", [rows, heads]) if opts.get("lse") else None
    ops.kv_attention(c, i32(dev, table), ops.Rows(x, 8, stride, rows, heads, dim), i32(dev, starts), i32(dev, lengths),
                     most if most is not None else int(max(np.diff(starts).max(), 1)), out, max_len=opts.get("max_len", 0),
                     window=opts.get("window", 0), mask=up(dev, mask, "U8", list(mask.shape)) if mask is not None else None,
                     scale=opts.get("scale", 0.0), lse=lse, work=work)
    return ref.from_bits(out.to_numpy(), out_dt).reshape(rows, heads, dim), lse.to_numpy() if lse is not None else None


def check_attn(got, lse, want, used, what=""):
    out, wl, tol, ltol = want
    off = np.abs(got[:used].astype(np.float64) - out[:used])
    bad = ~(off <= tol[:used])
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(off / tol[:used]):.3g} of the bound at {np.argwhere(bad)[:3].tolist()}"
    assert (got[used:] == 55.0).all(), f"{what}: rows behind the last sequence were written"
    if lse is not None:
        with np.errstate(invalid="ignore"):
            same = np.isneginf(lse[:used]) & np.isneginf(wl[:used])
            assert (same | (np.abs(lse[:used] - wl[:used]) <= ltol[:used])).all(), f"{what}: lse"
        assert (lse[used:] == 44.0).all()


@pytest.fixture(scope="module")
def dev_cus2():
    """A context that sizes its grids for two compute units: calls of any size then take the tiles of large ones, without parts."""
    import os

    old = os.environ.get("H3S_CUS")
    os.environ["H3S_CUS"] = "2"
    try:
        d = Device.open()
    finally:
        if old is None:
            del os.environ["H3S_CUS"]
        else:
            os.environ["H3S_CUS"] = old
    yield d
    d.close()


@pytest.mark.parametrize("where", ["dev", "dev_cus2"])
@pytest.mark.parametrize("seqs,heads,group,dim,dt,out_dt,opts", ATTN + ATTN_ROWS)
def test_attention(request, where, seqs, heads, group, dim, dt, out_dt, opts):
    dev = request.getfixturevalue(where)
    case = attn_case(dev, seqs, heads, group, dim, dt, opts)
    cache, table, starts, lengths, bits, q, rows, stride, mask = case
    got, lse = run_attn(dev, *case, group, dt, out_dt, opts)
    want = ref.attention(cache, table, starts, lengths, q, group, dt, out_dt, opts.get("scale"), opts.get("window", 0), mask)
    check_attn(got, lse, want, int(starts[-1]), str(seqs))
    # a sequence with no row is asked nothing; max_len only splits the work otherwise
    got2, lse2 = run_attn(dev, *case, group, dt, out_dt, {**opts, "max_len": 1})
    check_attn(got2, lse2, want, int(starts[-1]), f"{seqs} max_len 1")


@pytest.mark.parametrize("spread", [1e-4, 30.0])
@pytest.mark.parametrize("dt", ["BF16", "F16", "F32"])
def test_attention_scores_flat_and_peaked(dev, dt, spread):
    """Scores near zero (a plain mean) and of hundreds (one key wins, probabilities underflow)."""
    seqs, heads, group, dim = [(3, 500), (50, 190)], 2, 4, 128
    case = attn_case(dev, seqs, heads, group, dim, dt, {}, seed=21, spread=spread)
    cache, table, starts, lengths, bits, q, rows, stride, mask = case
    got, lse = run_attn(dev, *case, group, dt, "F32", {"lse": True})
    check_attn(got, lse, ref.attention(cache, table, starts, lengths, q, group, dt, "F32"), int(starts[-1]))


@pytest.mark.parametrize("new", [1, 60])
def test_attention_hidden_tokens_have_no_effect(dev, new):
    """Blocks that are not there, masked blocks whose scales are NaN or infinite, tokens behind the length in the last block, codes in
    the padding: the results are those without them. A row whose mask leaves nothing gets zeros."""
    heads, group, dim, dt = 2, 4, 80, "BF16"
    seqs = [(new, 300), (new, 200), (new, 130)]
    cache, table, starts, lengths, bits, q, rows, stride, _ = attn_case(dev, seqs, heads, group, dim, dt, {}, seed=31)
    mask = np.ones((3, 300), np.uint8)
    mask[0, 64:128] = 0
    cache.s[0, table[0, 1]], cache.s[1, table[0, 1]] = np.nan, np.inf            # block 1 of sequence 0: masked
    table[0, 2] = -1                                                           # block 2 is not there
    table[1, 0] = cache.blocks                                                 # nor this
    mask[2, :] = 0                                                             # nothing left for sequence 2
    cache.s[:, table[2, 0]] = np.nan
    got, lse = run_attn(dev, cache, table, starts, lengths, bits, q, rows, stride, mask, group, dt, "BF16", {"lse": True})
    want = ref.attention(cache, table, starts, lengths, q, group, dt, "BF16", mask=mask)
    check_attn(got, lse, want, int(starts[-1]))
    assert (got[starts[2]:starts[3]] == 0).all() and np.isneginf(lse[starts[2]:starts[3]]).all()
    # what lies behind the sequences' lengths and in the padding changes nothing
    other = ref.Cache(cache.blocks, heads, dim, 31)
    other.s[:] = cache.s
    w = ref.width(dim)
    g = np.random.default_rng(1)
    other.k[..., dim:] = g.integers(-127, 128, other.k[..., dim:].shape)
    other.v[:, :, dim:] = g.integers(-127, 128, other.v[:, :, dim:].shape)
    for b, l in enumerate(lengths):
        if l % BLOCK and 0 <= table[b, l // BLOCK] < cache.blocks:
            other.k[table[b, l // BLOCK], :, l % BLOCK:] = 127
            other.v[table[b, l // BLOCK], :, :, l % BLOCK:] = -127
    assert w > dim
    again, lse2 = run_attn(dev, other, table, starts, lengths, bits, q, rows, stride, mask, group, dt, "BF16", {"lse": True})
    assert np.array_equal(got, again) and np.array_equal(lse, lse2)


def test_attention_nan_in_sight(dev):
    """A visible block with a NaN scale gives NaN to the rows that see it and to no other."""
    heads, group, dim, dt = 2, 2, 64, "BF16"
    cache, table, starts, lengths, bits, q, rows, stride, _ = attn_case(dev, [(1, 200), (1, 200)], heads, group, dim, dt, {}, seed=41)
    cache.s[1, table[1, 1], 0] = np.nan
    got, _ = run_attn(dev, cache, table, starts, lengths, bits, q, rows, stride, None, group, dt, "F32", {})
    assert np.isfinite(got[0]).all() and np.isnan(got[1, :group]).all() and np.isfinite(got[1, group:]).all()


def test_attention_lengths_and_starts_out_of_range(dev):
    """Lengths past the table are cut to it, below zero to none; starts are cut to the rows."""
    heads, group, dim, dt = 1, 4, 64, "BF16"
    cache, table, starts, lengths, bits, q, rows, stride, _ = attn_case(dev, [(2, 128), (2, 128), (2, 128)], heads, group, dim, dt, {}, seed=51)
    wild = np.array([1 << 30, -5, 100])
    got, _ = run_attn(dev, cache, table, starts, wild, bits, q, rows, stride, None, group, dt, "F32", {})
    want = ref.attention(cache, table, starts, np.array([128, 0, 100]), q, group, dt, "F32")
    check_attn(got, None, want, int(starts[-1]))
    got, _ = run_attn(dev, cache, table, np.array([-3, 2, 1 << 29, 1 << 30]), lengths, bits, q, rows, stride, None, group, dt, "F32", {}, most=2)
    first = ref.attention(cache, table[:1], starts[:2], lengths[:1], q, group, dt, "F32")
    assert (np.abs(got[:2] - first[0][:2]) <= first[2][:2]).all()


def test_cache_past_32_bits(dev):
    """Blocks whose codes lie beyond 4 GiB."""
    heads, dim, group = 8, 128, 2
    blocks = 66500                                                              # 66500 * 64 KiB
    c = ops.KvCache.new(dev, blocks, heads, dim)
    seqs = [(100, 150), (1, 90)]
    table = np.array([[66499, 3, 66001], [65999, 66498, -1]], np.int32)
    starts = np.array([0, 150, 240])
    g = np.random.default_rng(6)
    bits = ref.to_bits(g.standard_normal((240, 2 * heads * dim)), "BF16")
    x = up(dev, bits, "BF16", [240, 2 * heads * dim])
    r = [ops.Rows(x, i * heads * dim, 2 * heads * dim, 240, heads, dim) for i in (0, 1)]
    ops.kv_write(c, i32(dev, table), r[0], r[1], i32(dev, starts), i32(dev, [0, 0]), 150)
    # the same in a small pool
    small = ref.Cache(6, heads, dim)
    where = {66499: 0, 3: 1, 66001: 2, 65999: 3, 66498: 4, -1: -1}
    stable = np.vectorize(where.get)(table).astype(np.int32)
    kv = [ref.from_bits(bits, "BF16")[:, i * heads * dim:(i + 1) * heads * dim].reshape(240, heads, dim) for i in (0, 1)]
    small.write(stable, starts, [0, 0], kv)
    ko, vo = new(dev, "F32", [240, heads * dim]), new(dev, "F32", [240, heads * dim])
    ops.kv_read(c, i32(dev, table), i32(dev, starts), i32(dev, [0, 0]), 150, ops.Rows(ko, 0, heads * dim, 240, heads, dim),
                ops.Rows(vo, 0, heads * dim, 240, heads, dim))
    for i, y in enumerate((ko, vo)):
        for b in (0, 1):
            want, _ = small.values(i, stable[b], np.arange(starts[b + 1] - starts[b]))
            assert np.array_equal(y.to_numpy()[starts[b]:starts[b + 1]], want.transpose(1, 0, 2).reshape(-1, heads * dim))
    qs = np.array([0, 100, 101])
    qbits = ref.to_bits(g.standard_normal((103, heads * group * dim + 24)), "BF16")
    q = ref.from_bits(qbits, "BF16")[:, 8:8 + heads * group * dim].reshape(103, heads * group, dim)
    got, _ = run_attn(dev, small, table, qs, np.array([150, 90]), qbits, q, 103, heads * group * dim + 24, None, group, "BF16", "BF16", {}, c=c)
    check_attn(got, None, ref.attention(small, stable, qs, np.array([150, 90]), q, group, "BF16", "BF16"), 101, str(seqs))
    for t in (c.k, c.v):
        t._owner.free()


def test_attention_window_past_every_length(dev):
    """A window of any size is the largest that matters; the work is split as without one."""
    seqs = [(1, 1500), (1, 700)]
    cache, table, starts, lengths, bits, q, rows, stride, _ = attn_case(dev, seqs, 2, 4, 64, "BF16", {}, seed=61)
    c, t, x = upload(dev, cache), i32(dev, table), up(dev, bits, "BF16", [rows, stride])
    r, st, ln = ops.Rows(x, 8, stride, rows, 8, 64), i32(dev, starts), i32(dev, lengths)
    got = []
    for window in (0, 1 << 31, (1 << 63) - 1):
        assert ops.kv_attention_work(c, t, r, st, 1, window=window) == ops.kv_attention_work(c, t, r, st, 1)
        out = new(dev, "F32", [rows, 8 * 64])
        ops.kv_attention(c, t, r, st, ln, 1, out, window=window)
        got.append(out.to_numpy()[:int(starts[-1])])
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_attention_two_contexts_at_once(dev):
    """Two contexts' calls, queued in turn without a wait, each with its own split and its own scratch."""
    other = Device.open()
    made = []
    for d in (dev, other):
        for seed, seqs in ((71, [(1, 1900)]), (72, [(1, 900), (2, 1300)])):
            cache, table, starts, lengths, bits, q, rows, stride, _ = attn_case(d, seqs, 2, 4, 64, "BF16", {}, seed=seed)
            out = up(d, np.full((rows, 8 * 64), 55.0, np.float32), "F32", [rows, 8 * 64])
            args = (upload(d, cache), i32(d, table), ops.Rows(up(d, bits, "BF16", [rows, stride]), 8, stride, rows, 8, 64),
                    i32(d, starts), i32(d, lengths), max(n for n, _ in seqs), out)
            made.append((args, ref.attention(cache, table, starts, lengths, q, 4, "BF16", "F32"), int(starts[-1])))
    for _ in range(3):
        for i in (0, 2, 1, 3):
            ops.kv_attention(*made[i][0])
    for d in (dev, other):
        d.wait()
    for args, want, used in made:
        check_attn(args[6].to_numpy().reshape(-1, 8, 64), None, want, used, str(used))
    del made, args
    other.close()


class Recorded:
    """What `call` queues on the context's stream, recorded into a HIP graph (and not run)."""

    def __init__(self, dev, call):
        import ctypes as C

        self.dev, self.hip, self.C = dev, dev.api.lib, C
        stream, graph, self.exec = C.c_void_p(dev.stream()), C.c_void_p(), C.c_void_p()
        assert self.hip.hipStreamBeginCapture(stream, 2) == 0                      # relaxed
        try:
            call()
        finally:
            rc = self.hip.hipStreamEndCapture(stream, C.byref(graph))
        assert rc == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)) == 0
        assert self.hip.hipGraphDestroy(graph) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exec, self.C.c_void_p(self.dev.stream())) == 0
        self.dev.wait()

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.exec) == 0


def test_attention_workspace_and_graph(dev):
    """The context's scratch, a workspace of the caller's and a recorded call give the same bits; a recorded call without one is
    refused; a replay follows the lengths that are in memory then."""
    heads, group, dim, dt = 1, 8, 128, "BF16"
    cache, table, starts, lengths, bits, q, rows, stride, _ = attn_case(dev, [(1, 2000)], heads, group, dim, dt, {}, seed=61)
    eager, _ = run_attn(dev, cache, table, starts, lengths, bits, q, rows, stride, None, group, dt, "F32", {})
    c, t, x = upload(dev, cache), i32(dev, table), up(dev, bits, dt, [rows, stride])
    st, lt, out = i32(dev, starts), i32(dev, lengths), up(dev, np.zeros((rows, heads * group * dim), np.float32), "F32", [rows, heads * group * dim])
    rq = ops.Rows(x, 8, stride, rows, heads * group, dim)
    size = ops.kv_attention_work(c, t, rq, st, 1)
    assert size > 0
    work, small = new(dev, "U8", [size]), new(dev, "U8", [size - 16])

    def call(w):
        ops.kv_attention(c, t, rq, st, lt, 1, out, work=w)

    call(work)
    assert np.array_equal(out.to_numpy().reshape(eager.shape)[:1], eager[:1])
    with pytest.raises(Error, match="smaller"):
        call(small)

    def record():
        with pytest.raises(Error, match="workspace of its own"):
            call(None)
        call(work)

    g = Recorded(dev, record)
    for length in (2000, 1, 777, 64, 2000):
        lt._owner.write(np.array([length], np.int32))
        out._owner.write(np.zeros(out.elements(), np.float32))
        g.replay()
        want = ref.attention(cache, table, starts, np.array([length]), q, group, dt, "F32")
        assert (np.abs(out.to_numpy().reshape(eager.shape)[:1] - want[0][:1]) <= want[2][:1]).all(), length
        call(None)                                                                # eager work of the context between the replays
    g.close()


def test_a_step_recorded_and_replayed(dev):
    """A whole step of two sequences - 4-bit projections, rotation, cache write, attention, 4-bit output layer - run eagerly and
    as one recorded graph over a growing sequence: the same bits at every step, and each stage within its bounds of the stage
    before it."""
    heads, group, dim, hidden, seqs, steps = 2, 4, 64, 256, 2, 70
    qh = heads * group
    wide = (qh + 2 * heads) * dim
    g = np.random.default_rng(8)
    qkv, _, qc, qsc, qz, qb = linear4_case(dev, 1, hidden, wide, 32, True, "BF16", "F16", True, seed=1)
    proj, _, pc, psc, pz, pb = linear4_case(dev, 1, qh * dim, hidden, 64, False, "BF16", "F16", False, seed=2)
    table = np.array([[3, 0], [1, 4]], np.int32)
    ones = up(dev, np.ones(dim, np.float32), "F32", [dim])
    xb = [ref.to_bits(g.standard_normal((seqs, hidden)), "BF16") for _ in range(steps)]
    angle = (np.arange(steps)[:, None] * 0.02 ** (np.arange(dim // 2) / (dim // 2))).astype(np.float32)
    cs_of = [np.repeat(np.stack([np.cos(a), np.sin(a)], -1)[None], seqs, 0).astype(np.float32) for a in angle]

    def make():
        s = {"cache": upload(dev, ref.Cache(5, heads, dim, 3)), "t": i32(dev, table), "starts": i32(dev, [0, 1, 2]), "past": i32(dev, [0, 40]),
             "len": i32(dev, [1, 41]), "x": new(dev, "BF16", [seqs, hidden]), "rows": new(dev, "BF16", [seqs, wide]),
             "cs": new(dev, "F32", [seqs, dim // 2, 2]), "att": new(dev, "BF16", [seqs, qh * dim]), "y": new(dev, "BF16", [seqs, hidden])}
        s["q"] = ops.Rows(s["rows"], 0, wide, seqs, qh, dim)
        s["k"] = ops.Rows(s["rows"], qh * dim, wide, seqs, heads, dim)
        s["v"] = ops.Rows(s["rows"], (qh + heads) * dim, wide, seqs, heads, dim)
        s["work"] = new(dev, "U8", [max(16, ops.kv_attention_work(s["cache"], s["t"], s["q"], s["starts"], 1))])
        return s

    def step(s):
        qkv.forward(s["x"], s["rows"])
        ops.rms_rope(s["q"], ones, 1e-6, s["cs"], dim)
        ops.rms_rope(s["k"], ones, 1e-6, s["cs"], dim)
        ops.kv_write(s["cache"], s["t"], s["k"], s["v"], s["starts"], s["past"], 1)
        ops.kv_attention(s["cache"], s["t"], s["q"], s["starts"], s["len"], 1, s["att"], work=s["work"])
        proj.forward(s["att"], s["y"])

    def feed(s, n):
        s["x"]._owner.write(xb[n])
        s["cs"]._owner.write(cs_of[n])
        s["past"]._owner.write(np.array([n, 40 + n], np.int32))
        s["len"]._owner.write(np.array([n + 1, 41 + n], np.int32))

    eager, replayed, mirror = make(), make(), ref.Cache(5, heads, dim, 3)
    step(make())                                                                  # (a first call of every kernel)
    graph = Recorded(dev, lambda: step(replayed))
    for n in range(steps):
        feed(eager, n)
        step(eager)
        feed(replayed, n)
        graph.replay()
        for name in ("rows", "att", "y"):
            assert np.array_equal(eager[name].to_numpy(), replayed[name].to_numpy()), (n, name)
        rows = ref.from_bits(eager["rows"].to_numpy(), "BF16")
        kv = [rows[:, at * dim:(at + heads) * dim].reshape(seqs, heads, dim) for at in (qh, qh + heads)]
        mirror.write(table, [0, 1, 2], [n, 40 + n], kv)
        want, _, tol, _ = ref.attention(mirror, table, [0, 1, 2], [n + 1, 41 + n], rows[:, :qh * dim].reshape(seqs, qh, dim), group, "BF16", "BF16")
        att = ref.from_bits(eager["att"].to_numpy(), "BF16")
        assert (np.abs(att.reshape(want.shape) - want) <= tol).all(), n
        y, ytol = ref.linear4(att, pc, psc, pz, pb, "BF16")
        assert (np.abs(ref.from_bits(eager["y"].to_numpy(), "BF16") - y) <= ytol).all(), n
        v, vtol = ref.linear4(ref.from_bits(xb[n], "BF16"), qc, qsc, qz, qb, "BF16")
        at = (qh + heads) * dim                                                   # (q and k are normalized and rotated in place)
        assert (np.abs(rows[:, at:] - v[:, at:]) <= vtol[:, at:]).all(), n
    compare_cache(eager["cache"], mirror)
    graph.close()


def test_attention_kernels_taken(dev):
    """Which kernel and how many blocks of threads a call takes: few rows share the cache blocks among four wavefronts, many have
    wavefronts of their own, long caches and few rows are split and joined."""
    def names(seqs, heads, group, dim, dt, opts):
        case = attn_case(dev, seqs, heads, group, dim, dt, opts)
        cache, table, starts, lengths, bits, q, rows, stride, mask = case
        c, t, x = upload(dev, cache), i32(dev, table), up(dev, bits, dt, [rows, stride])
        out, st, lt = new(dev, "F32", [rows, heads * group * dim]), i32(dev, starts), i32(dev, lengths)
        rq = ops.Rows(x, 8, stride, rows, heads * group, dim)
        work = new(dev, "U8", [max(ops.kv_attention_work(c, t, rq, st, max(n for n, _ in seqs)), 16)])
        return launches(dev, lambda: ops.kv_attention(c, t, rq, st, lt, max(n for n, _ in seqs), out, work=work))

    few = names([(1, 200)] * 3, 2, 8, 128, "BF16", {})
    assert len(few) == 1 and few[0][0].startswith("kv_attn_kernel<2, 1, false") and few[0][1] == 6, few
    split = names([(1, 2000)], 1, 8, 128, "F32", {})
    assert len(split) == 2 and split[0][0].startswith("kv_attn_kernel<2, 1, true") and split[0][1] >= 4, split
    some = names([(100, 100)], 2, 4, 64, "F16", {})
    assert len(some) == 1 and some[0][0].startswith("kv_attn_rows_kernel<1, 1, false") and some[0][1] == 14, some
    shared = names([(4, 100)] * 3, 2, 8, 128, "BF16", {})
    assert len(shared) == 1 and shared[0][0].startswith("kv_attn_kernel<2, 2, false") and shared[0][1] == 6, shared
    own = names([(5, 100)] * 3, 2, 8, 128, "BF16", {})
    assert len(own) == 1 and own[0][0].startswith("kv_attn_rows_kernel<2, 1, false") and own[0][1] == 6, own
    wide = names([(4, 100)] * 3, 2, 8, 256, "F32", {})
    assert len(wide) == 1 and wide[0][0].startswith("kv_attn_rows_kernel<4, 1, true") and wide[0][1] == 6, wide
    halves = names([(130, 130)], 16, 16, 64, "F32", {})
    assert len(halves) == 1 and halves[0][0].startswith("kv_attn_rows_kernel<1, 1, true") and halves[0][1] == 33 * 16, halves
    many = names([(130, 130)], 16, 16, 64, "F16", {})
    assert len(many) == 1 and many[0][0].startswith("kv_attn_rows_kernel<1, 2, false") and many[0][1] == 17 * 16, many


# ---- linear4 -------------------------------------------------------------------------------------------------------------------

LINEAR4 = [
    # M, K, N, group, minima, type, out type, scale type, bias
    (1, 128, 16, 32, False, "BF16", "BF16", "F16", False),
    (1, 5376, 100, 32, True, "BF16", "BF16", "F16", True),
    (4, 1024, 33, 64, False, "F16", "F16", "F32", True),
    (5, 1024, 70, 128, True, "F16", "F32", "BF16", False),
    (16, 896, 48, 32, False, "BF16", "F32", "F16", True),               # 28 groups
    (3, 160, 20, 32, True, "BF16", "F32", "F16", True),                 # a row that ends inside a run of 128; odd groups
    (7, 288, 50, 96, True, "F16", "F16", "F16", False),                 # groups that a run of 128 straddles
    (2, 32, 5, 32, False, "F32", "F32", "F32", True),
    (17, 512, 40, 256, False, "F32", "F32", "F16", True),
    (40, 1152, 64, 192, True, "BF16", "BF16", "F32", True),
    (65, 768, 31, 64, True, "F32", "BF16", "BF16", True),
    (130, 1024, 96, 128, False, "BF16", "BF16", "F16", False),
    (300, 640, 130, 32, True, "BF16", "F32", "F16", True),
    (64, 256, 1, 32, False, "F16", "F32", "F16", True),
]
# rows of weights in several chunks or steps a wavefront, and more columns than the blocks of a grid take at once
LINEAR4_LONG = [
    (1, 14336, 40, 64, True, "BF16", "BF16", "F16", True),
    (1, 8192, 40, 128, False, "F32", "F32", "F32", True),
    (1, 20000 * 32, 5, 32, True, "BF16", "F32", "F16", False),
    (1, 512, 20011, 128, False, "F16", "F32", "F16", True),
    (2, 6400, 33, 32, True, "F16", "F16", "F16", True),
    (2, 544, 9001, 32, True, "F32", "F32", "F32", False),
    (4, 5632, 18, 256, False, "BF16", "BF16", "BF16", True),
    (3, 8192, 50, 64, True, "BF16", "F32", "F16", True),
    (9, 14336, 35, 32, True, "BF16", "BF16", "F16", True),
    (16, 512, 20011, 64, False, "BF16", "BF16", "F16", True),
    (7, 1 << 20, 3, 128, False, "F16", "F32", "F32", True),
    (12, 6176, 100, 32, True, "F32", "F32", "F16", True),
    (33, 14336, 150, 64, True, "BF16", "BF16", "F16", True),
    (70, 6240, 140, 96, False, "F16", "F32", "F32", True),
    (20, 5376, 5376, 32, True, "BF16", "BF16", "F16", True),                    # 42 blocks of 128 columns: in 168 of 32
    (50, 1568, 4100, 32, True, "F16", "F16", "F16", True),                      # 33 blocks: in 66 of 64
    (32, 2048, 8200, 128, False, "BF16", "BF16", "F32", False),                 # 65: in 130 of 64
    (100, 640, 17000, 64, True, "BF16", "BF16", "F16", True),                   # 266: as they are
    (33, 1024, 5000, 64, False, "F32", "F32", "F16", True),
    (27, 5376, 5300, 32, True, "F32", "F32", "F16", True),                      # in 166 blocks of 16 rows x 64 columns
]


def linear4_case(dev, M, K, N, group, mins, dt, scale_dt, bias, seed=5):
    g = np.random.default_rng(seed + M + K + N)
    xb = ref.to_bits(g.standard_normal((M, K)) * np.exp(g.normal(0, 1, (M, 1))), dt)
    codes = g.integers(0, 256, (N, K // 2), dtype=np.uint8)
    sb = ref.to_bits(np.exp(g.normal(-4, 0.5, (N, K // group))) * np.where(g.random((N, K // group)) < 0.1, -1, 1), scale_dt)
    mb = ref.to_bits(g.standard_normal((N, K // group)) * 0.1, scale_dt) if mins else None
    b = g.standard_normal(N).astype(np.float32) if bias else None
    layer = ops.Int4Linear(up(dev, codes, "U8", [N, K // 2]), up(dev, sb, scale_dt, [N, K // group]),
                           up(dev, mb, scale_dt, [N, K // group]) if mins else None, up(dev, b, "F32", [N]) if bias else None)
    return layer, xb, codes, ref.from_bits(sb, scale_dt), ref.from_bits(mb, scale_dt) if mins else None, b


@pytest.mark.parametrize("M,K,N,group,mins,dt,out_dt,scale_dt,bias", LINEAR4 + LINEAR4_LONG)
def test_linear4(dev, M, K, N, group, mins, dt, out_dt, scale_dt, bias):
    layer, xb, codes, s, z, b = linear4_case(dev, M, K, N, group, mins, dt, scale_dt, bias)
    mark = ref.to_bits(np.full((M + 1, N), 9.0), out_dt)
    whole = up(dev, mark, out_dt, [M + 1, N])
    out = Tensor(whole.dtype, [M, N], whole.ptr(), whole, dev)
    layer.forward(up(dev, xb, dt, [M, K]), out)
    got = ref.from_bits(whole.to_numpy(), out_dt).astype(np.float64)
    want, tol = ref.linear4(ref.from_bits(xb, dt), codes, s, z, b, out_dt)
    off = np.abs(got[:M] - want)
    assert (off <= tol).all(), f"worst {np.max(off / tol):.3g} of the bound at {np.argwhere(off > tol)[:3].tolist()}"
    assert (got[M] == 9.0).all()


@pytest.mark.parametrize("M", [1, 9, 33])
@pytest.mark.parametrize("at", ["scale", "mins"])
def test_linear4_scales_off_a_boundary(dev, M, at):
    """Scales or minima that start on a 2-byte boundary only."""
    K, N, group = 512, 40, 32
    layer, xb, codes, s, z, b = linear4_case(dev, M, K, N, group, True, "BF16", "F16", True, seed=9)
    bits = ref.to_bits(s if at == "scale" else z, "F16").ravel()
    whole = up(dev, np.concatenate([bits[:1], bits]), "F16", [bits.size + 1])
    moved = Tensor(whole.dtype, [N, K // group], whole.ptr() + 2, whole, dev)
    if at == "scale":
        layer.scale = moved
    else:
        layer.mins = moved
    out = new(dev, "F32", [M, N])
    layer.forward(up(dev, xb, "BF16", [M, K]), out)
    want, tol = ref.linear4(ref.from_bits(xb, "BF16"), codes, s, z, b, "F32")
    assert (np.abs(out.to_numpy() - want) <= tol).all()


def test_linear4_odd_values(dev):
    """An infinity or NaN in a row of x stays in that row; in a group's scale, in that column."""
    M, K, N = 6, 256, 24
    layer, xb, codes, s, z, b = linear4_case(dev, M, K, N, 32, False, "F32", "F32", True)
    x = xb.copy()
    x[2, 100], x[4, 3] = np.inf, np.nan
    s2 = s.copy()
    s2[7, 1] = np.nan
    layer.scale = up(dev, s2, "F32", list(s.shape))
    out = new(dev, "F32", [M, N])
    layer.forward(up(dev, x, "F32", [M, K]), out)
    got = out.to_numpy()
    want, tol = ref.linear4(xb, codes, s, z, b, "F32")
    rows, cols = [0, 1, 3, 5], [c for c in range(N) if c != 7]
    assert (np.abs(got - want) <= tol)[np.ix_(rows, cols)].all()
    assert not np.isfinite(got[[2, 4]]).any() and np.isnan(got[rows, 7]).all()
