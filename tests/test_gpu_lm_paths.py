"""The cache's reads and writes at their edges, and the attention's paths by mask alignment and head size."""
import numpy as np
import pytest

import lm_reference as ref
from helpers import launches, new, up
from test_gpu_lm import attn_case, check_attn, compare_cache, i32, tables, upload

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import Tensor, ops  # noqa: E402

BLOCK = ref.BLOCK


@pytest.mark.parametrize("wide", [0, 16, -16, 3])
@pytest.mark.parametrize("apart", [0, 1, 8])
@pytest.mark.parametrize("seqs,heads,group,dim,dt", [
    ([(1, 400), (2, 64), (1, 1)], 2, 4, 128, "BF16"),
    ([(1, 1300)], 1, 8, 64, "F16"),
    ([(70, 400), (9, 50)], 2, 4, 80, "BF16"),
    ([(40, 333)], 1, 4, 128, "F32"),
])
def test_attention_masks_by_width_and_place(dev, seqs, heads, group, dim, dt, wide, apart):
    """Masks as wide as 16-byte pieces and not, wider and narrower than the lengths, from a 16-byte boundary on and off it."""
    case = attn_case(dev, seqs, heads, group, dim, dt, {}, seed=101)
    cache, table, starts, lengths, bits, q, rows, stride, _ = case
    g = np.random.default_rng(102)
    n = (int(lengths.max()) + 15) // 16 * 16 + wide
    mask = (g.random((len(seqs), n)) < 0.7).astype(np.uint8) * g.integers(1, 256, (len(seqs), n)).astype(np.uint8)
    if n > 64:
        mask[0, :64] = 0                                                          # a whole block
    whole = up(dev, np.concatenate([np.full(apart, 255, np.uint8), mask.ravel()]), "U8", [apart + mask.size])
    held = Tensor(whole.dtype, [len(seqs), n], whole.ptr() + apart, whole, dev)
    mark = ref.to_bits(np.full((rows, heads * group * dim), 55.0), "F32")
    out, lse = up(dev, mark, "F32", list(mark.shape)), up(dev, np.full((rows, heads * group), 44.0, np.float32), "F32", [rows, heads * group])
    x = up(dev, bits, dt, [rows, stride])
    ops.kv_attention(upload(dev, cache), i32(dev, table), ops.Rows(x, 8, stride, rows, heads * group, dim), i32(dev, starts), i32(dev, lengths),
                     int(np.diff(starts).max()), out, mask=held, lse=lse)
    want = ref.attention(cache, table, starts, lengths, q, group, dt, "F32", mask=mask)
    check_attn(out.to_numpy().reshape(rows, heads * group, dim), lse.to_numpy(), want, int(starts[-1]), f"mask {n} wide, {apart} off")


def test_attention_heads_of_129_to_192(dev):
    """Few and many rows of both kinds of queries, each through the kernel that the head size and the rows choose."""
    for seqs, heads, group, dim, dt, kernel in [
        ([(1, 300), (2, 70)], 2, 4, 192, "F32", "kv_attn_kernel<3, 1, true"),
        ([(1, 1500)], 1, 8, 130, "F32", "kv_attn_kernel<3, 1, true"),
        ([(1, 1500)], 1, 8, 160, "BF16", "kv_attn_kernel<3, 1, false"),
        ([(30, 150), (7, 7)], 2, 4, 192, "BF16", "kv_attn_rows_kernel<3, 1, false"),
        ([(90, 400)], 2, 3, 160, "F16", "kv_attn_rows_kernel<3, 1, false"),
        ([(45, 200), (3, 300)], 2, 2, 144, "F32", "kv_attn_rows_kernel<3, 1, true"),
        ([(130, 130)], 16, 16, 176, "BF16", "kv_attn_rows_kernel<3, 2, false"),
    ]:
        case = attn_case(dev, seqs, heads, group, dim, dt, {}, seed=103)
        cache, table, starts, lengths, bits, q, rows, stride, _ = case
        c, t, x = upload(dev, cache), i32(dev, table), up(dev, bits, dt, [rows, stride])
        out, lse = new(dev, "F32", [rows, heads * group * dim]), new(dev, "F32", [rows, heads * group])
        rq, st, lt, most = ops.Rows(x, 8, stride, rows, heads * group, dim), i32(dev, starts), i32(dev, lengths), int(np.diff(starts).max())
        work = new(dev, "U8", [max(ops.kv_attention_work(c, t, rq, st, most), 16)])
        ran = launches(dev, lambda: ops.kv_attention(c, t, rq, st, lt, most, out, lse=lse, work=work))
        assert ran[0][0].startswith(kernel), (seqs, dim, ran)
        used = int(starts[-1])
        got, gl = out.to_numpy().reshape(rows, heads * group, dim), lse.to_numpy()
        if heads * group > 64:                                                     # (a few rows of the many)
            picks = [0, 1, 63, 64, used - 1]
            tb, st2, ln2 = np.repeat(table, len(picks), 0), np.arange(len(picks) + 1), lengths[0] - used + 1 + np.array(picks)
            want = ref.attention(cache, tb, st2, ln2, q[picks], group, dt, "F32")
            check_attn(got[picks], gl[picks], want, len(picks), str((seqs, dim, dt)))
        else:
            want = ref.attention(cache, table, starts, lengths, q, group, dt, "F32")
            off = np.abs(got[:used] - want[0][:used])
            assert (off <= want[2][:used]).all(), (seqs, dim, dt, np.nanmax(off / want[2][:used]))
            assert (np.abs(gl[:used] - want[1][:used]) <= want[3][:used]).all()


def test_write_starts_out_of_order_and_range(dev):
    """Starts that run back, below zero and past the rows are cut to the rows; what no sequence then has is not touched."""
    heads, dim, rows = 2, 64, 40
    table, blocks = tables([3] * 6, seed=104)
    cache = ref.Cache(blocks, heads, dim, 104)
    g = np.random.default_rng(104)
    val = g.standard_normal((rows, 2 * heads * dim)).astype(np.float32)
    wild = np.array([-9, 4, 2, 11, 1 << 30, -(1 << 31), 38])                        # rows 0 .. 4, none, 2 .. 11, 11 .. 40, none, 0 .. 38
    past = np.array([60, 5, 0, 70, 9, 150])
    cut = [(0, 4), (4, 4), (2, 11), (11, 40), (40, 40), (0, 38)]
    c = upload(dev, cache)
    x = up(dev, val, "F32", [rows, 2 * heads * dim])
    r = [ops.Rows(x, i * heads * dim, 2 * heads * dim, rows, heads, dim) for i in (0, 1)]
    ops.kv_write(c, i32(dev, table), r[0], r[1], i32(dev, wild), i32(dev, past), rows)
    for b, (lo, hi) in enumerate(cut):
        kv = [val[lo:hi, i * heads * dim:(i + 1) * heads * dim].reshape(hi - lo, heads, dim) for i in (0, 1)]
        if hi > lo:
            cache.write(table[b:b + 1], [0, hi - lo], past[b:b + 1], kv)
    compare_cache(c, cache)


@pytest.mark.parametrize("dt", ["F32", "BF16", "F16"])
def test_read_where_nothing_is(dev, dt):
    """Blocks that are not there and tokens past the table's end read as zeros, a first token below 0 counts as 0, rows of no sequence stay."""
    heads, dim, width = 2, 100, 3
    g = np.random.default_rng(105)
    table = np.array([[0, -1, 1], [2, 3, 7], [4, 5, 6], [1 << 30, -(1 << 31), 0]], np.int32)
    cache = ref.Cache(7, heads, dim, 105)
    first = np.array([-5, 100, 190, 0])
    counts = [150, 80, 300, 100]                                                     # the second ends in a block past the pool, the third past the table
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows, stride = int(starts[-1]) + 4, heads * dim + 4
    mark = ref.to_bits(np.full((2 * rows, stride), 77.0), dt)
    y = up(dev, mark, dt, [2 * rows, stride])
    o = [ops.Rows(y, i * rows * stride, stride, rows, heads, dim) for i in (0, 1)]
    ops.kv_read(upload(dev, cache), i32(dev, table), i32(dev, starts), i32(dev, first), max(counts), o[0], o[1])
    want = mark.copy()
    for b in range(4):
        at = max(first[b], 0) + np.arange(counts[b])
        for i in (0, 1):
            val, there = cache.values(i, table[b], at)
            assert not there.all()
            want[i * rows + starts[b]:i * rows + starts[b + 1], :heads * dim] = ref.to_bits(val.transpose(1, 0, 2).reshape(-1, heads * dim), dt)
    assert np.array_equal(y.to_numpy(), want)


def test_a_table_of_no_blocks(dev):
    """No cache block anywhere: writes do nothing, reads and attention give zeros."""
    heads, dim = 2, 64
    cache = ref.Cache(2, heads, dim, 106)
    c = upload(dev, cache)
    table, starts, past = new(dev, "I32", [2, 0]), i32(dev, [0, 1, 4]), i32(dev, [0, 90])
    x = up(dev, np.ones((4, 2 * heads * dim), np.float32), "F32", [4, 2 * heads * dim])
    r = [ops.Rows(x, i * heads * dim, 2 * heads * dim, 4, heads, dim) for i in (0, 1)]
    ops.kv_write(c, table, r[0], r[1], starts, past, 3)
    compare_cache(c, cache)
    out, lse = up(dev, np.ones((4, heads * dim), np.float32), "F32", [4, heads * dim]), new(dev, "F32", [4, heads])
    ops.kv_attention(c, table, r[0], starts, past, 3, out, lse=lse)
    assert (out.to_numpy() == 0).all() and np.isneginf(lse.to_numpy()).all()
    ops.kv_read(c, table, starts, past, 3, r[0], r[1])
    assert (x.to_numpy() == 0).all()
