"""Attention over the key/value cache behind a window with first tokens that stay visible, and over tokens that groups of sequences share
(include/h3lm.h, kv_attention_spans), against its restatement in numpy (spans_reference.py)."""
import os

import numpy as np
import pytest

import lm_reference as lm
import spans_reference as ref
from helpers import launches, new, up
from test_gpu_lm import Recorded, check_attn, i32, tables, upload

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import Device, Error, ops  # noqa: E402

BLOCK = lm.BLOCK


def context(cus):
    """A context that sizes its grids for so many compute units: shared tokens are a launch of their own from fewer bytes on."""
    old = os.environ.get("H3S_CUS")
    os.environ["H3S_CUS"] = str(cus)
    try:
        return Device.open()
    finally:
        if old is None:
            del os.environ["H3S_CUS"]
        else:
            os.environ["H3S_CUS"] = old


@pytest.fixture(scope="module")
def dev2():
    d = context(2)
    yield d
    d.close()


@pytest.fixture(scope="module")
def dev16():
    d = context(16)
    yield d
    d.close()


class Case:
    """seqs: (new tokens, tokens in the cache after them). groups: (first sequence, sequence behind the last, shared tokens); the shared
    blocks stand in the first sequence's row of the table only, the others' rows there name blocks that are not."""

    def __init__(self, dev, seqs, heads, group, dim, dt, groups=(), seed=21, mask=None):
        g = np.random.default_rng(seed)
        self.table, blocks = tables([(n + BLOCK - 1) // BLOCK for _, n in seqs], seed=seed)
        self.cache = lm.Cache(blocks, heads, dim, seed)
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int64)
        self.lengths = np.array([n for _, n in seqs])
        self.rows, self.stride = int(self.starts[-1]) + 2, heads * group * dim + 24
        self.bits = lm.to_bits(g.standard_normal((self.rows, self.stride)), dt)
        self.q = lm.from_bits(self.bits, dt)[:, 8:8 + heads * group * dim].reshape(self.rows, heads * group, dim)
        self.mask = None if mask is None else (g.random((len(seqs), int(self.lengths.max()))) < mask).astype(np.uint8)
        self.dev, self.heads, self.group, self.dim, self.dt = dev, heads, group, dim, dt
        self.first, self.tokens = [], []
        for a, e, n in groups:
            assert not self.first or self.first[-1] == a
            self.first = self.first or [a]
            self.first.append(e)
            self.tokens.append(n)
            for b in range(a + 1, e):
                self.table[b, :max(n, 0) // BLOCK] = (1 << 30) + b
        self.most = int(max(np.diff(self.starts).max(), 1))

    def upload(self, dev=None):
        dev = dev or self.dev
        x = up(dev, self.bits, self.dt, [self.rows, self.stride])
        shared = ops.KvShared(i32(dev, self.first), i32(dev, self.tokens), max(max(self.tokens), 0)) if self.tokens else None
        mask = up(dev, self.mask, "U8", list(self.mask.shape)) if self.mask is not None else None
        return (upload(dev, self.cache), i32(dev, self.table), ops.Rows(x, 8, self.stride, self.rows, self.heads * self.group, self.dim),
                i32(dev, self.starts), i32(dev, self.lengths), self.most), shared, mask

    def run(self, out_dt="F32", window=0, sinks=0, scale=0.0, max_len=0, dev=None):
        dev = dev or self.dev
        args, shared, mask = self.upload(dev)
        wide = self.heads * self.group
        out = up(dev, lm.to_bits(np.full((self.rows, wide * self.dim), 55.0), out_dt), out_dt, [self.rows, wide * self.dim])
        lse = up(dev, np.full((self.rows, wide), 44.0, np.float32), "F32", [self.rows, wide])
        ops.kv_attention(*args, out, window=window, sinks=sinks, shared=shared, mask=mask, scale=scale, max_len=max_len, lse=lse)
        return lm.from_bits(out.to_numpy(), out_dt).reshape(self.rows, wide, self.dim), lse.to_numpy()

    def want(self, out_dt="F32", window=0, sinks=0, scale=None):
        return ref.attention(self.cache, self.table, self.starts, self.lengths, self.q, self.group, self.dt, out_dt, scale, window, sinks,
                             self.mask, self.first, self.tokens)

    def check(self, got, want, what=""):
        check_attn(*got, want, int(self.starts[-1]), what)


SINKS = [
    # (new, length) of each sequence, heads, group, dim, type, window, sinks
    ([(1, 300)], 2, 8, 128, "BF16", 64, 4),
    ([(1, 700), (1, 5), (2, 64), (0, 9), (1, 65)], 2, 4, 64, "F16", 100, 1),
    ([(1, 500), (3, 400)], 1, 8, 80, "F32", 33, 70),
    ([(1, 450)], 2, 2, 256, "BF16", 64, 64),
    ([(70, 333)], 2, 4, 128, "BF16", 50, 16),
    ([(40, 400), (1, 300), (90, 90)], 1, 8, 64, "F32", 128, 130),
    ([(130, 500)], 1, 7, 96, "F16", 1, 3),
    ([(33, 200)], 2, 4, 192, "BF16", 20, 200),
    ([(60, 250)], 1, 4, 256, "F32", 90, 5),
    ([(2, 260)], 3, 3, 33, "BF16", 10, 1 << 40),
    ([(2, 260), (1, 70)], 1, 40, 64, "F16", 50, 7),
]


@pytest.mark.parametrize("seqs,heads,group,dim,dt,window,sinks", SINKS)
def test_first_tokens_behind_a_window(dev, seqs, heads, group, dim, dt, window, sinks):
    case = Case(dev, seqs, heads, group, dim, dt)
    for out_dt in ("F32", dt if dt != "F32" else "F16"):
        case.check(case.run(out_dt, window, sinks), case.want(out_dt, window, sinks), out_dt)
    masked = Case(dev, seqs, heads, group, dim, dt, mask=0.5)
    masked.check(masked.run("F32", window, sinks, scale=0.2), masked.want("F32", window, sinks, scale=np.float32(0.2)), "mask")


def test_blocks_that_no_row_sees_are_not_needed(dev):
    """The blocks between the first tokens and the window are taken out of the table: the same bits."""
    for seqs, window, sinks in (([(1, 900), (1, 333)], 130, 4), ([(40, 900)], 70, 66)):
        case = Case(dev, seqs, 2, 4, 128, "BF16")
        want = case.run("F32", window, sinks)
        for b, (n, length) in enumerate(seqs):
            case.table[b, (sinks + BLOCK - 1) // BLOCK:max(length - n + 1 - window, 0) // BLOCK] = -1
        got = case.run("F32", window, sinks)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        case.check(got, case.want("F32", window, sinks))


SHARED = [
    # sequences, (first, behind, shared tokens) of the groups, heads, group, dim, type
    ([(1, 200), (1, 150), (1, 129)], [(0, 3, 128)], 2, 8, 128, "BF16"),
    ([(1, 900), (1, 700), (1, 650), (1, 1000)], [(0, 4, 640)], 2, 2, 64, "F16"),
    ([(1, 300)] * 9 + [(1, 90), (2, 400)], [(0, 4, 256), (4, 4, 64), (4, 9, 130)], 1, 4, 80, "F32"),
    ([(1, 40), (1, 500), (1, 300), (1, 77)], [(1, 3, 191)], 2, 4, 96, "BF16"),
    ([(2, 330), (0, 320), (5, 400), (1, 321)], [(0, 4, 320)], 2, 4, 128, "F32"),
    ([(30, 330), (1, 320), (70, 400)], [(0, 3, 250)], 1, 8, 128, "BF16"),
    ([(50, 350), (50, 360)], [(0, 2, 256)], 2, 4, 64, "F16"),
    ([(17, 350), (20, 360), (3, 300), (1, 300)], [(0, 2, 256), (2, 4, 128)], 1, 4, 256, "F32"),
    ([(9, 200), (12, 190)], [(0, 2, 128)], 2, 3, 192, "BF16"),
    ([(1, 130)] * 70, [(b, b + 1, 64) for b in range(70)], 1, 1, 64, "BF16"),
    ([(1, 200), (1, 200)], [(0, 2, 1 << 30)], 1, 4, 64, "F32"),
    ([(1, 200), (1, 200)], [(0, 2, -5)], 1, 4, 64, "F32"),
    ([(1, 64), (1, 100), (3, 20)], [(0, 3, 128)], 1, 4, 64, "BF16"),
    ([(1, 300), (3, 200), (1, 256)], [(0, 3, 128)], 1, 48, 64, "BF16"),
    ([(1, 300), (2, 200)], [(0, 2, 128)], 1, 17, 200, "F16"),
]


@pytest.mark.parametrize("seqs,groups,heads,group,dim,dt", SHARED)
@pytest.mark.parametrize("apart", [False, True])
def test_shared_tokens(dev, dev2, seqs, groups, heads, group, dim, dt, apart):
    """Through a launch of their own and not."""
    dev = dev2 if apart else dev
    case = Case(dev, seqs, heads, group, dim, dt, groups)
    for out_dt in ("F32", dt if dt != "F32" else "BF16"):
        case.check(case.run(out_dt), case.want(out_dt), out_dt)
    case.check(case.run(max_len=1, scale=0.3), case.want(scale=np.float32(0.3)), "scale")
    case.check(case.run(window=90, sinks=20), case.want(window=90, sinks=20), "window")
    masked = Case(dev, seqs, heads, group, dim, dt, groups, mask=0.4)
    masked.check(masked.run(), masked.want(), "mask")
    masked.check(masked.run(window=100, sinks=3), masked.want(window=100, sinks=3), "mask, window")


@pytest.mark.parametrize("seqs,groups,dim,dt", [
    ([(1, 2100), (1, 1900), (2, 1500)], [(0, 3, 1000)], 256, "BF16"),
    ([(30, 1100), (1, 1900), (2, 1500)], [(0, 3, 960)], 128, "F32"),
])
def test_shared_tokens_in_parts(dev16, seqs, groups, dim, dt):
    """Both the shared tokens and the sequences' own in several parts, which a launch of its own joins."""
    case = Case(dev16, seqs, 4, 2, dim, dt, groups)
    args, shared, _ = case.upload()
    out = new(dev16, "F32", [case.rows, 8 * dim])
    work = new(dev16, "U8", [ops.kv_attention_work(*args[:4], case.most, shared=shared)])
    ran = [name.split("<")[0] for name, _, _ in launches(dev16, lambda: ops.kv_attention(*args, out, shared=shared, work=work))]
    assert "kv_join_kernel" in ran, ran
    case.check(case.run(), case.want())
    case.check(case.run(window=700, sinks=100), case.want(window=700, sinks=100), "window")


@pytest.mark.parametrize("apart", [False, True])
def test_shared_blocks_that_are_not_there(dev, dev2, apart):
    dev = dev2 if apart else dev
    case = Case(dev, [(1, 600), (1, 500), (40, 480)], 2, 4, 64, "BF16", [(0, 3, 448)])
    case.table[0, [1, 2, 6]] = [-1, 1 << 29, -(1 << 31)]
    case.check(case.run(), case.want())
    case.table[0, :7] = -1
    case.check(case.run(), case.want(), "none")
    case.table[:] = -1
    got = case.run()
    assert (got[0][:42] == 0).all() and np.isneginf(got[1][:42]).all()


@pytest.mark.parametrize("apart", [False, True])
def test_infinite_scales_of_shared_blocks(dev, dev2, apart):
    """A shared block whose scale is NaN, hidden by the mask or by the window, has no effect; seen, it makes its rows NaN."""
    dev = dev2 if apart else dev
    for seqs in ([(1, 300), (1, 260)], [(50, 300), (20, 260)]):
        case = Case(dev, seqs, 1, 4, 64, "BF16", [(0, 2, 192)])
        case.cache.s[:, case.table[0, 0]] = np.nan
        case.mask = np.ones((2, 300), np.uint8)
        case.mask[:, :64] = 0
        case.check(case.run(), case.want(), "mask")
        case.mask = None
        case.check(case.run(window=60, sinks=0), case.want(window=60, sinks=0), "window")
        assert np.isnan(case.run()[0][:int(case.starts[-1])]).all()


@pytest.mark.parametrize("apart", [False, True])
def test_groups_out_of_order_and_range(dev, dev2, apart):
    """Firsts that run back, below zero or past the sequences: nothing outside the buffers is touched, sequences in no group are right."""
    dev = dev2 if apart else dev
    for first in ([-5, 2, 1, 9], [3, 1, 4, 2], [1 << 30, -(1 << 31), 5, 0], [0, 0, 0, 0]):
        case = Case(dev, [(1, 200), (2, 300), (1, 150), (1, 90)], 1, 4, 64, "F32")
        args, _, _ = case.upload()
        out = up(dev, np.full((case.rows, 256), 55.0, np.float32), "F32", [case.rows, 256])
        ops.kv_attention(*args, out, shared=ops.KvShared(i32(dev, first), i32(dev, [64, 64, 64]), 64))
        got = out.to_numpy()
        assert (got[int(case.starts[-1]):] == 55.0).all()
        if first == [0, 0, 0, 0]:
            want = case.want()
            assert (np.abs(got.reshape(case.rows, 4, 64)[:5] - want[0][:5]) <= want[2][:5]).all()


def test_without_first_tokens_or_groups_it_is_kv_attention(dev):
    """First tokens without a window, and no groups, are kv_attention, bit for bit. Behind a window past everything they see the same in parts of
    their own choice, whose sums may differ in their order: held to the bounds."""
    case = Case(dev, [(1, 200), (40, 300)], 2, 4, 64, "BF16")
    args, _, _ = case.upload()
    outs = [new(dev, "F32", [case.rows, 512]) for _ in range(3)]
    ops.kv_attention(*args, outs[0])
    ops.kv_attention(*args, outs[1], sinks=9)                                       # (all is visible without a window)
    ops.kv_attention(*args, outs[2], shared=ops.KvShared(i32(dev, [0]), new(dev, "I32", [0])))
    used = int(case.starts[-1])
    for o in outs[1:]:
        assert np.array_equal(o.to_numpy()[:used], outs[0].to_numpy()[:used])
    case.check(case.run(window=1 << 40, sinks=9), case.want())


@pytest.mark.parametrize("sinks", [0, 70])
def test_workspace_and_graph(dev16, sinks):
    """With a workspace of its own a call can be recorded, and replayed on new lengths and shared tokens; a smaller one is refused, and so
    is none while a graph is recorded. Two graphs, each with its own, take turns with eager calls."""
    dev, made = dev16, []
    for seed in (31, 32):
        case = Case(dev, [(1, 900), (1, 1200), (2, 800), (1, 1000)], 2, 4, 128, "BF16", [(0, 3, 700)] if not sinks else (), seed=seed)
        args, shared, _ = case.upload()
        n = ops.kv_attention_work(*args[:4], case.most, window=900 if sinks else 0, sinks=sinks, shared=shared)
        assert n > 0
        out, work = new(dev, "F32", [case.rows, 1024]), new(dev, "U8", [n])
        kw = dict(window=900 if sinks else 0, sinks=sinks, shared=shared)
        graph = Recorded(dev, lambda: ops.kv_attention(*args, out, work=work, **kw))
        with pytest.raises(Error, match="smaller"):
            ops.kv_attention(*args, out, work=new(dev, "U8", [n - 16]), **kw)
        with pytest.raises(Error, match="workspace of its own"):
            Recorded(dev, lambda: ops.kv_attention(*args, out, **kw))
        made.append((case, args, shared, out, kw, graph))
    for step in range(4):
        for case, args, shared, out, kw, graph in made:
            case.lengths = np.array([900, 1200, 800, 1000]) - 60 * step
            args[4]._owner.write(case.lengths.astype(np.int32))
            if shared:
                shared.tokens._owner.write(np.array([704 - 128 * step], np.int32))
            graph.replay()
        for case, args, shared, out, kw, graph in made:
            got = out.to_numpy()
            ops.kv_attention(*args, out, **kw)
            assert np.array_equal(got[:5], out.to_numpy()[:5]), step
            case.tokens = [704 - 128 * step] if shared else []
            want = case.want(window=kw["window"], sinks=sinks)
            assert (np.abs(got[:5].reshape(5, 8, 128) - want[0][:5]) <= want[2][:5]).all(), step
    for m in made:
        m[5].close()


def test_two_contexts(dev):
    """Two contexts on streams of their own, called in turn without a wait between: each its own scratch."""
    other = context(2)
    case = [Case(d, [(1, 900), (1, 1200), (1, 800)], 2, 4, 128, "BF16", [(0, 3, 700)], seed=33 + i) for i, d in enumerate((dev, other))]
    held = [(c.upload(), new(c.dev, "F32", [c.rows, 1024])) for c in case]
    for _ in range(20):
        for (args, shared, _), out in held:
            ops.kv_attention(*args, out, shared=shared)
    for c, (_, out) in zip(case, held):
        c.dev.wait()
        want = c.want()
        assert (np.abs(out.to_numpy()[:3].reshape(3, 8, 128) - want[0][:3]) <= want[2][:3]).all()
    del held
    other.close()


def test_which_kernels_run(dev, dev2):
    """A small batch goes through the shared tokens for each sequence; a larger one (for the context) has a launch of them, whose sums the
    sequences' own launch takes up."""
    for d, out_dt, want in ((dev, "F32", ["kv_attn_kernel<2, 1, false, 1>", "kv_join_kernel<2, 16>"]),
                            (dev2, "BF16", ["kv_attn_rows_kernel<2, 1, false, 2, false>", "kv_attn_kernel<2, 1, false, 1>"]),
                            (dev2, "F32", ["kv_attn_rows_kernel<2, 1, false, 2, true>", "kv_attn_kernel<2, 1, false, 1>"])):
        case = Case(d, [(1, 1000)] * 8, 2, 8, 128, "BF16", [(0, 8, 256)])
        args, shared, _ = case.upload()
        out = new(d, out_dt, [case.rows, 2 * 8 * 128])
        work = new(d, "U8", [ops.kv_attention_work(*args[:4], 1, shared=shared)])
        ran = [name for name, _, _ in launches(d, lambda: ops.kv_attention(*args, out, shared=shared, work=work))]
        assert len(ran) == 2 and all(r.startswith(w) for r, w in zip(ran, want)), ran


@pytest.mark.parametrize("dt", ["BF16", "F16"])
@pytest.mark.parametrize("apart", [False, True])
def test_answers_over_shared_tokens_in_float32(dev, dev2, dt, apart):
    """Float32 results of 16-bit queries are float32's, shared or not: a term's error is that of its score, below 2^3, in float32 (2^-20 of the
    term; probabilities as two halves add 2^-22), and terms and errors add up alike. Eight times that is allowed. (Probabilities as one
    half are off by up to 2^-11 each.)"""
    case = Case(dev2 if apart else dev, [(1, 260 + b) for b in range(8)], 2, 8, 128, dt, [(0, 8, 256)])
    got, want = case.run(scale=0.02)[0][:8], case.want(scale=np.float32(0.02))[0][:8]
    assert np.sqrt(((got - want) ** 2).mean()) <= 2.0 ** -17 * np.sqrt((want ** 2).mean())
