"""lin_attention's ways: which kernels a batch takes, segments, workspaces, graphs, streams and contexts, and a text model's layers of both kinds
over a growing conversation."""
import numpy as np
import pytest

import lin_reference as ref
import lm_reference as lm
import spans_reference as spans
from helpers import launches, new, up
from test_gpu_lin import Case, i32, run
from test_gpu_lm import Recorded
from test_gpu_spans import context

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import Device, Error, Tensor, ops  # noqa: E402


@pytest.fixture(scope="module")
def dev1():
    d = context(1)
    yield d
    d.close()


@pytest.fixture(scope="module")
def dev8():
    d = context(8)
    yield d
    d.close()


def test_which_kernels_run(dev, dev1):
    """Few tokens: one launch; many: pieces, split into segments where heads are few; both where a batch has both and fills the device."""
    for dev, counts, heads, each, want in (
        (dev, [1, 1, 3], 2, (1, 1, 1), ["lin_step_kernel"]),
        (dev, [600], 2, (1, 1, 1), ["lin_chunk_kernel", "lin_scan_kernel", "lin_chunk_kernel"]),
        (dev, [100, 90], 2, (1, 1, 1), ["lin_chunk_kernel"]),
        (dev, [1, 600, 1, 1], 2, (1, 1, 1), ["lin_chunk_kernel", "lin_scan_kernel", "lin_chunk_kernel"]),
        (dev1, [1, 600, 6, 1, 7, 1], 2, (1, 1, 1), ["lin_step_kernel", "lin_chunk_kernel"]),
    ):
        case = Case(dev, counts, heads, each, 64, 64, "BF16", 51)
        args = case.operands()
        out = new(dev, "F32", [case.rows, heads * 64])
        n = ops.lin_attention_work(args[0], *args[2:3], *args[5:])
        work = new(dev, "U8", [max(n, 16)])
        ran = [k.split("<")[0] for k, _, _ in launches(dev, lambda: ops.lin_attention(*args, out, work=work))]
        assert ran == want, (counts, ran)
        case.check(*run(case), "F32", what=str(counts))


@pytest.mark.parametrize("dt", ["BF16", "F16", "F32"])
@pytest.mark.parametrize("dk,dv", [(32, 64), (32, 128), (64, 128), (96, 100), (128, 64), (128, 200), (160, 48), (192, 128), (256, 256)])
@pytest.mark.parametrize("full", [False, True])
def test_every_width(dev, dev1, dk, dv, dt, full):
    """Each number of steps over the keys' features and of values a block has, whole pieces and rests. (A device that is full takes 128 features
    of values a block, where there are more than 64.)"""
    dev = dev1 if full else dev
    case = Case(dev, [259, 64, 17, 1], 2, (1, 2, 1), dk, dv, dt, 52 + dk + dv, begin=[1])
    case.check(*run(case), "F32")
    case = Case(dev, [70, 31], 1, (1, 1, 1), dk, dv, dt, 53 + dk + dv, begin=[1], offset=3, pad=2)
    case.check(*run(case, dt), dt, what="rows off 16 bytes")


def kernels(case):
    args = case.operands()
    out = new(case.dev, "F32", [case.rows, case.state.shape[1] * case.dv])
    work = new(case.dev, "U8", [max(ops.lin_attention_work(args[0], *args[2:3], *args[5:]), 16)])
    return [k for k, _, _ in launches(case.dev, lambda: ops.lin_attention(*args, out, work=work))]


@pytest.mark.parametrize("dt", ["BF16", "F16", "F32"])
@pytest.mark.parametrize("dk,dv", [(32, 128), (64, 100), (96, 128), (128, 100), (192, 128)])
def test_segments_of_every_width(dev, dev8, dk, dv, dt):
    """Several segments, in blocks of 64 and of 128 features of values."""
    for d, counts, wide in ((dev, [1100, 40], False), (dev8, [1100], True)):
        case = Case(d, counts, 2, (1, 1, 1), dk, dv, dt, 59 + dk, begin=[0])
        ran = kernels(case)
        assert [k.split("<")[0] for k in ran] == ["lin_chunk_kernel", "lin_scan_kernel", "lin_chunk_kernel"], ran
        waves, tiles = (int(x) for x in ran[0].split("<")[1].split(",")[2:4])
        assert 16 * waves * tiles == (128 if wide else 64), ran
        case.check(*run(case), "F32", what=str(wide))


def test_states_off_16_bytes_and_wide_rows(dev):
    """States from a 4-byte boundary on, few and many tokens; rows so far apart that pieces are read row by row."""
    for counts in ([3, 1], [150]):
        case = Case(dev, counts, 2, (1, 1, 1), 32, 36, "F32", 54)
        args = list(case.operands())
        whole = up(dev, np.concatenate([[7.0], case.state.ravel()]).astype(np.float32), "F32", [1 + case.state.size])
        args[0] = ops.LinState(Tensor(whole.dtype, list(case.state.shape), whole.ptr() + 4, whole, dev))
        out = new(dev, "F32", [case.rows, 2 * 36])
        ops.lin_attention(*args, out)
        got = whole.to_numpy()
        assert got[0] == 7.0
        case.check(out.to_numpy(), got[1:].reshape(case.state.shape), "F32", what=str(counts))
    case = Case(dev, [40], 1, (1, 1, 1), 32, 32, "BF16", 55, tail=0, pad=(1 << 22) - 104)
    assert case.stride == 1 << 22
    case.check(*run(case), "F32", what="wide rows")


def test_states_past_32_bits(dev):
    """The last slots of a pool of more than 2^31 numbers (and its one before the last of the first 2^31), few tokens and many, as in a small pool."""
    heads, d, rows = 64, 128, 73
    x = lm.to_bits(np.random.default_rng(64).standard_normal((rows, 3 * heads * d)), "BF16")
    decay = up(dev, np.linspace(0, 0.3, heads).astype(np.float32), "F32", [heads])
    x = up(dev, x, "BF16", [rows, 3 * heads * d])
    r = [ops.Rows(x, i * heads * d, 3 * heads * d, rows, heads, d) for i in range(3)]
    got = []
    for slots, a, b in ((3, 0, 2), ((1 << 31) // (heads * d * d) + 6, (1 << 31) // (heads * d * d) - 1, (1 << 31) // (heads * d * d) + 5)):
        state = ops.LinState.new(dev, slots, heads, d, d)
        out = new(dev, "F32", [rows, heads * d])
        ops.lin_attention(state, decay, *r, i32(dev, [0, 3]), i32(dev, [-1]), i32(dev, [a]), 3, out)
        ops.lin_attention(state, decay, *r, i32(dev, [3, rows]), i32(dev, [a]), i32(dev, [b]), rows - 3, out)
        ops.lin_attention(state, decay, *r, i32(dev, [0, 2]), i32(dev, [b]), i32(dev, [b]), 2, out)
        got.append(out.to_numpy())
        del state
    assert np.isfinite(got[0]).all() and np.array_equal(*got)


def test_a_batch_past_one_segment_each(dev):
    """Ragged prompts whose segments begin anywhere among the rows, against one prompt at a time: within the bounds, states and all."""
    counts = [513, 128, 0, 129, 127, 1, 700, 64]
    case = Case(dev, counts, 2, (1, 1, 1), 64, 64, "BF16", 56, begin=[0, 3])
    case.check(*run(case), "F32")


def test_most_is_more_than_there_is(dev):
    """`most` above every sequence's rows changes nothing but how the work is split."""
    case = Case(dev, [40, 130], 2, (1, 1, 1), 64, 64, "F16", 57)
    for most in (130, 1000, 1 << 40):
        case.most = most
        case.check(*run(case), "F32", what=str(most))


def test_a_sequence_of_more_rows_than_most(dev):
    """More rows than `most` says: nothing outside the buffers is touched, the other sequences and slots are as they should be."""
    for counts, most in (([30, 300, 9], 40), ([9, 300, 3], 10)):
        case = Case(dev, counts, 2, (1, 1, 1), 64, 64, "BF16", 58)
        case.most = most
        out, state = run(case)
        y, s, tol, stol = ref.run(case.state, case.decay, *case.values(), case.starts, case.source, case.target, "BF16", "F32")
        ok = np.abs(out.reshape(case.rows, 2, 64) - y) <= tol
        a, e = case.starts[1], case.starts[2]
        assert ok[:a].all() and ok[e:case.starts[-1]].all() and ok[a:a + most].all()
        keep = np.arange(len(state)) != case.target[1]
        assert (np.abs(state - s) <= stol)[keep].all()


def test_workspace_and_graph(dev):
    """With a workspace of its own a call can be recorded and replayed: the state goes on from replay to replay as in eager calls, bit for bit.
    A smaller workspace is refused, and so is none while a graph is recorded. Two graphs take turns."""
    made = []
    for seed, counts in ((61, [900, 40]), (62, [1, 2])):
        case = Case(dev, counts, 2, (1, 1, 1), 64, 64, "BF16", seed)
        eager, held = case.operands(), case.operands()
        n = ops.lin_attention_work(held[0], *held[2:3], *held[5:])
        assert (n > 0) == (counts[0] == 900)
        out, want = new(dev, "F32", [case.rows, 128]), new(dev, "F32", [case.rows, 128])
        work = new(dev, "U8", [n]) if n else None
        graph = Recorded(dev, lambda: ops.lin_attention(*held, out, work=work))
        if n:
            with pytest.raises(Error, match="smaller"):
                ops.lin_attention(*held, out, work=new(dev, "U8", [n - 16]))
            with pytest.raises(Error, match="workspace of its own"):
                Recorded(dev, lambda: ops.lin_attention(*held, out))
        made.append((case, eager, held, out, want, graph))
    for step in range(4):
        for case, eager, held, out, want, graph in made:
            graph.replay()
        for case, eager, held, out, want, graph in made:
            ops.lin_attention(*eager, want)
            used = int(case.starts[-1])
            assert np.array_equal(out.to_numpy()[:used], want.to_numpy()[:used]), step
            assert np.array_equal(eager[0].s.to_numpy(), held[0].s.to_numpy()), step
    for m in made:
        m[5].close()


def test_two_contexts(dev):
    """Two contexts on streams of their own, called in turn without a wait between: each its own scratch."""
    other = Device.open()
    case = [Case(d, [1000, 70], 2, (1, 1, 1), 64, 64, "BF16", 63 + i) for i, d in enumerate((dev, other))]
    held = [(c.operands(), new(c.dev, "F32", [c.rows, 128])) for c in case]
    for args, out in held:
        args[6]._owner.write(np.array([-1, -1], np.int32))                           # (every call begins anew)
    for _ in range(20):
        for args, out in held:
            ops.lin_attention(*args, out)
    for c, (args, out) in zip(case, held):
        c.dev.wait()
        c.source = np.array([-1, -1])
        c.check(out.to_numpy(), args[0].s.to_numpy(), "F32")
    del held, args, out
    other.close()


def test_both_kinds_of_layers_over_a_conversation(dev):
    """Three conversations that share their first 128 tokens go through a layer with a cache (a window, first tokens, the shared ones once for
    all) and a linear one: the prompt, then answers token by token as one recorded graph. Every stage is within its bounds of the stage before;
    the recorded steps give what eager ones give, bit for bit."""
    heads, group, dim, width, seqs = 2, 2, 64, 6, 3
    g = np.random.default_rng(71)
    block = lm.BLOCK
    table = np.array([[0, 1, 2, 3, 4, 5], [0, 1, 6, 7, 8, 9], [0, 1, 10, 11, 12, 13]], np.int32)
    window, sinks, wide = 150, 5, heads * group * dim
    qkv = (heads * group + 2 * heads) * dim

    class Model:
        def __init__(self):
            self.cache, self.host = ops.KvCache.new(dev, 14, heads, dim), lm.Cache(14, heads, dim, 72)
            w = lm.width(dim)
            for t, a in ((self.cache.k, self.host.k), (self.cache.v, self.host.v), (self.cache.k_scale, self.host.s[0]), (self.cache.v_scale, self.host.s[1])):
                t._owner.write(np.ascontiguousarray(a))
            assert w == dim
            self.state = ops.LinState(up(dev, np.zeros((seqs + 1, heads * group, dim, dim), np.float32), "F32", [seqs + 1, heads * group, dim, dim]))
            self.decay = up(dev, np.array([0.01, 0.1, 0.5, 2.0], np.float32), "F32", [4])
            self.table, self.past, self.lengths = i32(dev, table), i32(dev, [0] * seqs), i32(dev, [0] * seqs)
            self.shared = ops.KvShared(i32(dev, [0, seqs]), i32(dev, [2 * block]), 2 * block)

        def rows(self, x, n, off=0):
            return [ops.Rows(x, off + a, qkv, n, h, dim) for a, h in ((0, heads * group), (wide, heads), (wide + heads * dim, heads))]

        def write(self, x, n, starts, most, tb=None):
            r = self.rows(x, n)
            ops.kv_write(self.cache, tb or self.table, r[1], r[2], starts, self.past, most)

        def layers(self, x, n, starts, source, target, most, mid, out, work=None, work2=None):
            """The cache's layer into mid, and the linear layer over mid as queries, the same keys and values."""
            r = self.rows(x, n)
            ops.kv_attention(self.cache, self.table, r[0], starts, self.lengths, most, mid, window=window, sinks=sinks, shared=self.shared, work=work)
            ops.lin_attention(self.state, self.decay, ops.Rows(mid, 0, wide, n, heads * group, dim), *[ops.Rows(x, v.offset, qkv, n, heads, dim) for v in r[1:]],
                              starts, source, target, most, out, work=work2)

    def bf16(a):
        return lm.from_bits(lm.to_bits(a, "BF16"), "BF16")

    def check(model, val, n_of, lengths, mid, out, state_before, source, target):
        starts = np.concatenate([[0], np.cumsum(n_of)])
        q = val[:, :wide].reshape(-1, heads * group, dim)
        want = spans.attention(model.host, table, starts, lengths, q, group, "BF16", "BF16", None, window, sinks, None, [0, seqs], [2 * block])
        got = lm.from_bits(mid.to_numpy(), "BF16").reshape(-1, heads * group, dim)
        assert (np.abs(got - want[0]) <= want[2]).all()
        kv = [val[:, a:a + heads * dim].reshape(-1, heads, dim) for a in (wide, wide + heads * dim)]
        y, s, tol, stol = ref.run(state_before, np.array([0.01, 0.1, 0.5, 2.0], np.float32), got, *kv, starts, source, target, "BF16", "F32")
        off = np.abs(out.to_numpy().reshape(y.shape) - y)
        assert (off <= tol).all(), np.nanmax(off / tol)
        after = model.state.s.to_numpy()
        assert (np.abs(after - s) <= stol).all()
        return after

    # the shared tokens are written and taken up once (slot 3 holds the state behind them), then each goes on with its own prompt
    models = [Model(), Model()]
    prefix = bf16(g.standard_normal((2 * block, qkv)).astype(np.float32))
    own = [70, 1, 40]
    prompts = bf16(g.standard_normal((sum(own), qkv)).astype(np.float32))
    for m in models:
        x = up(dev, lm.to_bits(prefix, "BF16"), "BF16", list(prefix.shape))
        m.write(x, 2 * block, i32(dev, [0, 2 * block]), 2 * block, Tensor(m.table.dtype, [1, width], m.table.ptr(), m.table, dev))
        m.host.write(table[:1], [0, 2 * block], [0], [prefix[:, a:a + heads * dim].reshape(-1, heads, dim) for a in (wide, wide + heads * dim)])
        first = new(dev, "F32", [2 * block, wide])
        r = m.rows(x, 2 * block)
        ops.lin_attention(m.state, m.decay, *[ops.Rows(x, v.offset, qkv, 2 * block, v.heads, dim) for v in r], i32(dev, [0, 2 * block]), i32(dev, [-1]),
                          i32(dev, [3]), 2 * block, first)
        before = m.state.s.to_numpy()
        n, starts = sum(own), i32(dev, np.concatenate([[0], np.cumsum(own)]))
        lengths = np.array([2 * block + c for c in own])
        m.past._owner.write(np.array([2 * block] * seqs, np.int32))
        m.lengths._owner.write(lengths.astype(np.int32))
        x = up(dev, lm.to_bits(prompts, "BF16"), "BF16", list(prompts.shape))
        m.write(x, n, starts, max(own))
        m.host.write(table, np.concatenate([[0], np.cumsum(own)]), np.array([2 * block] * seqs),
                     [prompts[:, a:a + heads * dim].reshape(-1, heads, dim) for a in (wide, wide + heads * dim)])
        mid, out = new(dev, "BF16", [n, wide]), new(dev, "F32", [n, wide])
        m.layers(x, n, starts, i32(dev, [3, 3, 3]), i32(dev, [0, 1, 2]), max(own), mid, out)
        m.after = check(m, prompts, own, lengths, mid, out, before, [3, 3, 3], [0, 1, 2])
        m.len = lengths
    # answers: eager in one model, a recorded graph in the other
    starts, slots = i32(dev, [0, 1, 2, 3]), i32(dev, [0, 1, 2])
    held = []
    for m in models:
        x, mid, out = new(dev, "BF16", [seqs, qkv]), new(dev, "BF16", [seqs, wide]), new(dev, "F32", [seqs, wide])
        r = m.rows(x, seqs)
        n = ops.kv_attention_work(m.cache, m.table, r[0], starts, 1, window=window, sinks=sinks, shared=m.shared)
        work = new(dev, "U8", [max(n, 16)])

        def step(m=m, x=x, mid=mid, out=out, work=work):
            m.write(x, seqs, starts, 1)
            m.layers(x, seqs, starts, slots, slots, 1, mid, out, work)

        held.append((m, x, mid, out, step))
    graph = Recorded(dev, held[1][4])
    for i in range(5):
        val = bf16(g.standard_normal((seqs, qkv)).astype(np.float32))
        for k, (m, x, mid, out, step) in enumerate(held):
            past = m.len + i
            x._owner.write(lm.to_bits(val, "BF16"))
            m.past._owner.write(past.astype(np.int32))
            m.lengths._owner.write((past + 1).astype(np.int32))
            m.host.write(table, [0, 1, 2, 3], past, [val[:, a:a + heads * dim].reshape(-1, heads, dim) for a in (wide, wide + heads * dim)])
            if k:
                graph.replay()
            else:
                step()
            m.after = check(m, val, [1] * seqs, past + 1, mid, out, m.after, [0, 1, 2], [0, 1, 2])
        assert np.array_equal(held[0][2].to_numpy(), held[1][2].to_numpy()) and np.array_equal(held[0][3].to_numpy(), held[1][3].to_numpy())
        assert np.array_equal(models[0].after, models[1].after)
    graph.close()
