"""Linear attention with a decay for each head (include/h3lm.h, lin_attention) against its restatement in numpy, within bounds derived
from the types (lin_reference.py)."""
import numpy as np
import pytest

import lin_reference as ref
import lm_reference as lm
from helpers import new, up

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import ops  # noqa: E402


def i32(dev, a):
    a = np.ascontiguousarray(a, np.int32)
    return up(dev, a, "I32", list(a.shape))


class Case:
    """Sequences of `counts` tokens over `heads` states of dk x dv, q, k and v with heads / each of their own, in one row of a wider
    buffer; some sequences begin, some are carried on; a few rows and slots behind the last."""

    def __init__(self, dev, counts, heads, each, dk, dv, dt, seed, begin=(), drop=(), decay=None, tail=3, offset=8, pad=8):
        g = np.random.default_rng(seed)
        n = len(counts)
        self.counts, self.dt, self.most = counts, dt, max([*counts, 1])
        self.heads, self.dk, self.dv = [heads // x for x in each], dk, dv
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
        self.rows = int(self.starts[-1]) + tail
        slots = g.permutation(n + 2)[:n]
        self.source, self.target = slots.copy(), slots.copy()
        self.source[list(begin)], self.target[list(drop)] = -1, -1
        self.state = (4 * g.standard_normal((n + 2, heads, dk, dv))).astype(np.float32)
        self.decay = (2.0 ** -g.uniform(0, 8, heads)).astype(np.float32) if decay is None else np.asarray(decay, np.float32)
        sizes = [h * d for h, d in zip(self.heads, (dk, dk, dv))]
        self.at = [offset, offset + sizes[0], offset + sizes[0] + sizes[1]]
        self.stride = offset + sum(sizes) + pad
        self.bits = lm.to_bits(g.standard_normal((self.rows, self.stride)), dt)
        self.dev = dev

    def values(self):
        val = lm.from_bits(self.bits, self.dt)
        return [val[:, a:a + h * d].reshape(self.rows, h, d) for a, h, d in zip(self.at, self.heads, (self.dk, self.dk, self.dv))]

    def operands(self, dev=None):
        dev = dev or self.dev
        x = up(dev, self.bits, self.dt, [self.rows, self.stride])
        r = [ops.Rows(x, a, self.stride, self.rows, h, d) for a, h, d in zip(self.at, self.heads, (self.dk, self.dk, self.dv))]
        s = ops.LinState(up(dev, self.state, "F32", list(self.state.shape)))
        return s, up(dev, self.decay, "F32", [len(self.decay)]), *r, i32(dev, self.starts), i32(dev, self.source), i32(dev, self.target), self.most

    def check(self, out, state, out_dt, scale=None, what=""):
        """out: the values of its type [rows, heads * dv]; state: the slots after the call."""
        heads, used = self.state.shape[1], int(self.starts[-1])
        y, s, tol, stol = ref.run(self.state, self.decay, *self.values(), self.starts, self.source, self.target, self.dt, out_dt, scale)
        got = np.asarray(out, np.float64).reshape(self.rows, heads, self.dv)[:used]
        off = np.abs(got - y[:used])
        assert (off <= tol[:used]).all(), f"{what} out: {(off > tol[:used]).sum()} of {off.size}, {np.nanmax(off / tol[:used]):.2f} of the bound at {np.argwhere(~(off <= tol[:used]))[:3]}"
        off = np.abs(np.asarray(state, np.float64) - s)
        assert (off <= stol).all(), f"{what} state: {(off > stol).sum()} of {off.size}, {np.nanmax(off / stol):.2f} of the bound at {np.argwhere(~(off <= stol))[:3]}"


def run(case, out_dt="F32", scale=0.0, dev=None):
    dev = dev or case.dev
    wide = case.state.shape[1] * case.dv
    mark = lm.to_bits(np.full((case.rows, wide), 55.0), out_dt)
    out = up(dev, mark, out_dt, [case.rows, wide])
    operands = case.operands(dev)
    ops.lin_attention(*operands, out, scale=scale)
    got = out.to_numpy()
    assert np.array_equal(got[case.starts[-1]:], mark[case.starts[-1]:])
    return lm.from_bits(got, out_dt), operands[0].s.to_numpy()


CASES = [
    # tokens of each sequence, heads, states a head of q, k, v, dk, dv, type
    ([1], 4, (1, 1, 1), 128, 128, "BF16"),
    ([1] * 9, 2, (1, 1, 1), 128, 128, "F16"),
    ([0, 1, 2, 0, 5, 8, 9], 3, (1, 1, 1), 64, 64, "F32"),
    ([17, 1, 33], 4, (1, 4, 4), 80, 96, "BF16"),
    ([64, 65, 63], 2, (2, 2, 1), 128, 128, "BF16"),
    ([130, 3], 4, (4, 1, 2), 96, 32, "F16"),
    ([200], 2, (1, 1, 1), 256, 64, "F32"),
    ([70, 1], 2, (1, 2, 2), 192, 256, "BF16"),
    ([97], 1, (1, 1, 1), 1, 1, "F32"),
    ([66, 5], 2, (1, 1, 1), 7, 33, "F16"),
    ([129], 2, (1, 1, 1), 100, 130, "F32"),
    ([300, 1, 256], 2, (1, 1, 1), 33, 250, "BF16"),
    ([700], 2, (1, 1, 1), 128, 128, "F32"),
    ([1000, 20], 1, (1, 1, 1), 128, 64, "F16"),
]


@pytest.mark.parametrize("counts,heads,each,dk,dv,dt", CASES)
def test_lin_attention(dev, counts, heads, each, dk, dv, dt):
    n = len(counts)
    case = Case(dev, counts, heads, each, dk, dv, dt, 11 + dk + dv, begin=range(0, n, 3), drop=range(2, n, 5))
    for out_dt in ("F32", dt if dt != "F32" else "BF16"):
        case.check(*run(case, out_dt), out_dt, what=out_dt)
    case.check(*run(case, scale=0.75), "F32", 0.75, what="scale")


@pytest.mark.parametrize("dt", ["BF16", "F16", "F32"])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 2), (3, 0), (4, 4)])
def test_lin_strides(dev, dt, offset, pad):
    """Rows on and off 16-byte boundaries, few tokens and many."""
    for counts in ([3, 1], [90]):
        case = Case(dev, counts, 2, (1, 1, 1), 64, 36, dt, 12, offset=offset, pad=pad)
        case.check(*run(case), "F32", what=str(counts))


@pytest.mark.parametrize("dt", ["BF16", "F32"])
def test_lin_decays(dev, dt):
    """No decay, decays so small that only their distance from 1 tells, one so strong that a token is forgotten within a piece, infinity."""
    case = Case(dev, [3, 333, 64], 7, (1, 1, 1), 64, 64, dt, 13, decay=[0, 1e-7, 1e-4, 0.01, 2, 90, np.inf])
    case.check(*run(case), "F32")


def test_lin_token_by_token_is_the_prompt(dev):
    """A sequence in one call, in pieces and token by token: all within the bounds, the state carried on in place."""
    case = Case(dev, [150], 2, (1, 1, 1), 64, 96, "BF16", 14, begin=[0], tail=0)
    case.check(*run(case), "F32")
    heads = 2
    for sizes in ([1] * 150, [64, 64, 22], [7, 100, 1, 42]):
        s, decay, q, k, v, _, source, target, _ = case.operands()
        out = new(dev, "F32", [case.rows, heads * case.dv])
        at = 0
        for n in sizes:
            part = [ops.Rows(r.t, r.offset + at * r.stride, r.stride, n, r.heads, r.dim) for r in (q, k, v)]
            piece = new(dev, "F32", [n, heads * case.dv])
            ops.lin_attention(s, decay, *part, i32(dev, [0, n]), source, target, n, piece)
            out._owner.write(piece.to_numpy(), at * heads * case.dv * 4)
            source = target
            at += n
        case.check(out.to_numpy(), s.s.to_numpy(), "F32", what=str(sizes[:4]))


def test_lin_slots(dev):
    """States from one slot into another; slots that are none: zeros, and dropped; what no sequence leaves its state in stays."""
    case = Case(dev, [2, 80, 1, 70, 0, 5], 2, (1, 1, 1), 64, 64, "BF16", 15)
    slots = case.state.shape[0]
    case.source = np.array([0, 0, slots, 1 << 30, 3, -7])
    case.target = np.array([2, 4, 5, slots, 6, -(1 << 31)])
    out, state = run(case)
    case.check(out, state, "F32")
    for i in (0, 1, 3, 6, 7):
        assert np.array_equal(state[i], case.state[i]), i


def test_lin_starts_out_of_order(dev):
    """Starts that run back, below zero and past the rows are cut to the rows."""
    case = Case(dev, [4, 9, 29], 1, (1, 1, 1), 32, 32, "F32", 16, tail=0)
    rows = case.rows
    wild = np.array([-9, 4, 2, 1 << 30])                                              # 0 .. 4, none, 2 .. rows
    s, decay, q, k, v, _, source, target, _ = case.operands()
    out = new(dev, "F32", [rows, 32])
    ops.lin_attention(s, decay, q, k, v, i32(dev, wild), source, target, rows, out)
    case.starts, case.source, case.target = np.array([2, rows]), case.source[2:], case.target[2:]
    val = case.values()
    y, _, tol, _ = ref.run(case.state, case.decay, *val, case.starts, case.source, case.target, "F32", "F32")
    got = out.to_numpy().reshape(rows, 1, 32)
    assert (np.abs(got - y) <= tol)[4:].all()                                         # (rows 2 and 3 are two sequences')


@pytest.mark.parametrize("dt", ["BF16", "F16", "F32"])
@pytest.mark.parametrize("count", [5, 150])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_lin_infinities_and_nans(dev, dt, count, which):
    """An infinity or NaN of one head's token has no effect on earlier tokens, other heads and other sequences; where the definition gives
    an infinity or NaN, the result is one."""
    for bad in (np.inf, np.nan):
        case = Case(dev, [count, count], 2, (1, 1, 1), 64, 64, dt, 17)
        clean = case.bits.copy()
        at = count * 2 // 3
        case.bits[at, case.at[which] + 3] = lm.to_bits(np.array([bad]), dt)[0]       # head 0, sequence 0
        out, state = run(case)
        y, s, tol, stol = ref.run(case.state, case.decay, *case.values(), case.starts, case.source, case.target, dt, "F32")
        assert not np.isfinite(out.reshape(case.rows, 2, -1)[:2 * count][~np.isfinite(y[:2 * count])]).any()
        assert not np.isfinite(state[~np.isfinite(s)]).any()
        case.bits = clean
        y, s, tol, stol = ref.run(case.state, case.decay, *case.values(), case.starts, case.source, case.target, dt, "F32")
        ok = np.abs(out.reshape(case.rows, 2, -1) - y) <= tol
        assert ok[:at, 0].all() and ok[:count, 1].all() and ok[count:2 * count].all()
        mine = case.target[0]
        ok = np.abs(state - s) <= stol
        ok[mine, 0] = True
        assert ok.all()
        if which == 0:
            assert (np.abs(state - s) <= stol).all()                                  # (queries have no part in states)
