"""Attention over the key/value cache (include/h3lm.h, kv_attention and kv_attention_spans): to how many bits sequences of few rows have their
results beside longer ones, against the restatement in numpy (spans_reference.py)."""
import numpy as np
import pytest

import lm_reference as lm
import spans_reference as ref
from helpers import launches, new
from test_gpu_spans import Case, context

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import ops  # noqa: E402


@pytest.fixture(scope="module")
def dev2():
    d = context(2)
    yield d
    d.close()


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
