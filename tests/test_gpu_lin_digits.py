"""To how many digits linear attention in pieces has its results and states: the root mean square of their errors against 64 bits, within
limits that the same arithmetic with a part less exceeds (test_lin_digits.py)."""
import numpy as np
import pytest

import lin_pieces as digits
import lin_reference as ref
from test_gpu_lin import Case, run
from test_gpu_spans import context

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev1():
    d = context(1)
    yield d
    d.close()


@pytest.mark.parametrize("dt", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("dk,dv", digits.SHAPES)
@pytest.mark.parametrize("full", [False, True])
def test_digits_of_results_and_states(dev, dev1, dk, dv, dt, full):
    """Of each sequence and head, in segments of blocks of 64 features of values and whole in blocks of 128."""
    case = Case(dev1 if full else dev, digits.COUNTS, 3, (1, 1, 1), dk, dv, dt, 92, begin=range(4), decay=digits.DECAYS)
    out, state = run(case)
    y, s, _, _ = ref.run(case.state, case.decay, *case.values(), case.starts, case.source, case.target, dt, "F32")
    out = out.reshape(y.shape)
    for b in range(4):
        a, e = case.starts[b], case.starts[b + 1]
        for h in range(3):
            off = digits.error(out[a:e, h], y[a:e, h])
            assert off <= (digits.FULL if dt == "F32" else digits.HELD), (b, h, off)
            off = digits.error(state[case.target[b], h], s[case.target[b], h])
            assert off <= digits.FULL, (b, h, off)
