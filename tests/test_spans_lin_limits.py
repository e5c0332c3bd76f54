"""How large kv_attention_spans' and lin_attention's calls (include/h3lm.h) may be, without a GPU: every address is made up, and no call here
reaches a launch."""
import ctypes as C

import pytest

from sycl_minimax_h3_amd import api as A
from test_spans_lin_abi import P, batch, cache, lm, refused, shared  # noqa: F401


@pytest.mark.parametrize("groups,fits", [((1 << 24) - 1, True), (1 << 24, False), ((1 << 30) + 1, False), ((1 << 31) - 2, False)])
def test_spans_by_groups(lm, groups, fits):  # noqa: F811
    """The kernels look a sequence's group up in steps of 64 that are ints: past 2^30 groups they would leave an int, and the search would not end."""
    word, s = "no context" if fits else "too many groups", C.byref(shared(groups=groups))
    refused(lm.kv_attention_spans(None, C.byref(cache()), C.byref(batch()), s, P, 0, P, 512, A.BF16, 4, 0.0, 9, 3, None, 0, P, A.BF16, None, None, 0), word)
    refused(lm.kv_attention_spans_work(None, C.byref(cache()), C.byref(batch()), s, 0, 4, 9, 3), word)
