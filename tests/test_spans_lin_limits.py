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


@pytest.mark.parametrize("d,seqs,most,fits", [
    # 64 heads. Up to 32 tokens: a block of 256 threads for 32 features of values and, beside it, one of as many for 64 (of 512 for 128 where
    # keys have more than 128 features): the first is the more; 2^32 threads are 2^24 of them
    (128, 4096, 7, True), (128, 65535, 7, True), (128, 65536, 7, False), (128, 65535, 32, True),
    (256, 1024, 7, True), (256, 32767, 7, True), (256, 32768, 7, False),
    # more: the walk over segments has a block of 256 threads for 16 features of keys and 64 of values
    (128, 16383, 40, True), (128, 16384, 40, False), (256, 4095, 33, True), (256, 4096, 33, False),
    (64, 65535, 40, True), (64, 65536, 40, False),
])
def test_lin_sequences(lm, d, seqs, most, fits):  # noqa: F811
    s = C.byref(A.LinState(s=P, slots=3, heads=64, dk=d, dv=d))
    b = C.byref(A.LinBatch(starts=P, source=P, target=P, seqs=seqs, rows=seqs + 104, most=most))
    word = "no context" if fits else "too many blocks of work"
    refused(lm.lin_attention(None, s, b, P, P, 64 * d, 64, P, 64 * d, 64, P, 64 * d, 64, A.BF16, 0.0, P, A.BF16, None, 0), word)
    refused(lm.lin_attention_work(None, s, b, A.BF16), word)
