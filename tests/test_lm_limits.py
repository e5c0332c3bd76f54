"""What include/h3lm.h's operators refuse by size, without a GPU: every address is made up, and no call here reaches a launch."""
import ctypes as C

import pytest

from sycl_minimax_h3_amd import api as A

P = 1 << 20   # a 16-byte aligned address that is never dereferenced


@pytest.fixture(scope="module")
def lm():
    return A.load().lm


def cache(**k):
    return C.byref(A.KvCache(**{**dict(k=P, v=P, k_scale=P, v_scale=P, blocks=4, heads=2, dim=128), **k}))


def batch(**k):
    return C.byref(A.KvBatch(**{**dict(table=P, starts=P, seqs=2, width=2, rows=8, most=4), **k}))


def refused(rc, word):
    assert rc == -1 and word in A.load().error(), (rc, A.load().error())


@pytest.mark.parametrize("heads,b,fits", [
    (32, dict(seqs=1024, width=1024, rows=1024 + 16400, most=16400), True),      # 263168 blocks a head, were all as long
    (8, dict(seqs=2048, width=1024, rows=2048 + 32768, most=32768), True),
    (8, dict(seqs=1, width=1 << 20, rows=1 << 25, most=1 << 25), True),
    (64, dict(seqs=1, width=1 << 20, rows=1 << 25, most=1 << 25), False),         # 2^32 threads and more
    (2, dict(seqs=1 << 22, width=1, rows=1 << 22, most=1), False),
    (1, dict(seqs=1 << 21, width=4, rows=1 << 23, most=70), True),
    (1, dict(seqs=1 << 23, width=4, rows=1 << 23, most=70), False),
])
def test_rows_of_the_cache_by_threads(lm, heads, b, fits):
    for fn in (lm.kv_write, lm.kv_read):
        rc = fn(None, cache(heads=heads, dim=8), batch(**b), P, P, 8 * heads, P, 8 * heads, A.F32)
        refused(rc, "no context" if fits else "too many blocks of work")


@pytest.mark.parametrize("m,n,fits", [(1 << 31, 5376, True), ((1 << 31) + 1, 32, False), (7, 1 << 30, False), (1 << 20, 1 << 29, True)])
def test_linear4_by_threads(lm, m, n, fits):
    rc = lm.linear4(None, P, A.BF16, m, 32, P, n, P, None, A.F16, 32, None, P, A.BF16)
    refused(rc, "no context" if fits else "too many rows or columns")


def test_attention_rows_past_32_bits(lm):
    """Rows times heads of a group are counted in 32 bits, by the call and by the size of its workspace alike."""
    for b, heads, fits in ((dict(rows=1 << 30, most=4), 2, False), (dict(rows=1 << 30, most=4), 1, True), (dict(rows=(1 << 31) - 1, most=1 << 40, seqs=1 << 30), 65535, False)):
        refused(lm.kv_attention_work(None, cache(heads=1, dim=8), batch(**b), 0, heads, 0), "no context" if fits else "too many rows")
        refused(lm.kv_attention(None, cache(heads=1, dim=8), batch(**b), P, 0, P, 8 * heads, A.F32, heads, 0.0, 0, None, 0, P, A.F32, None, None, 0),
                "no context" if fits else "too many rows")
