"""What kv_attention_spans and lin_attention of include/h3lm.h refuse, without a GPU: every address is made up, and no call here reaches a
launch."""
import ctypes as C

import pytest

from sycl_minimax_h3_amd import DType, Error, Tensor, ops
from sycl_minimax_h3_amd import api as A

P = 1 << 20   # a 16-byte aligned address that is never dereferenced


@pytest.fixture(scope="module")
def lm():
    return A.load().lm


def refused(rc, word):
    assert rc == -1 and word in A.load().error(), (rc, A.load().error())


def cache(**k):
    return A.KvCache(**{**dict(k=P, v=P, k_scale=P, v_scale=P, blocks=4, heads=2, dim=128), **k})


def batch(**k):
    return A.KvBatch(**{**dict(table=P, starts=P, seqs=2, width=2, rows=8, most=4), **k})


def shared(**k):
    return A.KvShared(**{**dict(first=P, tokens=P, groups=1, most=64), **k})


def test_spans_arguments(lm):
    def spans(c=None, b=None, s=None, lengths=P, max_len=0, q=P, qs=512, dt=A.BF16, heads=4, scale=0.0, window=0, sinks=0, mask=None, mask_n=0,
              out=P, out_dt=A.BF16, work=None, n=0):
        return lm.kv_attention_spans(None, C.byref(c or cache()), C.byref(b or batch()), C.byref(s) if s else None, lengths, max_len, q, qs, dt,
                                     heads, scale, window, sinks, mask, mask_n, out, out_dt, None, work, n)

    refused(spans(heads=5), "multiple")
    refused(spans(max_len=-1), "negative")
    refused(spans(window=-1), "negative")
    refused(spans(sinks=-1), "first tokens")
    refused(spans(s=shared(groups=-1)), "groups")
    refused(spans(s=shared(most=-1)), "shared tokens")
    refused(spans(s=shared(groups=1 << 31)), "too many groups")
    refused(spans(s=shared(first=None)), "required")
    refused(spans(s=shared(tokens=None)), "required")
    refused(spans(mask=P, mask_n=-1), "mask")
    refused(spans(scale=-1.0), "scale")
    refused(spans(scale=float("nan")), "scale")
    refused(spans(dt=3), "element type")
    refused(spans(out_dt=-1), "element type")
    refused(spans(qs=511), "stride")
    refused(spans(lengths=None), "required")
    refused(spans(work=P + 4, n=64), "aligned")
    refused(spans(cache(dim=0)), "features")
    for s in (None, shared(), shared(groups=0, first=None, tokens=None)):
        refused(spans(s=s, sinks=3, window=9), "no context")
        refused(lm.kv_attention_spans_work(None, C.byref(cache()), C.byref(batch()), C.byref(s) if s else None, 0, 4, 9, 3), "no context")
    refused(lm.kv_attention_spans_work(None, C.byref(cache()), C.byref(batch()), None, 0, 3, 0, 0), "multiple")
    refused(lm.kv_attention_spans_work(None, C.byref(cache()), C.byref(batch()), None, 0, 4, 0, -1), "first tokens")
    for b in (batch(seqs=0), batch(rows=0), batch(most=0)):
        assert spans(b=b, s=shared(), q=None, out=None, lengths=None) == 0


def state(**k):
    return A.LinState(**{**dict(s=P, slots=3, heads=4, dk=64, dv=96), **k})


def lin_batch(**k):
    return A.LinBatch(**{**dict(starts=P, source=P, target=P, seqs=2, rows=8, most=4), **k})


def test_lin_arguments(lm):
    def lin(s=None, b=None, decay=P, q=P, qs=256, qh=4, k=P, ks=128, kh=2, v=P, vs=96, vh=1, dt=A.BF16, scale=0.0, out=P, out_dt=A.F32, work=None, n=0):
        return lm.lin_attention(None, C.byref(s or state()), C.byref(b or lin_batch()), decay, q, qs, qh, k, ks, kh, v, vs, vh, dt, scale, out,
                                out_dt, work, n)

    refused(lm.lin_attention(None, None, C.byref(lin_batch()), P, P, 256, 4, P, 128, 2, P, 96, 1, 0, 0.0, P, 0, None, 0), "required")
    refused(lm.lin_attention(None, C.byref(state()), None, P, P, 256, 4, P, 128, 2, P, 96, 1, 0, 0.0, P, 0, None, 0), "required")
    for bad in (dict(dk=0), dict(dv=257), dict(slots=0), dict(heads=0)):
        refused(lin(state(**bad)), "256")
    refused(lin(state(slots=1 << 31)), "too many slots")
    refused(lin(state(heads=65536)), "too many slots or heads")
    refused(lin(state(s=None)), "required")
    refused(lin(state(s=P + 2)), "aligned")
    refused(lin(b=lin_batch(seqs=-1)), "negative")
    refused(lin(b=lin_batch(rows=1 << 31)), "32 bits")
    refused(lin(qh=3, qs=999), "multiple")
    refused(lin(kh=0), "multiple")
    refused(lin(vh=8, vs=999), "multiple")
    refused(lin(scale=float("inf")), "scale")
    refused(lin(scale=-1.0), "scale")
    refused(lin(dt=7), "element type")
    refused(lin(out_dt=7), "element type")
    refused(lin(qs=255), "stride")
    refused(lin(ks=127), "stride")
    refused(lin(vs=95), "stride")
    for name in ("decay", "q", "k", "v", "out"):
        refused(lin(**{name: None}), "required")
    for name in ("starts", "source", "target"):
        refused(lin(b=lin_batch(**{name: None})), "required")
    refused(lin(work=P + 8, n=64), "aligned")
    refused(lin(), "no context")
    refused(lm.lin_attention_work(None, C.byref(state()), C.byref(lin_batch()), 2), "no context")
    refused(lm.lin_attention_work(None, C.byref(state()), C.byref(lin_batch()), 9), "element type")
    for b in (lin_batch(seqs=0), lin_batch(rows=0), lin_batch(most=0)):
        assert lin(b=b, decay=None, q=None, k=None, v=None, out=None) == 0


@pytest.mark.parametrize("heads,b,fits", [
    (64, dict(seqs=1 << 16, rows=1 << 16, most=1), True),
    (64, dict(seqs=1 << 17, rows=1 << 17, most=1), False),                      # 3 blocks of 256 threads a head: past 2^24
    (1, dict(seqs=1, rows=(1 << 31) - 1, most=1 << 31), True),                  # (in at most 256 segments)
    (1, dict(seqs=1 << 22, rows=1 << 27, most=40), False),                      # 2^22 segments of a sequence each, and as many more
    (1, dict(seqs=1, rows=1 << 29, most=1 << 29), True),
    (1, dict(seqs=1 << 21, rows=1 << 28, most=300), False),
    (1, dict(seqs=1 << 18, rows=1 << 25, most=300), True),
])
def test_lin_by_threads(lm, heads, b, fits):
    s, lb = C.byref(state(heads=heads)), C.byref(lin_batch(**b))
    word = "no context" if fits else "too many blocks of work"
    refused(lm.lin_attention(None, s, lb, P, P, 64 * heads, heads, P, 64 * heads, heads, P, 96 * heads, heads, 0, 0.0, P, 0, None, 0), word)
    refused(lm.lin_attention_work(None, s, lb, 0), word)


def test_ops_layer_checks():
    class D:
        pass

    d = D()
    t = lambda dt, shape: Tensor(DType[dt], shape, P, None, d)  # noqa: E731
    with pytest.raises(Error, match="float32"):
        ops.LinState(t("BF16", [3, 4, 64, 96]))
    with pytest.raises(Error, match="float32"):
        ops.LinState(t("F32", [3, 4, 64]))
    with pytest.raises(Error, match="256"):
        ops.LinState(t("F32", [3, 4, 64, 257]))
    s = ops.LinState(t("F32", [3, 4, 64, 96]))
    x = t("BF16", [8, 1000])
    q, k, v = ops.Rows(x, 0, 1000, 8, 4, 64), ops.Rows(x, 256, 1000, 8, 2, 64), ops.Rows(x, 384, 1000, 8, 1, 96)
    i2, i3, decay, out = t("I32", [2]), t("I32", [3]), t("F32", [4]), t("F32", [8, 384])
    with pytest.raises(Error, match="for states of"):
        ops.lin_attention(s, decay, v, k, v, i3, i2, i2, 4, out)
    with pytest.raises(Error, match="share"):
        ops.lin_attention(s, decay, q, ops.Rows(t("F16", [8, 1000]), 0, 1000, 8, 2, 64), v, i3, i2, i2, 4, out)
    with pytest.raises(Error, match="share"):
        ops.lin_attention(s, decay, q, ops.Rows(x, 256, 1000, 7, 2, 64), v, i3, i2, i2, 4, out)
    with pytest.raises(Error, match="out"):
        ops.lin_attention(s, decay, q, k, v, i3, i2, i2, 4, t("F32", [8, 383]))
    with pytest.raises(Error, match="same sequences"):
        ops.lin_attention(s, decay, q, k, v, i3, i3, i2, 4, out)
    with pytest.raises(Error, match="int32"):
        ops.lin_attention(s, decay, q, k, v, i3, t("I64", [2]), i2, 4, out)
    with pytest.raises(Error, match="decay"):
        ops.lin_attention(s, t("F32", [3]), q, k, v, i3, i2, i2, 4, out)
    with pytest.raises(Error, match="most rows"):
        ops.lin_attention(s, decay, q, k, v, i3, i2, i2, -1, out)
    with pytest.raises(Error, match="same groups"):
        ops.KvShared(i3, i3)
    with pytest.raises(Error, match="int32"):
        ops.KvShared(t("F32", [3]), i2)
    with pytest.raises(Error, match="shared tokens"):
        ops.KvShared(i3, i2, -1)
