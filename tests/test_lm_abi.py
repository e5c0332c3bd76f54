"""The table of include/h3lm.h without a GPU: it is there, its entries are the header's, and bad arguments are refused with a message
before the device is touched. No call here launches a kernel."""
import ctypes as C
import os
import re

import pytest

from sycl_minimax_h3_amd import DType, Error, Tensor, ops
from sycl_minimax_h3_amd import api as A

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20   # a 16-byte aligned address that is never dereferenced


@pytest.fixture(scope="module")
def lm():
    return A.load().lm


def test_table_and_header_agree(lm):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "h3lm.h")).read(), flags=re.S)
    names = re.findall(r"\(\*(\w+)\)\(", text)
    assert names == [n for n, _ in A.LmApi._fields_[1:]]
    for n in names:
        args = re.search(r"\(\*%s\)\(([^)]*)\)" % n, text, re.S).group(1)
        assert len(args.split(",")) == len(dict(A.LmApi._fields_)[n]._argtypes_), n
    assert lm.size == C.sizeof(A.LmApi) == 8 * (1 + len(names))
    assert re.search(r"H3_KV_BLOCK = (\d+)", text).group(1) == str(A.KV_BLOCK)


def cache(**k):
    return A.KvCache(**{**dict(k=P, v=P, k_scale=P, v_scale=P, blocks=4, heads=2, dim=128), **k})


def batch(**k):
    return A.KvBatch(**{**dict(table=P, starts=P, seqs=2, width=2, rows=8, most=4), **k})


def refused(rc, word):
    assert rc == -1 and word in A.load().error(), (rc, A.load().error())


def test_cache_arguments(lm):
    def write(c, b, past=P, k=P, ks=256, v=P, vs=256, dt=A.BF16):
        return lm.kv_write(None, C.byref(c) if c else None, C.byref(b) if b else None, past, k, ks, v, vs, dt)

    refused(write(None, batch()), "required")
    refused(write(cache(), None), "required")
    refused(write(cache(dim=257), batch()), "256")
    refused(write(cache(blocks=0), batch()), "blocks")
    refused(write(cache(k=P + 8), batch()), "aligned")
    refused(write(cache(v_scale=None), batch()), "required")
    refused(write(cache(), batch(seqs=-1)), "negative")
    refused(write(cache(), batch(width=1 << 30)), "32 bits")
    refused(write(cache(), batch(starts=None)), "required")
    refused(write(cache(), batch(), past=None), "past")
    refused(write(cache(), batch(), ks=255), "stride")
    refused(write(cache(), batch(), vs=255), "stride")
    refused(write(cache(), batch(), dt=5), "element type")
    refused(write(cache(), batch()), "no context")
    refused(lm.kv_read(None, C.byref(cache()), C.byref(batch()), None, P, 256, P, 256, 0), "first")
    refused(lm.kv_read(None, C.byref(cache()), C.byref(batch()), P, P, 256, P, 256, 0), "no context")
    for b in (batch(seqs=0), batch(rows=0), batch(most=0)):
        assert write(cache(), b, past=None, k=None, v=None) == 0
        assert lm.kv_read(None, C.byref(cache()), C.byref(b), None, None, 256, None, 256, 0) == 0


def test_attention_arguments(lm):
    def attn(c=None, b=None, lengths=P, max_len=0, q=P, qs=512, dt=A.BF16, heads=4, scale=0.0, window=0, mask=None, mask_n=0, out=P, out_dt=A.BF16,
             work=None, n=0):
        return lm.kv_attention(None, C.byref(c or cache()), C.byref(b or batch()), lengths, max_len, q, qs, dt, heads, scale, window, mask, mask_n,
                               out, out_dt, None, work, n)

    refused(attn(heads=5), "multiple")
    refused(attn(heads=0), "multiple")
    refused(attn(max_len=-1), "negative")
    refused(attn(window=-1), "negative")
    refused(attn(mask=P, mask_n=-1), "mask")
    refused(attn(scale=-1.0), "scale")
    refused(attn(scale=float("nan")), "scale")
    refused(attn(scale=float("inf")), "scale")
    refused(attn(dt=3), "element type")
    refused(attn(out_dt=-1), "element type")
    refused(attn(qs=511), "stride")
    refused(attn(lengths=None), "required")
    refused(attn(out=None), "required")
    refused(attn(work=P + 4, n=64), "aligned")
    refused(attn(cache(dim=0)), "features")
    refused(attn(), "no context")
    refused(lm.kv_attention_work(None, C.byref(cache()), C.byref(batch()), 0, 4, 0), "no context")
    refused(lm.kv_attention_work(None, C.byref(cache()), C.byref(batch()), 0, 3, 0), "multiple")
    for b in (batch(seqs=0), batch(rows=0), batch(most=0)):
        assert attn(b=b, q=None, out=None, lengths=None) == 0


def test_linear4_arguments(lm):
    def lin(x=P, dt=A.BF16, m=2, k=256, codes=P, n=8, scale=P, mins=None, sdt=A.F16, group=32, out=P, out_dt=A.BF16):
        return lm.linear4(None, x, dt, m, k, codes, n, scale, mins, sdt, group, None, out, out_dt)

    refused(lin(group=16), "multiple of 32")
    refused(lin(group=96), "divides")
    refused(lin(group=0), "multiple of 32")
    refused(lin(k=0), "divides")
    refused(lin(dt=4), "element type")
    refused(lin(sdt=4), "element type")
    refused(lin(x=P + 2), "aligned")
    refused(lin(codes=P + 1), "aligned")
    refused(lin(scale=None), "required")
    refused(lin(m=-1), "negative")
    refused(lin(), "no context")
    assert lin(m=0, x=None, out=None) == 0 and lin(n=0, codes=None) == 0


def test_ops_layer_checks():
    class D:
        pass

    d = D()
    t = lambda dt, shape: Tensor(DType[dt], shape, P, None, d)  # noqa: E731
    k, v, s = t("I8", [4, 2, 64, 128]), t("I8", [4, 2, 128, 64]), t("F32", [4, 2])
    c = ops.KvCache(k, v, s, s, 100)
    assert ops.KvCache.width(100) == 128 and ops.KvCache.width(64) == 64 and ops.KvCache.width(256) == 256
    with pytest.raises(Error, match="1 to 256"):
        ops.KvCache(k, v, s, s, 300)
    with pytest.raises(Error, match="k must be int8"):
        ops.KvCache(k, v, s, s, 64)
    with pytest.raises(Error, match="v must be int8"):
        ops.KvCache(k, k, s, s, 128)
    with pytest.raises(Error, match="v_scale"):
        ops.KvCache(k, v, s, t("F32", [4]), 128)
    x = t("BF16", [8, 400])
    r = ops.Rows(x, 0, 400, 8, 2, 100)
    table, starts, past = t("I32", [2, 2]), t("I32", [3]), t("I32", [2])
    with pytest.raises(Error, match="for a cache"):
        ops.kv_write(c, table, ops.Rows(x, 0, 400, 8, 2, 64), r, starts, past, 4)
    with pytest.raises(Error, match="starts"):
        ops.kv_write(c, table, r, r, past, past, 4)
    with pytest.raises(Error, match="past"):
        ops.kv_write(c, table, r, r, starts, t("I64", [2]), 4)
    with pytest.raises(Error, match="block table"):
        ops.kv_read(c, past, starts, past, 4, r, r)
    with pytest.raises(Error, match="q heads"):
        ops.kv_attention(c, table, ops.Rows(x, 0, 400, 8, 4, 64), starts, past, 4, x)
    q = ops.Rows(x, 0, 400, 8, 4, 100)
    with pytest.raises(Error, match="out"):
        ops.kv_attention(c, table, q, starts, past, 4, t("BF16", [8, 399]))
    with pytest.raises(Error, match="mask"):
        ops.kv_attention(c, table, q, starts, past, 4, x, mask=t("F32", [2, 5]))
    with pytest.raises(Error, match="lse"):
        ops.kv_attention(c, table, q, starts, past, 4, x, lse=t("F32", [8, 2]))
    w = t("U8", [16, 64])
    with pytest.raises(Error, match="uint8"):
        ops.Int4Linear(t("I8", [16, 64]), s).forward(x, x)
    with pytest.raises(Error, match="scales"):
        ops.Int4Linear(w, t("F16", [15, 4])).forward(t("BF16", [2, 128]), t("BF16", [2, 16]))
    with pytest.raises(Error, match="minima"):
        ops.Int4Linear(w, t("F16", [16, 4]), t("F32", [16, 4])).forward(t("BF16", [2, 128]), t("BF16", [2, 16]))
    with pytest.raises(Error, match="do not fit"):
        ops.Int4Linear(w, t("F16", [16, 4])).forward(t("BF16", [2, 120]), t("BF16", [2, 16]))
