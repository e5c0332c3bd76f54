"""lin_attention (include/h3lm.h) of thousands of sequences in one call, against its restatement in numpy (lin_reference.py)."""
import numpy as np
import pytest

import lin_reference as ref
import lm_reference as lm
from helpers import launches, new, up
from test_gpu_lin import i32

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import ops  # noqa: E402


@pytest.mark.parametrize("seqs,heads,d,most,want", [
    (4100, 64, 128, 7, ["lin_step_kernel", "lin_chunk_kernel"]),
    (1500, 64, 256, 40, ["lin_step_kernel", "lin_chunk_kernel"]),
    (2000, 4, 128, 1500, ["lin_step_kernel", "lin_chunk_kernel", "lin_scan_kernel", "lin_chunk_kernel"]),
])
def test_thousands_of_sequences(dev, seqs, heads, d, most, want):
    """A token each beside one longer sequence. A few states are kept, the others' dropped."""
    g = np.random.default_rng(81)
    counts = np.ones(seqs, np.int64)
    counts[[3, 700]], counts[seqs - 2] = 0, most
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1])
    bits = lm.to_bits(g.standard_normal((rows, 3 * d)), "BF16")
    state = (4 * g.standard_normal((4, heads, d, d))).astype(np.float32)
    decay = (2.0 ** -g.uniform(0, 8, heads)).astype(np.float32)
    source, target = np.full(seqs, -1), np.full(seqs, -1)
    kept = [0, 1234, seqs - 2, seqs - 1]
    source[kept[:3]], target[kept] = [0, 1, 2], [0, 1, 2, 3]
    x, held = up(dev, bits, "BF16", [rows, 3 * d]), ops.LinState(up(dev, state, "F32", list(state.shape)))
    r = [ops.Rows(x, a * d, 3 * d, rows, 1, d) for a in range(3)]
    args = (held, up(dev, decay, "F32", [heads]), *r, i32(dev, starts), i32(dev, source), i32(dev, target), most)
    out = new(dev, "F32", [rows, heads * d])
    work = new(dev, "U8", [max(ops.lin_attention_work(held, r[0], *args[5:8], most), 16)])
    ran = [k.split("<")[0] for k, _, _ in launches(dev, lambda: ops.lin_attention(*args, out, work=work))]
    assert ran == want, ran
    held.s._owner.write(state)
    ops.lin_attention(*args, out, work=work)
    got, after = out.to_numpy().reshape(rows, heads, d), held.s.to_numpy()
    picks = [*kept, 2, 4, 701, seqs // 2]
    val = lm.from_bits(bits, "BF16").reshape(rows, 3, 1, d)
    at = np.concatenate([np.arange(starts[b], starts[b + 1]) for b in picks])
    y, s, tol, stol = ref.run(state, decay, *(val[at, i] for i in range(3)), np.concatenate([[0], np.cumsum(counts[picks])]), source[picks], target[picks],
                              "BF16", "F32")
    assert (np.abs(got[at] - y) <= tol).all()
    assert (np.abs(after - s) <= stol).all()
    assert np.isfinite(got).all()
