"""kv_attention_spans (include/h3lm.h) restated: what each row sees is written out as a mask of its own, over a table with the shared
tokens' blocks in their places, and handed to the float64 attention of lm_reference.py, which gives the bounds too."""
import numpy as np

import lm_reference as lm


def attention(cache, table, starts, lengths, q, group, q_dt, out_dt, scale=None, window=0, sinks=0, mask=None, first=(), tokens=(), rows=None):
    """As lm_reference.attention, of the given rows (None: all)."""
    seqs, width = table.shape
    merged = table.copy()
    for g in range(len(tokens)):
        n = min(max(tokens[g], 0) // lm.BLOCK, width)
        merged[first[g]:first[g + 1], :n] = table[first[g], :n] if first[g] < seqs else 0
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    tol, ltol = np.full(q.shape, 1e-30), np.zeros(q.shape[:2])
    for b in range(seqs):
        n, length = starts[b + 1] - starts[b], min(lengths[b], width * lm.BLOCK)
        at = np.arange(max(length, 0))
        for j in range(n):
            pos, row = length - n + j, starts[b] + j
            if pos < 0 or (rows is not None and row not in rows):
                continue
            seen = np.ones(pos + 1, np.uint8)
            if window:
                seen[:max(pos - window + 1, 0)] = 0
                seen[:sinks] = 1
            if mask is not None:
                full = np.zeros(pos + 1, bool)
                full[:mask.shape[1]] = mask[b, :pos + 1] != 0
                seen &= full
            r = lm.attention(cache, merged[b:b + 1], [0, 1], [pos + 1], q[row:row + 1], group, q_dt, out_dt, scale, 0, seen[None])
            out[row], lse[row], tol[row], ltol[row] = (x[0] for x in r)
    return out, lse, tol, ltol
