"""Linear attention with a decay for each head (include/h3lm.h, lin_attention) restated in numpy, token by token in float64, with error
bounds derived from the types and the number of tokens."""
import numpy as np

from lm_reference import HALF


def run(state, decay, q, k, v, starts, source, target, dt, out_dt, scale=None):
    """state float32 [slots, heads, dk, dv]; q, k, v float32 [rows, their heads, dk or dv] (values of their type dt). Returns out float64
    [rows, heads, dv], the states after the call, and how far either may be off."""
    slots, heads, dk, dv = state.shape
    scale = dk ** -0.5 if scale is None else float(np.float32(scale))
    q, k, v = (np.repeat(x.astype(np.float64), heads // x.shape[1], 1) for x in (q, k, v))
    with np.errstate(all="ignore"):
        fade = np.where(np.isinf(decay), 0.0, np.exp(-decay.astype(np.float64)))[:, None, None]
    out, tol = np.zeros((len(q), heads, dv)), np.zeros((len(q), heads, dv))
    new, stol = state.astype(np.float64), np.zeros(state.shape)
    for b in range(len(starts) - 1):
        a, e = starts[b], starts[b + 1]
        if e <= a:
            continue
        s = state[source[b]].astype(np.float64) if 0 <= source[b] < slots else np.zeros((heads, dk, dv))
        most = np.abs(s)                             # the same sums of absolute values
        # Float32 roundings, of which a token adds at most four to what it carries (its decay's own error among them) and the sums over
        # the keys one for each: those of the token-by-token form, which in 64-token pieces are fewer. 16-bit inputs in pieces: a
        # value of a product of queries and keys and of a state is held as two bfloat16, 2^-9 of 2^-9 of it off, and the product of the two
        # second parts (2^-18) is left out, for two factors each.
        steps = (4 * (e - a) + dk + 80) * 2.0 ** -24
        parts = 0.0 if dt == "F32" else 2.0 ** -15
        for i in range(a, e):
            with np.errstate(all="ignore"):
                s = fade * s + k[i][:, :, None] * v[i][:, None, :]
                out[i] = (q[i][:, :, None] * s).sum(1) * scale
            most = fade * most + np.abs(k[i][:, :, None] * v[i][:, None, :])
            tol[i] = (np.abs(q[i])[:, :, None] * most).sum(1) * scale * (steps + parts)
        if 0 <= target[b] < slots:
            new[target[b]], stol[target[b]] = s, most * steps
    return out, new, HALF[out_dt] * np.abs(out) + 1.01 * tol + 1e-37, 1.01 * stol + 1e-37
