"""The operators of include/h3lm.h restated in numpy: the cache's writes and reads in the float32 arithmetic that the header
states (bit for bit), the attention and the 4-bit linear layer in float64, with error bounds derived from the types."""
import numpy as np

BLOCK = 64
HALF = {"BF16": 2.0 ** -8, "F16": 2.0 ** -11, "F32": 2.0 ** -24}       # half a step of a type, relative


def width(dim):
    return (dim + 63) // 64 * 64


def to_bits(x, dt):
    """float32 values as the tensor's bits (float32 stays)."""
    from oracle import oracle as o

    return np.ascontiguousarray(o.to_dt(np.ascontiguousarray(x, np.float32).ravel(), getattr(o, dt))).reshape(np.shape(x))


def from_bits(b, dt):
    from oracle import oracle as o

    return o.from_dt(np.ascontiguousarray(b).ravel(), getattr(o, dt)).astype(np.float32).reshape(np.shape(b))


class Cache:
    """The codes and scales of one layer as arrays: k [blocks, heads, 64, w], v [blocks, heads, w, 64], scales [2, blocks, heads]."""

    def __init__(self, blocks, heads, dim, seed=0):
        g = np.random.default_rng(seed)
        self.dim, self.heads, self.blocks, w = dim, heads, blocks, width(dim)
        self.k = g.integers(-127, 128, (blocks, heads, BLOCK, w), dtype=np.int8)
        self.v = g.integers(-127, 128, (blocks, heads, w, BLOCK), dtype=np.int8)
        self.s = np.exp(g.normal(-4.5, 0.4, (2, blocks, heads))).astype(np.float32)

    def side(self, i, page):
        """[heads, 64, w] of a block, as a view."""
        return self.k[page] if i == 0 else self.v[page].transpose(0, 2, 1)

    def write(self, table, starts, past, rows):
        """rows: (k, v) float32 [rows, heads, dim]."""
        f = np.float32
        for b in range(len(table)):
            n = starts[b + 1] - starts[b]
            end = min(past[b] + n, table.shape[1] * BLOCK)
            for j in range(past[b] // BLOCK, (end + BLOCK - 1) // BLOCK):
                page, lo, hi = table[b, j], j * BLOCK, min(end, (j + 1) * BLOCK)
                if hi <= past[b] or not 0 <= page < self.blocks:
                    continue
                keep = max(past[b] - lo, 0)
                for i in (0, 1):
                    x = rows[i][starts[b] + lo + keep - past[b]:starts[b] + hi - past[b]].transpose(1, 0, 2)
                    with np.errstate(all="ignore"):
                        top = np.abs(x).max((1, 2)) / f(127)
                        was = self.s[i, page] if keep else np.zeros(self.heads, f)
                        s = np.maximum(np.maximum(top, was), f(1e-30))             # (numpy's maximum keeps NaN)
                        c = np.zeros((self.heads, BLOCK, width(self.dim)), f)
                        ratio = (was / s).astype(f)
                        c[:, :keep] = np.rint(self.side(i, page)[:, :keep].astype(f) * ratio[:, None, None])
                        c[:, keep:hi - lo, :self.dim] = np.clip(np.rint((x / s[:, None, None]).astype(f)), -127, 127)
                    self.s[i, page] = s
                    good = np.isfinite(s)
                    self.side(i, page)[good] = c[good].astype(np.int8)             # (else: the codes say nothing)

    def values(self, i, table_row, tokens):
        """float32 [heads, tokens, dim] of a sequence's tokens (zeros where there is no block), and whether there is one."""
        at = np.asarray(tokens)
        out = np.zeros((self.heads, len(at), self.dim), np.float32)
        there = np.zeros(len(at), bool)
        for n, p in enumerate(at):
            page = table_row[p // BLOCK] if 0 <= p < len(table_row) * BLOCK else -1
            if 0 <= page < self.blocks:
                there[n] = True
                out[:, n] = self.side(i, page)[:, p % BLOCK, :self.dim].astype(np.float32) * self.s[i, page][:, None]
        return out, there


def attention(cache, table, starts, lengths, q, group, q_dt, out_dt, scale=None, window=0, mask=None):
    """q float32 [rows, heads * group, dim] (values of its type). Returns out and lse in float64 and the most they may be off by."""
    rows, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    out, lse = np.zeros((rows, heads, dim)), np.full((rows, heads), -np.inf)
    tol, ltol = np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    u_p = 2.0 ** -22 if q_dt == "F32" else 2.0 ** -11
    for b in range(len(table)):
        n, length = starts[b + 1] - starts[b], min(lengths[b], table.shape[1] * BLOCK)
        if length <= 0 or n == 0:
            continue
        k, there = cache.values(0, table[b], np.arange(length))
        v, _ = cache.values(1, table[b], np.arange(length))
        at = np.arange(length)
        for j in range(n):
            pos = length - n + j
            seen = there & (at <= pos)
            if window:
                seen &= at > pos - window
            if mask is not None:
                full = np.zeros(length, bool)
                full[:mask.shape[1]] = mask[b, :length] != 0
                seen &= full
            if not seen.any():
                continue
            for h in range(heads):
                kk, vv, qq = k[h // group][seen].astype(np.float64), v[h // group][seen].astype(np.float64), q[starts[b] + j, h].astype(np.float64)
                s = kk @ qq * scale
                # scores: float32 sums of dim products of the codes, and a factor of three roundings; float32 queries to 2^-22
                ds = ((dim + 16) * 2.0 ** -24 * (np.abs(kk) @ np.abs(qq)) * abs(scale)).max() + 2.0 ** -22 * np.abs(s).max()
                top = s.max()
                p = np.exp(s - top)
                total = p.sum()
                out[starts[b] + j, h] = p @ vv / total
                lse[starts[b] + j, h] = top + np.log(total)
                # probabilities to half a step of half (two halves: 2^-22), a float32 sum of their products, both of a sum
                a = p @ np.abs(vv) / total
                rel = u_p + 2 * ds + 2.0 ** -21 + (len(s) + 64) * 2.0 ** -24
                # Probabilities are held as half times 2^15, the row's largest as 2^15: below 2^-29 of it half's steps are 2^-24, so
                # half a step is 2^-25 / 2^15 = 2^-40 of it, whatever the probability. (Where the largest probability meets a value
                # of 0, the row's result is made of these alone, and they are no longer small against it.)
                least = 2.0 ** -40 * np.abs(vv).sum(0) / total
                tol[starts[b] + j, h] = HALF[out_dt] * np.abs(out[starts[b] + j, h]) + 1.01 * (a * rel + least)
                ltol[starts[b] + j, h] = ds + 2.0 ** -21 + (len(s) + 64) * 2.0 ** -24 + 2.0 ** -22 * abs(lse[starts[b] + j, h])
    return out, lse, tol + 1e-30, ltol


def linear4(x, codes, scale, mins, bias, out_dt):
    """x float32 [M, K], codes uint8 [N, K / 2], scale and mins float32 [N, groups]: float64 result and bound."""
    n, half = codes.shape
    c = np.empty((n, 2 * half))
    c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
    g = 2 * half // scale.shape[1]
    s = np.repeat(scale.astype(np.float64), g, 1)
    z = 8 * s if mins is None else np.repeat(mins.astype(np.float64), g, 1)
    x = x.astype(np.float64)
    y = x @ (s * c - z).T + (0 if bias is None else bias.astype(np.float64))
    # sums of x (16 + c) and of x in float32: 32 terms in one instruction, the groups one by one, eight wavefronts
    terms = np.abs(x) @ (np.abs(s) * (16 + c) + np.abs(16 * s + z)).T + (0 if bias is None else np.abs(bias))
    return y, HALF[out_dt] * np.abs(y) + 1.01 * (32 + 2 * half // 32 + 24) * 2.0 ** -24 * terms + 1e-37
