"""How many digits linear attention in pieces (include/h3lm.h, lin_attention) has: its arithmetic restated in numpy, with operands as sums of
bfloat16 parts, the limits that its errors are held to, and the inputs they are taken at."""
import numpy as np

import lm_reference as lm

F = np.float32
PARTS = {"BF16": 1, "F16": 2, "F32": 3}              # of an input, exact

# A value's error against 64 bits, as the root of its mean square over that of the results. A rounding of a float32 sum is off by up to half a step,
# 2^-24 of it, 2^-24 / sqrt(3) in the mean, and R of them add up as squares: sqrt(R / 3) 2^-24. Of up to 700 tokens in pieces of 32 and up to
# 256 features of keys a float32 result meets 6 products of parts for each 32 features twice (96), those of a piece's values (6), up to 22
# updates of the state of 7 roundings each, of which those before a half of it weigh less than a half (about 80), and six factors: below
# 192, so 8 times 2^-24. A state meets its updates alone. (Two parts are off by up to 2^-18 a term.)
FULL = 2.0 ** -21
# 16-bit inputs, float32 results: states and weights as two parts, a term off by up to 2^-18 for either and for the product that is left out
HELD = 2.0 ** -17

DECAYS = np.array([0.004, 0.03, 0.2], np.float32)
COUNTS = [700, 40, 100, 300]
SHAPES = [(64, 64), (128, 128), (96, 100), (32, 64), (192, 64), (256, 256)]


def error(got, want):
    return np.sqrt(((got - want) ** 2).mean() / (want ** 2).mean())


def nearest(x):
    return lm.from_bits(lm.to_bits(x, "BF16"), "BF16")


def cut(x):
    return (np.ascontiguousarray(x, F).view(np.uint32) & np.uint32(0xffff0000)).view(F).reshape(np.shape(x))


def split(x, n):
    """x as n bfloat16 parts: to the nearest, three of them exact."""
    if n == 1:
        return [nearest(x)]
    if n == 2:
        return [nearest(x), nearest(x - nearest(x))]
    return [cut(x), cut(x - cut(x)), nearest(x - cut(x) - cut(x - cut(x)))]


def products(acc, a, b, limit):
    """acc + a b of the parts, 32 terms in one float32 step, without those of places `limit` and on together."""
    for u in range(0, a[0].shape[1], 32):
        for y, ay in enumerate(a):
            for z, bz in enumerate(b):
                if y + z < limit:
                    acc = (acc + ay[:, u:u + 32].astype(np.float64) @ bz[u:u + 32].astype(np.float64)).astype(F)
    return acc


def pieces(q, k, v, decay, dt, held=None, taken=3, inputs=None):
    """One head of one sequence from an empty state on: out and the state. held: the parts of a state and of a piece's products as operands; taken:
    of the decayed values that the state takes up; inputs: of q, k and v (None: as the kernel has them)."""
    inputs, held = inputs or PARTS[dt], held or (3 if dt == "F32" else 2)
    n, dk = q.shape
    size, scale = 64 if dt == "BF16" and dk <= 128 else 32, F(dk ** -0.5)
    fade = lambda steps: np.exp2((F(-decay * F(1.4426950408889634)) * steps).astype(F).astype(np.float64)).astype(F)  # noqa: E731
    out, s, at = np.zeros((n, v.shape[1]), F), np.zeros((dk, v.shape[1]), F), np.arange(size)
    for c in range(0, n, size):
        m = min(size, n - c)
        none = size - m                              # a short piece's tokens stand at its end
        qq, kk, vv = (np.concatenate([np.zeros((none, x.shape[1]), F), x[c:c + m]]) for x in (q, k, v))
        qp, kp, vp = split(qq, inputs), split(kk.T.copy(), inputs), split(vv, inputs)
        steps = at[:, None] - at
        p = products(np.zeros((size, size), F), qp, kp, 3) * np.where(steps >= 0, fade(np.maximum(steps, 0)), 0).astype(F) * scale
        o = products(np.zeros(vv.shape, F), qp, split(s, held), held) * (fade(np.maximum(at + 1 - none, 0)) * scale)[:, None]
        out[c:c + m] = products(o, split(p, held), vp, held)[none:]
        s = (s * (1 + np.expm1(-np.float64(decay) * m))).astype(F)
        s = products(s, kp, split(vv * fade(size - 1 - at)[:, None], taken), 3)
    return out, s
