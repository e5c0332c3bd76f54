"""The 4-bit linear layer where float32 sums show: long rows of weights with few inputs that are not zero, so that each of them is seen, and
digits of sums whose codes lie around 8."""
import numpy as np
import pytest

import lm_reference as ref
from helpers import new, up

pytestmark = pytest.mark.gpu

from sycl_minimax_h3_amd import ops  # noqa: E402


def weights(codes, scale, mins):
    """W [N, K] in float64."""
    n, half = codes.shape
    c = np.empty((n, 2 * half))
    c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
    g = 2 * half // scale.shape[1]
    s = np.repeat(scale.astype(np.float64), g, 1)
    return s * c - (8 * s if mins is None else np.repeat(mins.astype(np.float64), g, 1)), s, c


def marks(K, group, count, g):
    """`count` inputs of a row: the first and last, both sides of the borders of runs, of groups and of what a wavefront takes, and others."""
    edges = {0, K - 1, 31, 32, 127, 128, 511, 512, group - 1, group, K - 32, K - 33, K // 2, K // group // 2 * group - 1}
    edges |= {k for n in (1, 2, 3, 7, 11, 12, 22, 44) for at in (512 * n, 6144 * n, K // 12 // 512 * 512 * n) for k in (at - 1, at)}
    edges = np.array(sorted(k for k in edges if 0 <= k < K))
    return np.unique(np.concatenate([edges, g.integers(0, K, count)]))


# M, K, N, group, minima, type, scale type: rows past what the one-row kernel holds, group numbers by multiplication at long rows, every kernel
LONG = [
    (1, 20000 * 32, 5, 32, True, "BF16", "F16"),
    (1, 1 << 20, 17, 64, False, "F16", "F16"),
    (1, 25600, 40, 128, False, "BF16", "F16"),
    (1, 6144, 40, 64, True, "BF16", "F16"),             # twelve wavefronts with one, two and four chunks of 512 each, and one input run more
    (1, 6176, 40, 32, False, "F32", "F16"),
    (1, 12288, 40, 128, True, "F32", "F32"),
    (1, 24576, 40, 32, True, "F16", "F16"),
    (1, 24608, 40, 32, False, "BF16", "F16"),
    (1, 22528, 40, 64, True, "F16", "F16"),
    (1, 14336, 40, 32, True, "F32", "F32"),
    (1, 96 * 9999, 3, 96, True, "BF16", "BF16"),
    (3, 96 * 10922, 5, 96, True, "F32", "F16"),
    (7, 1 << 20, 3, 128, False, "F16", "F32"),
    (16, 32 * 7777, 20, 32 * 7, True, "BF16", "F16"),
    (40, 1 << 17, 40, 32, True, "BF16", "F16"),
    (33, 96 * 1111, 35, 96, False, "F16", "BF16"),
    (20, 1 << 18, 33, 256, True, "F32", "F16"),
]


@pytest.mark.parametrize("M,K,N,group,mins,dt,scale_dt", LONG)
def test_linear4_long_rows_one_input_at_a_time(dev, M, K, N, group, mins, dt, scale_dt):
    """Rows of x that are zero but for one input each: every output is one weight, wherever in the row it lies."""
    g = np.random.default_rng(K + M)
    codes = g.integers(0, 256, (N, K // 2), dtype=np.uint8)
    s = ref.from_bits(ref.to_bits(np.exp(g.normal(-4, 0.5, (N, K // group))), scale_dt), scale_dt)
    z = ref.from_bits(ref.to_bits(g.standard_normal((N, K // group)) * 0.1, scale_dt), scale_dt) if mins else None
    layer = ops.Int4Linear(up(dev, codes, "U8", [N, K // 2]), up(dev, ref.to_bits(s, scale_dt), scale_dt, [N, K // group]),
                           up(dev, ref.to_bits(z, scale_dt), scale_dt, [N, K // group]) if mins else None)
    W, sw, c = weights(codes, s, z)
    at = marks(K, group, 8, g)
    at = np.concatenate([at, at[:-len(at) % M]]) if M > 1 else at
    out = new(dev, "F32", [M, N])
    for i in range(0, len(at), M):
        x = np.zeros((M, K), np.float32)
        x[np.arange(M), at[i:i + M]] = 1.0
        layer.forward(up(dev, ref.to_bits(x, dt), dt, [M, K]), out)
        want = W[:, at[i:i + M]].T
        # one product of at most 31 s and one of at most 16 s + |z|, four roundings of each
        tol = 4 * 2.0 ** -24 * (32 * sw + np.abs(W) + 24 * sw)[:, at[i:i + M]].T
        off = np.abs(out.to_numpy() - want)
        assert (off <= tol).all(), (at[i:i + M][np.argwhere(off > tol)[:3, 0]], off.max())
    assert np.median(tol / np.maximum(np.abs(want), 1e-9)) < 1e-3                 # (a bound that nothing could miss would say nothing)


@pytest.mark.parametrize("M", [1, 2, 8, 20, 40])
def test_linear4_values_below_the_normal_range(dev, M):
    """Halves below 2^-14 count in full."""
    K, N, group = 1024, 48, 64
    g = np.random.default_rng(91)
    xb = ref.to_bits(g.standard_normal((M, K)) * 2e-6, "F16")
    codes = g.integers(0, 256, (N, K // 2), dtype=np.uint8)
    s = np.exp(g.normal(-4, 0.5, (N, K // group))).astype(np.float32)
    out = new(dev, "F32", [M, N])
    ops.Int4Linear(up(dev, codes, "U8", [N, K // 2]), up(dev, s, "F32", [N, K // group])).forward(up(dev, xb, "F16", [M, K]), out)
    want, tol = ref.linear4(ref.from_bits(xb, "F16"), codes, s, None, None, "F32")
    assert (np.abs(out.to_numpy() - want) <= tol).all() and np.median(tol / np.abs(want)) < 0.01


def float32_sums(x, W32, s, c, z, group):
    """The layer in float32 as its formula stands: sums of 32 products x (c - 8), each rounded, added up by groups with their scales."""
    f = np.float32
    M, K = x.shape
    y = np.zeros((M, W32.shape[0]), f)
    for k in range(0, K, 32):
        run = np.zeros_like(y)
        sx = np.zeros((M, 1), f)
        for i in range(k, k + 32):
            run += x[:, i:i + 1] * (c[:, i] - 8).astype(f)[None]
            sx += x[:, i:i + 1]
        y += s[:, k // group].astype(f)[None] * run
        if z is not None:
            y -= sx * (z[:, k // group] - f(8) * s[:, k // group]).astype(f)[None]
    return y


@pytest.mark.parametrize("M,K", [(1, 5376), (1, 14336), (3, 5376), (16, 5376), (24, 5376), (40, 5376)])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("width,mean", [(2.5, 0.0), (2.5, 3.0), (0.7, 3.0)])
def test_linear4_digits_of_float32(dev, M, K, mins, width, mean):
    """float32 x, codes in a bell around 8, x off zero: the error against 64 bits is of the size that float32 sums of the same products have."""
    N, group = 64, 64
    g = np.random.default_rng(92)
    x = (g.standard_normal((M, K)) + mean).astype(np.float32)
    c = np.clip(np.rint(g.normal(8, width, (N, K))), 0, 15).astype(np.uint8)
    codes = c[:, 0::2] | c[:, 1::2] << 4
    s = (np.exp(g.normal(-4, 0.3, (N, K // group)))).astype(np.float32)
    z = (8 * s + 0.2 * s * g.standard_normal(s.shape)).astype(np.float32) if mins else None
    out = new(dev, "F32", [M, N])
    ops.Int4Linear(up(dev, codes, "U8", [N, K // 2]), up(dev, s, "F32", [N, K // group]),
                   up(dev, z, "F32", [N, K // group]) if mins else None).forward(up(dev, x, "F32", [M, K]), out)
    W, _, cc = weights(codes, s, z)
    want = x.astype(np.float64) @ W.T
    plain = float32_sums(x, W, s, cc, z, group)
    err, other = (np.linalg.norm(y.astype(np.float64) - want) for y in (out.to_numpy(), plain))
    # both are sums of the same terms with a rounding each, in other orders: within two bits of each other
    assert err <= 4 * other, f"{err / other:.1f} times the error of float32 sums ({err / np.linalg.norm(want):.2e} of the result)"


def test_linear4_more_blocks_than_a_launch_takes(dev):
    """2^35 outputs (64 GiB): more blocks of threads than one launch has."""
    M, K, N = (1 << 17) + 70, 32, 1 << 18
    if dev.api.mem_free(dev.ctx) < 80 << 30:
        pytest.skip("needs 80 GiB of the GPU's memory")
    g = np.random.default_rng(93)
    x = g.integers(-8, 9, (M, K)).astype(np.float32)
    codes = g.integers(0, 256, (N, K // 2), dtype=np.uint8)
    s = (2.0 ** g.integers(-2, 3, (N, 1))).astype(np.float32)
    out = new(dev, "BF16", [M, N])
    ops.Int4Linear(up(dev, codes, "U8", [N, K // 2]), up(dev, s, "F32", [N, 1])).forward(up(dev, x, "F32", [M, K]), out)
    W, _, _ = weights(codes, s, None)
    for m in (0, 31, 32, 65535, 65536, 100000, (1 << 17) - 1, 1 << 17, M - 1):
        got = ref.from_bits(out._owner.read(2 * N, 2 * N * m).view(np.uint16), "BF16")
        assert np.array_equal(got, ref.from_bits(ref.to_bits((x[m] @ W.T).astype(np.float32), "BF16"), "BF16")), m
    out._owner.free()
