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
