"""GPU tests of the rotation's angles against frequencies computed in 60 decimal digits.

x = (1, 0) and (0, 1) in fp32 give cos and sin themselves.  Tolerance: the turn's fraction becomes
fp32 in two halves, which rounds twice (relative 2^-24 each of the angle in (-pi, pi], so |angle| 2^-23
of cos and sin), sincospi is within 2 ulp and the product with the magnitude within half a step (2^-22 + 2^-24 of
the value; exact where cos or sin is 0), and the table's frequencies, four roundings of 2^-64 each
and half a step of 2^-64 turns, leave |position| f 2^-61 + |position| 2^-62 rad (of a 64-bit
mantissa)."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

pytestmark = pytest.mark.gpu
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


@pytest.fixture(scope="module")
def vk(cuda_ok):
    import vulcan_b200
    vulcan_b200.load()
    return vulcan_b200


def frequencies(dim, theta, scaling=None, factor=1.0, original_len=0.0, low=1.0, high=32.0):
    getcontext().prec = 60
    f = [(-(Decimal(theta).ln()) * 2 * i / dim).exp() for i in range(dim // 2)]
    factor, low, high = Decimal(factor), Decimal(low), Decimal(high)
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "by_wavelength":
        share = [min(max((Decimal(original_len) * x / (2 * PI) - low) / (high - low), Decimal(0)), Decimal(1)) for x in f]
        return [(1 - s) * x / factor + s * x for x, s in zip(f, share)]
    if scaling == "by_parts":
        def pair_of(turns):
            return dim * (Decimal(original_len) / (2 * PI * turns)).ln() / (2 * Decimal(theta).ln())
        first, last = max(math.floor(pair_of(high)), 0), min(math.ceil(pair_of(low)), dim - 1)
        share = [min(max(Decimal(i - first) / (last - first), Decimal(0)), Decimal(1)) for i in range(dim // 2)]
        return [x * (1 - s) + x / factor * s for x, s in zip(f, share)]
    return f


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dim,theta,scaling", [
    (128, 10000.0, {}), (64, 1e6, {}), (256, 5e5, {}), (2, 10000.0, {}), (64, 10000.0, dict(scaling="linear", factor=3.0)),
    (128, 5e5, dict(scaling="by_wavelength", factor=8.0, original_len=8192, low=1.0, high=4.0)),
    (64, 10000.0, dict(scaling="by_parts", factor=40.0, original_len=4096, magnitude=1.0)),
    (64, 10000.0, dict(scaling="by_parts", factor=4.0, original_len=65536, magnitude=1.0))])
def test_angles(vk, layout, dim, theta, scaling):
    """From one position, where slow pairs turn by 10^-7, to the ends of int32."""
    pos = [0, 1, 2, 3, 17, 1000, 4097, 131071, (1 << 20) + 3, (1 << 24) + 1, (1 << 30) + 7, (1 << 31) - 1, -1, -5, -99999, -(1 << 31)]
    rope = vk.RotaryEmbedding(dim, theta=theta, layout=layout, **scaling)
    f = frequencies(dim, theta, **{k: v for k, v in scaling.items() if k != "magnitude"})
    for a, b in zip(rope.frequencies()[0], f):
        assert abs(Decimal(a) / b - 1) < Decimal(2) ** -52
    n = dim // 2
    angle = torch.empty(len(pos), n, dtype=torch.float64)
    for i, p in enumerate(pos):
        for j, x in enumerate(f):
            turns = p * x / (2 * PI)
            angle[i, j] = float((turns - turns.to_integral_value()) * 2 * PI)
    x = torch.zeros(len(pos), 2, dim)
    ia, ib = (slice(0, n), slice(n, dim)) if layout == "half" else (slice(0, dim, 2), slice(1, dim, 2))
    x[:, 0, ia] = 1
    x[:, 1, ib] = 1
    y = rope.apply(x.cuda(), torch.tensor(pos, dtype=torch.int32, device="cuda")).cpu().double()
    p = torch.tensor(pos, dtype=torch.float64).abs()[:, None]
    ff = torch.tensor([float(v) for v in f], dtype=torch.float64)
    off = angle.abs() * 2.0 ** -23 + p * ff * 2.0 ** -61 + p * 2.0 ** -62
    for got, want in ((y[:, 0, ia], angle.cos()), (y[:, 0, ib], angle.sin()), (y[:, 1, ia], -angle.sin()), (y[:, 1, ib], angle.cos())):
        bound = off + want.abs() * (2.0 ** -22 + 2.0 ** -24) + 2.0 ** -52 * angle.abs()
        err = (got - want).abs()
        assert (err <= bound).all(), "worst %.3g of its bound" % (err / bound.clamp(min=1e-300)).max()
