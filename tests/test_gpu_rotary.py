"""GPU tests of vk_rotary_apply against the rotation in 64 bits.

Tolerance.  The angle's fraction of a turn is rounded to fp32 (2^-24 of half a
turn: an angle error of pi * 2^-24), sincospi is within 2 ulp (2^-22), so cos and
sin are within 2^-20 (times the magnitude m), and y = a cos - b sin within
(|a| + |b|) m 2^-20 plus three fp32 roundings, which 2^-21 (|a| + |b|) m covers.
One rounding to the type adds half a step: eps/2 of the value, or 2^-25 among
fp16's subnormals.  The frequency in 64 bits carries 2^-53, at position p an
angle of p f 2^-52 (the reference's product included)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def vk(cuda_ok):
    import vulcan_b200
    vulcan_b200.load()
    return vulcan_b200


def turned(x, positions, freqs, m, half):
    """x [tokens, heads, D] in 64 bits on the CPU, and the bound's (|a| + |b|) per element."""
    r = len(freqs)
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    ang = positions.double()[:, None] * torch.tensor(freqs, dtype=torch.float64)
    cos, sin = (ang.cos() * m)[:, None], (ang.sin() * m)[:, None]
    ia, ib = (slice(0, r), slice(r, 2 * r)) if half else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * cos - b * sin, a * sin + b * cos
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return y, size


def check(got, x, positions, rope, what=""):
    freqs, m = rope.frequencies()
    xc, pc = x.detach().cpu(), positions.cpu()
    xc = xc.reshape(-1, *xc.shape[-2:])
    want, size = turned(xc, pc, freqs, m, rope.layout == "half")
    err = (got.cpu().reshape(want.shape).double() - want).abs()
    far = pc.double().abs()[:, None, None] * max(freqs) * 2.0 ** -52
    bound = torch.finfo(x.dtype).eps / 2 * want.abs() + size * m * (2.0 ** -20 + 2.0 ** -21 + far) + 2.0 ** -25
    bound[..., rope.rotary_dim:] = 0  # copied
    assert torch.isfinite(err).all(), what
    assert (err <= bound).all(), "%s: worst %.3g of its bound" % (what, (err / bound.clamp(min=1e-30)).max())


CASES = [  # tokens, heads, kv_heads, head_dim, rotary_dim
    (1, 1, 1, 2, 2), (1, 8, 1, 64, 64), (7, 5, 1, 96, 96), (33, 3, 2, 128, 64), (64, 16, 8, 128, 128),
    (5, 2, 1, 100, 50), (9, 4, 4, 80, 24), (3, 40, 1, 256, 256), (300, 2, 1, 192, 48), (2, 300, 3, 64, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("case", CASES)
def test_rotation(vk, dtype, layout, case):
    tokens, heads, kv_heads, d, r = case
    g = torch.Generator(device="cuda").manual_seed(tokens * 1000 + d)
    q = torch.randn(tokens, heads, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(tokens, kv_heads, d, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 200000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    rope = vk.RotaryEmbedding(r, layout=layout)
    y, yk = rope.apply(q, pos, k=k)
    check(y, q, pos, rope, "q")
    check(yk, k, pos, rope, "k")
    assert torch.equal(y, rope.apply(q, pos))  # q alone, and bit for bit again


@pytest.mark.parametrize("scaling", [dict(), dict(scaling="linear", factor=3.0),
                                     dict(scaling="by_parts", factor=4.0, original_len=4096, low=1.0, high=32.0),
                                     dict(scaling="by_wavelength", factor=8.0, original_len=8192, low=1.0, high=4.0),
                                     dict(scaling="by_parts", factor=40.0, original_len=4096, low=1.0, high=32.0, magnitude=1.25)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_positions_far_and_negative(vk, layout, scaling):
    """Angles stay exact where fp32's pos * f has lost its fraction of a turn."""
    pos = torch.tensor([0, 1, 2, 4095, 4096, 131071, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -1, -100000, -(1 << 31)],
                       dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(len(pos), 3, 128, generator=g, device="cuda")
    rope = vk.RotaryEmbedding(128, layout=layout, theta=500000.0, **scaling)
    check(rope.apply(x, pos), x, pos, rope, str(scaling))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_views_in_place_and_batches(vk, dtype, layout):
    """Strided and misaligned views, part of a head, in place, a 4-D batch: the rest of the memory stays."""
    g = torch.Generator(device="cuda").manual_seed(5)
    rope = vk.RotaryEmbedding(64, layout=layout)
    pos = torch.arange(50, 50 + 22, dtype=torch.int32, device="cuda")
    # the last 64 elements of heads of 192, rotated in place
    big = torch.randn(22, 4, 192, generator=g, device="cuda").to(dtype)
    before = big.clone()
    part = big[..., 128:]
    assert rope.apply(part, pos, out=part) is part
    check(part, before[..., 128:], pos, rope, "slice in place")
    assert torch.equal(big[..., :128], before[..., :128])
    # an offset of one element: no 16-byte vectors
    flat = torch.randn(22 * 3 * 70 + 1, generator=g, device="cuda").to(dtype)
    odd = flat[1:].view(22, 3, 70)
    check(rope.apply(odd, pos), odd, pos, rope, "misaligned")
    before = flat.clone()
    rope.apply(odd, pos, out=odd)
    check(odd, before[1:].view(22, 3, 70), pos, rope, "misaligned in place")
    assert flat[0] == before[0] and torch.equal(odd[..., 64:], before[1:].view(22, 3, 70)[..., 64:])
    # heads before tokens in memory, and an output with gaps between its heads
    x = torch.randn(3, 22, 64, generator=g, device="cuda").to(dtype).transpose(0, 1)
    out = torch.full((22, 3, 80), 7.0, device="cuda").to(dtype)
    rope.apply(x, pos, out=out[..., :64])
    check(out[..., :64], x, pos, rope, "transposed")
    assert (out[..., 64:] == 7).all()
    # [batch, tokens, heads, D], and one token a sequence cut from a longer one
    x4 = torch.randn(2, 11, 3, 64, generator=g, device="cuda").to(dtype)
    y4 = rope.apply(x4, pos)
    assert y4.shape == x4.shape
    check(y4, x4, pos, rope, "4-D")
    cut = x4[:, 5:6]
    check(rope.apply(cut, pos[:2]), cut, pos[:2], rope, "one token of each")


def test_no_tokens_and_refusals(vk):
    rope = vk.RotaryEmbedding(64)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(4, 2, 64, device="cuda", dtype=torch.float16)
    assert rope.apply(x[:0], pos[:0]).shape == (0, 2, 64)
    with pytest.raises(ValueError):
        rope.apply(x, pos[:3])                       # positions
    with pytest.raises(TypeError):
        rope.apply(x, pos.long())
    with pytest.raises(TypeError):
        rope.apply(x.double(), pos)
    with pytest.raises(ValueError):
        rope.apply(x.cpu(), pos)
    with pytest.raises(ValueError):
        rope.apply(x, pos, k=x[:3])
    with pytest.raises(TypeError):
        rope.apply(x, pos, k=x.float())
    with pytest.raises(ValueError):
        rope.apply(x.transpose(1, 2), pos)           # d is not contiguous
    with pytest.raises(ValueError):
        rope.apply(x, pos, out=x[:3])
    with pytest.raises(ValueError):
        rope.apply(torch.zeros(2, 4, 2, 64, device="cuda", dtype=torch.float16)[:, :2], pos)  # batches apart
    with pytest.raises(vk.VKError):
        rope.apply(x[..., :62], pos)                 # head_dim < rotary_dim
    with pytest.raises(vk.VKError):                  # in place under other strides
        w = torch.zeros(4 * 4 * 64, device="cuda", dtype=torch.float16)
        rope.apply(w.view(4, 4, 64)[:, :2], pos, out=w[:512].view(4, 2, 64))


def test_graph_and_stream(vk):
    g = torch.Generator(device="cuda").manual_seed(9)
    rope = vk.RotaryEmbedding(128, layout="half", scaling="by_parts", factor=4.0, original_len=4096)
    x = torch.randn(16, 4, 128, generator=g, device="cuda").half()
    pos = torch.arange(16, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = rope.apply(x, pos, stream=side)
    side.synchronize()
    check(y, x, pos, rope, "side stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = rope.apply(x, pos)
    pos += 1000
    graph.replay()
    torch.cuda.synchronize()
    check(z, x, pos, rope, "replayed with new positions")
    assert math.isfinite(float(z.float().sum()))
