"""CPU tests of the rotary entry points: frequencies against formulas written apart from the library, and calls whose
tensors coincide."""
import ctypes
import math

import pytest

from vulcan_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def frequencies(lib, rotary_dim, theta=10000.0, scaling=0, factor=1.0, original=0.0, low=1.0, high=32.0):
    cfg = _lib.VkRotaryCfg(rotary_dim, 0, scaling, 0, theta, factor, original, low, high, 0.0)
    f = (ctypes.c_double * 128)()
    m = ctypes.c_double()
    assert lib.vk_rotary_frequencies(ctypes.byref(cfg), f, ctypes.byref(m)) == _lib.VK_OK
    return list(f)[:rotary_dim // 2], m.value


@pytest.mark.parametrize("rotary_dim,theta,original", [(64, 1e4, 65536), (16, 1e4, 32768), (128, 1e4, 1 << 20), (64, 5e5, 1 << 22),
                                                       (64, 1e4, 4096)])
def test_by_parts_ramp_runs_to_the_pair_that_makes_low_turns(lib, rotary_dim, theta, original):
    """The ramp's end may lie behind the last pair (up to rotary_dim - 1): pairs that make more than `low` turns are
    then never divided by the whole factor."""
    factor, low, high = 4.0, 1.0, 32.0
    got, _ = frequencies(lib, rotary_dim, theta, 2, factor, original, low, high)

    def pair_of(turns):
        return rotary_dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta))

    first, last = max(math.floor(pair_of(high)), 0), min(math.ceil(pair_of(low)), rotary_dim - 1)
    if original > 4096:
        assert last > rotary_dim // 2 - 1
    for i, f in enumerate(got):
        plain = theta ** (-2.0 * i / rotary_dim)
        share = min(max((i - first) / (last - first), 0.0), 1.0)
        assert abs(f / (plain * (1 - share) + plain / factor * share) - 1) < 1e-13, i
        if original * plain / (2 * math.pi) > low and i < last:
            assert f > plain / factor * (1 + 1e-9), i
    if (rotary_dim, original) == (64, 65536):
        assert abs(got[31] / 1e4 ** (-62 / 64) - 0.3654) < 1e-3 and abs(got[28] / 1e4 ** (-56 / 64) - 0.5385) < 1e-3


@pytest.mark.parametrize("original,share", [(3.0, 1.0), (1e40, 0.0)])
def test_by_parts_ends_outside_the_pairs(lib, original, share):
    """Contexts in which no pair makes `low` turns divide every pair; where all make more than `high`, none is."""
    got, _ = frequencies(lib, 64, 1e4, 2, 8.0, original)
    for i, f in enumerate(got):
        plain = 1e4 ** (-2.0 * i / 64)
        assert abs(f / (plain / 8.0 if share else plain) - 1) < 1e-13, i


def test_one_tensor_as_q_and_k_is_refused_as_an_output(lib):
    """Where one view's output is the other's input or output, both rotate the same elements."""
    out = ctypes.c_void_p()
    cfg = _lib.VkRotaryCfg(64, 0, 0, 0, 10000.0, 1.0, 0.0, 1.0, 32.0, 0.0)
    assert lib.vk_rotary_create(ctypes.byref(cfg), ctypes.byref(out)) == _lib.VK_OK
    a, b, c, d = 0x10000, 0x20000, 0x30000, 0x40000  # addresses that no refused call touches

    def refused(q, k, heads=2, tokens=3):
        views = [_lib.VkRotaryView(x, y, 128, 64, 128, 64, heads) for x, y in (q, k)]
        # without positions a call that passes is refused for that instead
        status = lib.vk_rotary_apply(out, 0, views[0], views[1], 64, None, tokens, None)
        assert status == (_lib.VK_INVALID_ARG if tokens and heads else _lib.VK_OK)
        return b"q and k" in lib.vk_last_error_string()

    for q, k in (((a, a), (a, a)), ((a, c), (b, c)), ((a, b), (b, d)), ((a, c), (b, a)), ((a, a), (a, c)), ((a, b), (b, b)), ((a, b), (b, a))):
        assert refused(q, k), (q, k)
    for q, k in (((a, a), (b, b)), ((a, c), (b, d)), ((a, c), (a, d)), ((a, a), (b, d))):
        assert not refused(q, k), (q, k)
    lib.vk_rotary_destroy(out)
