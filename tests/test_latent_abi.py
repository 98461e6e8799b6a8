"""CPU tests of the rotary and latent-cache entry points: refusals on the host
before any device call, and the scaled frequencies against their formulas."""
import ctypes
import math

import pytest

from vulcan_b200 import _lib

FAKE = 0x10000  # an aligned address that no refused call touches


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _rotary_cfg(rotary_dim=64, layout=0, scaling=0, theta=10000.0, factor=1.0, original=0.0, low=1.0, high=32.0, magnitude=0.0):
    return _lib.VkRotaryCfg(rotary_dim, layout, scaling, 0, theta, factor, original, low, high, magnitude)


def _frequencies(lib, cfg):
    f = (ctypes.c_double * 128)()
    m = ctypes.c_double()
    assert lib.vk_rotary_frequencies(ctypes.byref(cfg), f, ctypes.byref(m)) == _lib.VK_OK
    return list(f)[:cfg.rotary_dim // 2], m.value


def test_latent_pool_refusals(lib):
    out = ctypes.c_void_p()

    def create(layers=1, latent=512, rope=64, page=16, pages=4, dtype=0, mem=None, nbytes=0):
        cfg = _lib.VkLatentCfg(layers, latent, rope, page, pages, 0, dtype)
        return lib.vk_latent_pool_create(ctypes.byref(cfg), mem, nbytes, ctypes.byref(out))

    assert lib.vk_latent_pool_create(None, None, 0, ctypes.byref(out)) == _lib.VK_INVALID_ARG
    assert create(layers=0) == _lib.VK_INVALID_ARG
    assert create(pages=0) == _lib.VK_INVALID_ARG
    assert create(dtype=2) == _lib.VK_INVALID_ARG  # fp32 pages
    for latent in (0, 64, 192, 640):
        assert create(latent=latent) == _lib.VK_UNSUPPORTED
    for rope in (0, 8, 24, 80):
        assert create(rope=rope) == _lib.VK_UNSUPPORTED
    for page in (0, 8, 48, 128):
        assert create(page=page) == _lib.VK_UNSUPPORTED
    assert create(layers=64, pages=1 << 24, page=64) == _lib.VK_UNSUPPORTED  # 2^36 rows
    assert create(mem=0x1001, nbytes=1 << 30) == _lib.VK_INVALID_ARG         # misaligned
    assert create(mem=0x100000, nbytes=100) == _lib.VK_INVALID_ARG           # too small
    assert not out.value


def test_latent_calls_without_a_pool(lib):
    assert lib.vk_latent_append(None, 0, FAKE, 512, FAKE, 64, None, 0.0, None, FAKE, 1, FAKE, None, 1, 1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_latent_decode(None, 0, FAKE, 512, 512, FAKE, 64, 64, FAKE, None, FAKE, 1, FAKE, 1, 1, 1, 1.0, FAKE, 1 << 30,
                                None) == _lib.VK_INVALID_ARG
    assert lib.vk_latent_prefill(None, 0, FAKE, 192, 192, FAKE, 512, FAKE, FAKE, 1, FAKE, None, 1, 1, 1, 16, 1, 0.0, FAKE, 1 << 30,
                                 None) == _lib.VK_INVALID_ARG
    assert lib.vk_latent_decode_workspace_size(None, 1, 1, 1) == 0
    assert lib.vk_latent_prefill_workspace_size(None, 1, 1, 1) == 0


def test_rotary_cfg_refusals(lib):
    out = ctypes.c_void_p()
    bad = [dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=258), dict(layout=2), dict(layout=-1), dict(scaling=4),
           dict(theta=1.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(magnitude=-1.0),
           dict(magnitude=float("nan")), dict(scaling=1, factor=0.0), dict(scaling=1, factor=float("inf")),
           dict(scaling=1, factor=0.1),                      # a pair would turn by more than half a turn a position
           dict(scaling=2, factor=4.0), dict(scaling=2, factor=4.0, original=4096, low=4.0, high=4.0),
           dict(scaling=3, factor=4.0, original=4096, low=0.0, high=4.0)]
    for kw in bad:
        cfg = _rotary_cfg(**kw)
        assert lib.vk_rotary_create(ctypes.byref(cfg), ctypes.byref(out)) == _lib.VK_INVALID_ARG, kw
        assert not out.value
    assert lib.vk_rotary_create(None, ctypes.byref(out)) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_destroy(None) == _lib.VK_OK


def test_rotary_apply_refusals(lib):
    out = ctypes.c_void_p()
    cfg = _rotary_cfg()
    assert lib.vk_rotary_create(ctypes.byref(cfg), ctypes.byref(out)) == _lib.VK_OK
    view = lambda x=FAKE, y=FAKE + 4096, xt=128, xh=64, yt=128, yh=64, heads=2: _lib.VkRotaryView(x, y, xt, xh, yt, yh, heads)  # noqa: E731
    v = view()
    assert lib.vk_rotary_apply(None, 0, v, None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_apply(out, 7, v, None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG    # dtype
    assert lib.vk_rotary_apply(out, 0, None, None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_apply(out, 0, v, None, 62, FAKE, 1, None) == _lib.VK_INVALID_ARG    # head_dim < rotary_dim
    assert lib.vk_rotary_apply(out, 0, v, None, 64, FAKE, -1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_apply(out, 0, v, None, 64, None, 1, None) == _lib.VK_INVALID_ARG    # positions
    assert lib.vk_rotary_apply(out, 0, view(x=None), None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_apply(out, 0, view(x=FAKE + 1), None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_apply(out, 2, view(x=FAKE + 2), None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_apply(out, 0, view(heads=-1), None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG
    assert lib.vk_rotary_apply(out, 0, view(y=FAKE, yt=256), None, 64, FAKE, 1, None) == _lib.VK_INVALID_ARG  # in place, other strides
    assert lib.vk_rotary_apply(out, 0, v, None, 64, None, 0, None) == _lib.VK_OK             # nothing to do
    assert lib.vk_rotary_apply(out, 0, view(heads=0), None, 64, None, 5, None) == _lib.VK_OK
    lib.vk_rotary_destroy(out)


def test_rotary_outputs_that_share_elements(lib):
    out = ctypes.c_void_p()
    cfg = _rotary_cfg()
    assert lib.vk_rotary_create(ctypes.byref(cfg), ctypes.byref(out)) == _lib.VK_OK

    def apply(yt, yh, heads=2, tokens=3, in_place=False):
        v = _lib.VkRotaryView(FAKE, FAKE if in_place else FAKE + (1 << 20), yt if in_place else 128, yh if in_place else 64, yt, yh,
                              heads)
        # without positions a call whose strides pass is refused for that instead
        status = lib.vk_rotary_apply(out, 0, v, None, 64, None, tokens, None)
        assert status == _lib.VK_INVALID_ARG
        return b"share" in lib.vk_last_error_string()

    for in_place in (False, True):
        for yt, yh in ((128, 0), (0, 64), (0, 0), (64, 64), (127, 64), (96, 64), (128, 63), (63, 256), (64, 191)):
            assert apply(yt, yh, in_place=in_place), (yt, yh)
        for yt, yh in ((128, 64), (1024, 72), (64, 192), (72, 300), (-128, 64), (128, -64)):
            assert not apply(yt, yh, in_place=in_place), (yt, yh)
    assert not apply(0, 64, tokens=1) and not apply(64, 0, heads=1)
    assert apply(0, 0, tokens=1) and apply(0, 0, heads=1)
    lib.vk_rotary_destroy(out)


@pytest.mark.parametrize("rotary_dim", [2, 64, 128, 256])
def test_frequencies_plain_and_linear(lib, rotary_dim):
    f, m = _frequencies(lib, _rotary_cfg(rotary_dim))
    want = [10000.0 ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    assert m == 1.0 and all(abs(a / b - 1) < 1e-14 for a, b in zip(f, want))
    f, m = _frequencies(lib, _rotary_cfg(rotary_dim, scaling=1, factor=4.0, magnitude=1.5))
    assert m == 1.5 and all(abs(a * 4 / b - 1) < 1e-14 for a, b in zip(f, want))


def test_frequencies_by_parts(lib):
    """Fast pairs keep their frequency, slow ones are divided, with a linear ramp over the pair index between."""
    d, theta, length, factor, low, high = 128, 10000.0, 4096.0, 8.0, 1.0, 32.0
    f, m = _frequencies(lib, _rotary_cfg(d, scaling=2, factor=factor, original=length, low=low, high=high))
    assert abs(m - (0.1 * math.log(factor) + 1)) < 1e-15
    first = math.floor(d * math.log(length / (high * 2 * math.pi)) / (2 * math.log(theta)))
    last = math.ceil(d * math.log(length / (low * 2 * math.pi)) / (2 * math.log(theta)))
    assert 0 < first < last < d // 2
    for i, got in enumerate(f):
        plain = theta ** (-2.0 * i / d)
        ramp = min(max((i - first) / (last - first), 0.0), 1.0)
        assert abs(got / (plain * (1 - ramp) + plain / factor * ramp) - 1) < 1e-13
    assert f[0] == 1.0 and abs(f[-1] * factor / theta ** (-2.0 * (d // 2 - 1) / d) - 1) < 1e-13
    # a context factor of one changes nothing
    g, m = _frequencies(lib, _rotary_cfg(d, scaling=2, factor=1.0, original=length))
    assert m == 1.0 and all(abs(a / theta ** (-2.0 * i / d) - 1) < 1e-13 for i, a in enumerate(g))


def test_frequencies_by_wavelength(lib):
    d, theta, length, factor, low, high = 128, 500000.0, 8192.0, 8.0, 1.0, 4.0
    f, m = _frequencies(lib, _rotary_cfg(d, scaling=3, theta=theta, factor=factor, original=length, low=low, high=high))
    assert m == 1.0
    kinds = set()
    for i, got in enumerate(f):
        plain = theta ** (-2.0 * i / d)
        turns = length * plain / (2 * math.pi)
        if turns >= high:
            want, kind = plain, "kept"
        elif turns <= low:
            want, kind = plain / factor, "divided"
        else:
            s = (turns - low) / (high - low)
            want, kind = (1 - s) * plain / factor + s * plain, "blended"
        kinds.add(kind)
        assert abs(got / want - 1) < 1e-13, i
    assert kinds == {"kept", "blended", "divided"}


def test_python_refusals_without_a_gpu():
    import vulcan_b200 as vk
    with pytest.raises(ValueError):
        vk.RotaryEmbedding(64, layout="other")
    with pytest.raises(ValueError):
        vk.RotaryEmbedding(64, scaling="other")
    with pytest.raises(vk.VKError):
        vk.RotaryEmbedding(63)
    import torch
    with pytest.raises(TypeError):
        vk.LatentKVPool(1, 512, 64, 4, dtype=torch.float32)
    f, m = vk.RotaryEmbedding(64, theta=10000.0).frequencies()
    assert len(f) == 32 and f[0] == 1.0 and m == 1.0


def test_scheduler_counts_a_pools_own_page_size():
    from vulcan_b200.scheduler import PagedKVScheduler

    class Pool:
        page_bytes, page_tokens = 4, 64

        def __init__(self):
            self.left = list(range(6))

        def pages_available(self):
            return len(self.left)

        def alloc(self, n):
            got, self.left = self.left[:n], self.left[n:]
            return got

        def free(self, ids):
            self.left += ids

    sched = PagedKVScheduler(Pool())
    assert sched.admit(0, 130) and len(sched.seqs[0].pages) == 3
    for _ in range(62):
        assert sched.grow(0)
    assert sched.seqs[0].length == 192 and len(sched.seqs[0].pages) == 3
    assert sched.grow(0) and len(sched.seqs[0].pages) == 4
    assert PagedKVScheduler.pages_for(17) == 2
