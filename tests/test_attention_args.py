"""What the attention entry points refuse before they reach the device: the Python layer on host tensors, the C layer on sizes (no GPU needed)."""
import ctypes

import pytest
import torch

from patchaugnet_amd import _lib, attention


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        _lib.build()
    return _lib.lib()


def test_host_tensors_are_refused():
    q, k = torch.zeros(1, 4, 2, 32), torch.zeros(1, 4, 1, 32)
    table, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for f in (lambda: attention.qk_norm_rotary(q, k), lambda: attention.window_attention(q, k, k),
              lambda: attention.paged_attention(q[:, 0], k, k, table, n), lambda: attention.paged_append(k, k, k, k, table, n)):
        with pytest.raises(RuntimeError, match="MI355X"):
            f()
    with pytest.raises(TypeError):
        attention.window_attention(None, k, k)


def _window(lib, dtype=0, b=1, n=4, m=4, h=2, hk=1, d=32, left=-1, right=0, sinks=0, scale=1.0, back=False):
    p, z = ctypes.c_void_p(0), (ctypes.c_void_p(0), 0, 0, 0)
    if back:
        return lib.pa_window_attention_backward(dtype, b, n, m, h, hk, d, *z, *z, *z, p, p, p, *z, left, right, sinks, scale, p, p, p, p, p, p, p)
    return lib.pa_window_attention(dtype, b, n, m, h, hk, d, *z, *z, *z, left, right, sinks, scale, p, p, p, p, p, p, p)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(b=-1), dict(n=-1), dict(m=-1), dict(m=2 ** 28 + 1), dict(h=0), dict(hk=0), dict(h=3, hk=2), dict(d=0), dict(d=12), dict(d=136),
    dict(left=-2), dict(right=-2), dict(sinks=-1), dict(left=2 ** 28 + 1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(n=2 ** 27, h=8), dict()])
def test_window_attention_sizes(lib, bad, back):
    """The last one: null tensors."""
    assert _window(lib, back=back, **bad) == -1
    assert lib.pa_last_error()


def test_paged_sizes(lib):
    p, z = ctypes.c_void_p(0), (ctypes.c_void_p(0), 0, 0, 0)

    def attend(dtype=0, b=1, h=2, hk=1, d=32, pages=4, page=16, width=2, left=-1, sinks=0, scale=1.0):
        return lib.pa_paged_attention(dtype, b, h, hk, d, p, 0, 0, *z, *z, pages, page, p, width, p, left, sinks, scale, p, p, p)

    def append(dtype=0, b=1, t=1, hk=1, d=32, pages=4, page=16, width=2):
        return lib.pa_paged_append(dtype, b, t, hk, d, *z, *z, *z, *z, pages, page, p, width, p, p, p)

    for bad in (dict(dtype=7), dict(b=-1), dict(hk=0), dict(d=20), dict(d=256), dict(pages=-1), dict(page=0), dict(width=-1), dict(width=2 ** 20, page=2 ** 9), dict()):
        assert attend(**bad) == -1, bad
        assert append(**bad) == -1, bad
    for bad in (dict(h=3, hk=2), dict(left=-2), dict(sinks=-1), dict(scale=0.0)):
        assert attend(**bad) == -1, bad
    assert append(t=-1) == -1
    assert attend(b=0) == 0 and append(b=0) == 0 and append(t=0) == 0


def test_norm_sizes(lib):
    p, z = ctypes.c_void_p(0), (ctypes.c_void_p(0), 0, 0, 0)

    def norm(dtype=0, b=1, n=1, h=1, hk=1, d=32, axes=0, per=0, ptype=0, eps=1e-6, back=False):
        if back:
            return lib.pa_qk_norm_rotary_backward(dtype, b, n, h, hk, d, *z, *z, p, p, 0, p, ptype, 0, p, axes, per, eps, 0, *z, *z, p, p, p, p, p, p)
        return lib.pa_qk_norm_rotary(dtype, b, n, h, hk, d, *z, *z, p, p, 0, p, ptype, 0, p, axes, per, eps, 0, p, p, p)

    for back in (False, True):
        for bad in (dict(dtype=3), dict(b=-1), dict(n=-1), dict(h=0, hk=0), dict(d=0), dict(d=513), dict(axes=1, per=17), dict(axes=1, per=4), dict(ptype=3),
                    dict(eps=-1.0), dict(eps=float("inf")), dict()):
            assert norm(back=back, **bad) == -1, (bad, back)
        assert norm(b=0, back=back) == 0


def test_scratch_is_bounded(lib):
    """Splits need scratch only where the rows alone do not fill the chip, and never more than 64 parts of the output."""
    f, g, w = lib.pa_paged_attention_scratch_floats, lib.pa_window_attention_scratch_floats, lib.pa_window_attention_backward_scratch_floats
    assert f(1, 8, 2, 64, 16, 7, -1, 0) == 0                                        # 112 tokens: one run
    assert f(4, 8, 2, 64, 64, 256, -1, 0) > 0
    assert f(4, 8, 2, 64, 64, 256, 100, 4) == 0                                     # the window is short, whatever the cache's length
    assert g(32, 1024, 1024, 8, 8, 64, 64, 0, 4) == 0
    assert 0 < g(1, 16, 16384, 8, 8, 64, -1, 0, 0) <= 64 * 16 * 8 * (64 + 2)
    assert w(1, 64, 64, 8, 8, 64, -1, 0, 0) >= 64 * 8
    assert f(0, 8, 2, 64, 16, 7, -1, 0) == 0 and g(1, 0, 4, 2, 1, 32, 0, 0, 0) == 0


def test_misaligned_addresses_are_refused(lib):
    """Rows that do not start at multiples of 16 bytes (host addresses: the call ends before anything is launched)."""
    buf = (ctypes.c_char * 4096)()
    base = (ctypes.addressof(buf) + 15) // 16 * 16
    p, z = ctypes.c_void_p(0), (ctypes.c_void_p(base), 0, 32, 32)
    at, off = ctypes.c_void_p(base), (ctypes.c_void_p(base + 8), 0, 32, 32)
    skew = (ctypes.c_void_p(base), 0, 34, 32)
    for bad in (off, skew):
        assert lib.pa_window_attention(0, 1, 1, 1, 1, 1, 32, *bad, *z, *z, -1, 0, 0, 1.0, p, p, at, p, p, at, p) == -1
        assert b"16 bytes" in lib.pa_last_error()
        assert lib.pa_window_attention_backward(0, 1, 1, 1, 1, 1, 32, *z, *bad, *z, at, p, at, *z, -1, 0, 0, 1.0, p, p, at, at, at, at, p) == -1
        assert lib.pa_paged_attention(0, 1, 1, 1, 32, at, 0, 32, *bad, *z, 1, 1, at, 1, at, -1, 0, 1.0, at, at, p) == -1
        assert lib.pa_paged_append(0, 1, 1, 1, 32, *bad, *z, *z, *z, 1, 1, at, 1, at, p, p) == -1
        assert b"16 bytes" in lib.pa_last_error()


def test_backward_scratch_holds_what_the_launches_touch(lib):
    """Host arithmetic over small sizes, none of them left out: no queries, no keys, one of each; first tokens with and without rows behind their window."""
    plan, promise = lib.pa_window_attention_backward_plan_floats, lib.pa_window_attention_backward_scratch_floats
    plan.argtypes, plan.restype = [ctypes.c_int] * 11, ctypes.c_long
    for n in (0, 1, 2, 63, 700):
        for m in (0, 1, 5, 129, 900):
            for h, hk in ((1, 1), (4, 2), (40, 1)):
                for left, right in ((-1, 0), (0, 0), (3, 0), (200, 20)):
                    for sinks in (0, 1, 33, 2000):
                        for d in (8, 128):
                            for dtype in (0, 1, 2):
                                for started in (0, 1):
                                    case = (dtype, 2, n, m, h, hk, d, left, right, sinks, started)
                                    assert plan(*case) <= promise(*case[1:-1]), case


def test_more_threads_than_a_launch_holds_are_refused(lib):
    """Before anything runs (host addresses: the calls end there)."""
    buf = (ctypes.c_char * 4096)()
    base = (ctypes.addressof(buf) + 15) // 16 * 16
    p, at, z = ctypes.c_void_p(0), ctypes.c_void_p(base), (ctypes.c_void_p(base), 0, 8, 8)
    n = 2 ** 28
    assert lib.pa_window_attention(2, 8, n, 4, 2, 1, 8, *z, *z, *z, -1, 0, 0, 1.0, p, p, at, p, p, at, p) == -1                # 2^32 rows
    assert b"workgroups" in lib.pa_last_error()
    assert lib.pa_window_attention_backward(2, 8, n, 4, 2, 1, 8, *z, *z, *z, at, p, at, *z, -1, 0, 0, 1.0, p, p, at, at, at, at, p) == -1
    assert b"workgroups" in lib.pa_last_error()
    assert lib.pa_window_attention_backward(0, 8, 4, n, 1, 1, 8, *z, *z, *z, at, p, at, *z, 0, 0, 0, 1.0, p, p, at, at, at, at, p) == -1      # 2^31 keys
    assert b"workgroups" in lib.pa_last_error()
    assert lib.pa_paged_attention(0, 2 ** 24, 1, 1, 8, at, 0, 8, *z, *z, 1, 1, at, 1, at, -1, 0, 1.0, at, at, p) == -1
    assert b"workgroups" in lib.pa_last_error()


def test_first_tokens_behind_the_last_key_ask_for_no_splits(lib):
    """`sinks` beyond the keys means all of them, also where the work is cut."""
    g = lib.pa_window_attention_scratch_floats
    for n, m in ((64, 64), (3, 1000), (1, 5000), (40, 0)):
        for left in (-1, 0, 16, 300):
            assert g(1, n, m, 8, 8, 32, left, 0, 10 ** 6) == g(1, n, m, 8, 8, 32, left, 0, m), (n, m, left)
    assert g(1, 64, 64, 8, 8, 32, 16, 0, 10 ** 6) == 0


def test_scales_that_leave_32_bits_are_refused(lib):
    """The kernels multiply scores by scale log2(e) in 32 bits; in Python as a ValueError, whatever the number."""
    buf = (ctypes.c_char * 4096)()
    base = (ctypes.addressof(buf) + 15) // 16 * 16
    p, at, z = ctypes.c_void_p(0), ctypes.c_void_p(base), (ctypes.c_void_p(base), 0, 32, 32)
    for scale in (3e38, 2.4e38):
        assert lib.pa_window_attention(0, 1, 1, 1, 1, 1, 32, *z, *z, *z, -1, 0, 0, scale, p, p, at, p, p, at, p) == -1
        assert lib.pa_window_attention_backward(0, 1, 1, 1, 1, 1, 32, *z, *z, *z, at, p, at, *z, -1, 0, 0, scale, p, p, at, at, at, at, p) == -1
        assert lib.pa_paged_attention(0, 1, 1, 1, 32, at, 0, 32, *z, *z, 1, 1, at, 1, at, -1, 0, scale, at, at, p) == -1
    for scale in (3e38, 1e300, 1e-50, 0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            attention._scale("x", scale, 32)
    assert attention._scale("x", None, 64) == 0.125 and attention._scale("x", 1e38, 64) == 1e38
