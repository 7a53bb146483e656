"""What of rotary rows, forked and packed pages, shared prefixes and verified drafts needs no device: sizes, tables of frequencies, checks of arguments."""
import math

import numpy as np
import pytest

from caten_amd import _lib, ops


def test_workspaces():
    lib = _lib.load()
    for dh in (32, 64, 128):
        for rows, h in ((0, 0), (1, 12), (700, 64)):
            assert lib.cthip_sdpa_shared_paged_q4_workspace(rows, h, dh) == 4 * (4096 + 131072 * (dh + 2) + 2 * rows * h)
    assert lib.cthip_sdpa_shared_paged_q4_workspace(4, 12, 80) < 0 and lib.cthip_sdpa_shared_paged_q4_workspace(-1, 12, 64) < 0
    for n in (0, 1, 500, 100001):
        assert lib.cthip_kv_compact_paged_q4_workspace(n) == 64 + 8 * n and lib.cthip_draft_verify_workspace(n) == 2048 * n
    assert lib.cthip_kv_compact_paged_q4_workspace(-1) < 0 and lib.cthip_draft_verify_workspace(-1) < 0


@pytest.mark.parametrize("dim", [0, 2, 20, 64, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_frequencies(dim, base):
    # (a power is off by less than one step of 64 bits, a division by half of one)
    f = np.array([math.pow(base, -2.0 * i / dim) for i in range(dim // 2)])
    assert np.allclose(ops.rope_frequencies(dim, base), f, rtol=2.0 ** -51, atol=0)
    assert np.allclose(ops.rope_frequencies(dim, base, factor=4.0), f / 4, rtol=2.0 ** -51, atol=0)
    got = ops.rope_frequencies(dim, base, factor=8.0, trained=8192, slow=1.0, fast=4.0)
    turns = 8192 * f / (2 * math.pi)
    assert np.allclose(got[turns >= 4], f[turns >= 4], rtol=2.0 ** -51, atol=0) and np.allclose(got[turns <= 1], f[turns <= 1] / 8, rtol=2.0 ** -51, atol=0)
    keep = (turns - 1) / 3
    between = (turns > 1) & (turns < 4)
    assert np.allclose(got[between], (f * (keep + (1 - keep) / 8))[between], rtol=1e-14, atol=0)
    if dim >= 20:
        assert between.any() and (turns >= 4).any() and (turns <= 1).any()


@pytest.mark.parametrize("args", [(-2, 1e4, 1.0, 0, 1.0, 4.0), (3, 1e4, 1.0, 0, 1.0, 4.0), (4, 0.0, 1.0, 0, 1.0, 4.0), (4, math.nan, 1.0, 0, 1.0, 4.0), (4, 1e4, 0.0, 0, 1.0, 4.0),
                                  (4, 1e4, 1.0, -1, 1.0, 4.0), (4, 1e4, 2.0, 100, 4.0, 4.0), (4, 1e4, 2.0, 100, -1.0, 4.0), (4, 1e4, 2.0, 100, 1.0, math.nan), (4, 1e4, math.inf, 0, 1.0, 4.0)])
def test_frequencies_refused(args):
    lib, out = _lib.load(), np.zeros(8)
    assert lib.cthip_rope_frequencies(out.ctypes.data, *args) == _lib.E_BAD_ARG and b"cthip_rope_frequencies" in lib.cthip_last_error()
    assert not out.any()


def test_frequencies_without_a_place():
    assert _lib.load().cthip_rope_frequencies(None, 4, 1e4, 1.0, 0, 1.0, 4.0) == _lib.E_BAD_ARG and _lib.load().cthip_rope_frequencies(None, 0, 1e4, 1.0, 0, 1.0, 4.0) == 0


def test_shapes_refused():
    z = np.zeros
    for args in ((z((2, 3, 8)), z((3, 1, 8)), [0, 1], z(4)), (z((2, 3, 8)), z((2, 1, 4)), [0, 1], z(4)), (z((2, 3, 8)), None, [0], z(4)), (z((2, 24)), None, [0, 1], z(4))):
        with pytest.raises(ValueError):
            ops.rope_rows(*args)
    with pytest.raises(KeyError):
        ops.rope_rows(z((2, 3, 8)), None, [0, 1], z(4), layout="other")
    for args in ((z((3, 5)), z((3, 4)), z(3), z(3), [0, 3]), (z((3, 5)), None, z(2), z(3), [0, 3]), (z((3, 5)), None, z(3), z(2), [0, 3]), (z(5), None, z(5), z(5), [0, 3]),
                 (z((3, 5)), None, z(3), z(3), [])):
        with pytest.raises(ValueError):
            ops.draft_verify(*args)
    with pytest.raises(ValueError):
        ops.draft_verify(z((3, 5)), None, z(3), z(3), [0, 3], lens=[1, 2])
    with pytest.raises(ValueError):
        ops.draft_verify(z((3, 5)), None, z(3), z(3), [0, 3], positions=[1, 2])


def test_not_initialised():
    """Without a device every entry says so and touches nothing."""
    if _lib.is_initialised():
        pytest.skip("a device is in use")
    lib = _lib.load()
    calls = [lambda: lib.cthip_rope_rows(None, 0, None, 0, None, 0, None, 0, None, 0, 0, 0, 0, 0, 0, None, 1.0),
             lambda: lib.cthip_kv_fork_paged_q4(None, 1, None, 0, None, None, None, None, 0, 0, None, None, None, 0, None, None, 1, 64),
             lambda: lib.cthip_kv_compact_paged_q4(None, None, None, None, None, 0, 0, None, 1, None, 0, 1, 64, None),
             lambda: lib.cthip_sdpa_shared_paged_q4(None, None, 64, None, None, 0, None, 1, None, None, 0, 0, None, None, 0, 1, 1, 64, None),
             lambda: lib.cthip_draft_verify(None, None, None, None, 8, None, 8, None, None, None, None, None, 0, 0, 8, None)]
    for call in calls:
        assert call() == _lib.E_NOT_INIT
