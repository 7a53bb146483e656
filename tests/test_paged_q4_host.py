"""Sizes and argument checks of the 4-bit paged cache and of beam search that need no device."""
import numpy as np
import pytest

from caten_amd import _lib, ops


@pytest.mark.parametrize("kv,dh", [(1, 32), (12, 64), (8, 128), (65535, 128)])
def test_page_bytes(kv, dh):
    # 64 rows of kv * dh channels: 4 bits each, and 16 for every 32
    assert _lib.load().cthip_kv_page_bytes_q4(kv, dh) == 64 * kv * dh * 9 // 16


@pytest.mark.parametrize("kv,dh", [(0, 64), (-1, 64), (65536, 64), (4, 48), (4, 0), (4, 256)])
def test_page_bytes_refused(kv, dh):
    lib = _lib.load()
    assert lib.cthip_kv_page_bytes_q4(kv, dh) < 0 and b"cthip_kv_page_bytes_q4" in lib.cthip_last_error()


def test_workspaces():
    lib = _lib.load()
    for dh in (32, 64, 128):
        assert lib.cthip_sdpa_paged_q4_workspace(dh) == 4 * (2048 + 2048 * 16 * (dh + 2))
    assert lib.cthip_sdpa_paged_q4_workspace(80) < 0
    for n, k in ((0, 1), (1, 4), (48, 8), (1000, 32)):
        assert lib.cthip_beam_select_workspace(n, k) == 256 + 4 * n + 32 * n * k * (24 + 8 * k)
    assert lib.cthip_beam_select_workspace(-1, 4) < 0 and lib.cthip_beam_select_workspace(1, 0) < 0 and lib.cthip_beam_select_workspace(1, 33) < 0


def test_shapes_refused():
    with pytest.raises(ValueError):
        ops.kv_plan([1, 2], [1], np.zeros((2, 2)), [], 3)
    with pytest.raises(ValueError):
        ops.kv_plan([1, 2], [1, 1], np.zeros((3, 2)), [], 3)
    with pytest.raises(ValueError):
        ops.kv_plan([1], [1], np.zeros((1, 2)), [4, 5], 3, n_free=3)
    with pytest.raises(ValueError):
        ops.beam_select(np.zeros((2, 3, 4)), np.zeros((2, 2)))
    with pytest.raises(ValueError):
        ops.beam_select(np.zeros((3, 4)), np.zeros((3, 4)))
    with pytest.raises(ValueError):
        ops.beam_select(np.zeros((2, 3, 4)), np.zeros((2, 3)), finished=[0, 1])
