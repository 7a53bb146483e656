"""Captured steps of a batch over the 4-bit paged cache of which some sequences are refused."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_paged_q4 import PAGE, attention, close, quantised

pytestmark = pytest.mark.gpu


def test_a_replayed_step_that_refuses_a_sequence():
    """No page is left for two of four sequences: the others go on, the two stay as they were, in lengths, pages and the pool's bytes, and
    a later replay of the same graph, with pages given back, takes their rows."""
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(31)
    stream = C.c_void_p(lib.cthip_stream())
    n, H, kv, dh, table, n_pages = 4, 4, 2, 64, 4, 16
    lens0 = [2 * PAGE, 70, PAGE, 33]  # the first and the third need a page for one more row
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    d = {k: ops.DeviceArray.from_numpy(np.asarray(v, np.int32)) for k, v in dict(lens=[0] * n, tables=np.full((n, table), -1), free=rng.permutation(n_pages), n=[6], new=lens0, one=[1] * n).items()}
    o = {k: ops.DeviceArray((m,), np.int32) for k, m in dict(slots=400, positions=400, starts=n + 1, refused=1).items()}
    w = (H + 2 * kv) * dh
    qkv, out = ops.DeviceArray((400, w), np.float32), ops.DeviceArray((400, H, dh), np.float32)

    def step(new, rows):
        _lib.check(lib.cthip_kv_plan_paged(o["slots"].ptr, o["positions"].ptr, o["starts"].ptr, d["tables"].ptr, table, d["lens"].ptr, d["n"].ptr, o["refused"].ptr, d["lens"].ptr, new.ptr, n,
                                           d["free"].ptr, d["n"].ptr, rows))
        _lib.check(lib.cthip_kv_append_paged_q4(cache.k.ptr, cache.v.ptr, qkv.ptr + 4 * H * dh, qkv.ptr + 4 * (H + kv) * dh, w, w, o["slots"].ptr, rows, n_pages, kv, dh))
        _lib.check(lib.cthip_sdpa_paged_q4(out.ptr, qkv.ptr, w, cache.k.ptr, cache.v.ptr, n_pages, d["tables"].ptr, table, d["lens"].ptr, o["starts"].ptr, n, rows, H, kv, dh,
                                           cache.workspace.ptr))

    def feed(rows):
        x = rng.normal(0, 1, (rows, w)).astype(np.float32)
        _lib.check(lib.cthip_h2d(qkv.ptr, x.ctypes.data, x.nbytes))
        k, v = (quantised(x[:, (H + a) * dh:(H + a + kv) * dh].reshape(rows, kv, dh)) for a in (0, kv))
        return x[:, :H * dh].reshape(rows, H, dh), k, v

    _, k, v = feed(sum(lens0))
    step(d["new"], 400)
    assert o["refused"].numpy()[0] == 0 and d["n"].numpy()[0] == 0
    at = np.concatenate([[0], np.cumsum(lens0)])
    held = [[x[at[i]:at[i + 1]] for x in (k, v)] for i in range(n)]
    graph, run = C.c_void_p(), C.c_void_p()
    assert lib.hipStreamBeginCapture(stream, 1) == 0
    step(d["one"], n)
    assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for replay, pages in enumerate((0, 0, 5, 0)):
        if pages:  # given back by a sequence that has left
            x = np.array([pages], np.int32)
            _lib.check(lib.cthip_h2d(d["n"].ptr, x.ctypes.data, 4))
            free = np.setdiff1d(np.arange(n_pages), d["tables"].numpy())[:pages].astype(np.int32)
            _lib.check(lib.cthip_h2d(d["free"].ptr, free.ctypes.data, free.nbytes))
        before = d["lens"].numpy(), d["tables"].numpy()
        rows_before = [cache.rows([before[1][i, t // PAGE] * PAGE + t % PAGE for t in range(before[0][i])]) for i in range(n)]
        q, k, v = feed(n)
        assert lib.hipGraphLaunch(run, stream) == 0
        got, positions, lens = out.numpy()[:n], o["positions"].numpy()[:n], d["lens"].numpy()
        refused = [0, 2] if replay < 2 else []
        assert o["refused"].numpy()[0] == len(refused) and list(np.flatnonzero(positions < 0)) == refused
        for i in range(n):
            if i not in refused:
                held[i] = [np.concatenate([a, b[i:i + 1]]) for a, b in zip(held[i], (k, v))]
            close(got[i:i + 1], *attention(q[i:i + 1], *held[i]))  # (of a refused one: over the keys that it holds)
            assert lens[i] == len(held[i][0])
        for i in refused:
            assert np.array_equal(d["tables"].numpy()[i], before[1][i])
            again = cache.rows([before[1][i, t // PAGE] * PAGE + t % PAGE for t in range(before[0][i])])
            assert all(np.array_equal(a, b) for a, b in zip(again, rows_before[i]))
    lib.hipGraphExecDestroy(run)
    lib.hipGraphDestroy(graph)
