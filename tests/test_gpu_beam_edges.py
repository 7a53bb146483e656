"""Beam search's selection and reordering at their edges, against the definitions of include/caten_hip.h in NumPy."""
import numpy as np
import pytest

from tests.test_gpu_beam import PAGE, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [1, 2, 5])
def test_infinite_scores_and_logits(K):
    """A score of infinity and a logit of infinity in one beam: the other tokens' scores, infinity less infinity, count as minus infinity."""
    from caten_amd import ops
    rng = np.random.default_rng(K)
    V = 700
    logits = rng.normal(0, 2, (3, K, V)).astype(np.float32)
    scores = np.full((3, K), -np.inf, np.float32)
    scores[0, 0] = scores[1] = scores[2, K - 1] = np.inf
    logits[0, 0, 7] = logits[1, 0, 9] = logits[1, 0, 600] = np.inf
    got = ops.beam_select(logits, scores)
    # one candidate of infinity, then beam 0's others from the highest logit down
    order = np.argsort(-logits[0, 0], kind="stable")[:K]
    assert np.array_equal(got["tokens"][0], order) and not got["parents"][0].any()
    assert got["scores"][0, 0] == np.inf and (got["scores"][0, 1:] == -np.inf).all()
    # all finite tokens of the other beams of request 1 are at infinity, behind beam 0's two in the order of beams
    best = [(0, 9), (0, 600)] + [(k, t) for k in range(1, K) for t in np.argsort(-logits[1, k], kind="stable")[:K]]
    if K > 1:
        assert [tuple(x) for x in zip(got["parents"][1], got["tokens"][1])] == best[:K] and (got["scores"][1] == np.inf).all()
    # an infinite score alone: the logits' order
    assert np.array_equal(got["tokens"][2], np.argsort(-logits[2, K - 1], kind="stable")[:K]) and (got["parents"][2] == K - 1).all()


# ------------------------------------------------------------------------------------------------------- pages given back


def free_by_hand(tables, lens, n_pages):
    used = {int(p) for row, n in zip(tables, lens) for p in row[:-(-max(int(n), 0) // PAGE)]}
    return [p for p in range(n_pages) if p not in used]


@pytest.mark.parametrize("n,table,n_pages", [(1, 1, 1), (3, 4, 0), (0, 2, 5), (5, 3, 40), (64, 20, 1024), (300, 16, 9000), (4096, 7, 30011), (2, 300, 8192), (7, 5, 8193)])
def test_free_pages(n, table, n_pages):
    print(f"case: free pages, {n} sequences of up to {table}, {n_pages} in the pool", flush=True)
    from caten_amd import ops
    rng = np.random.default_rng(n + n_pages)
    tables = rng.integers(-3, n_pages + 3, (n, table)).astype(np.int32)  # (shared by some, outside the pool, and any behind a sequence's last)
    lens = rng.integers(-2, table * PAGE + 70, n).astype(np.int32)
    lens[::4] = lens[::4] // PAGE * PAGE
    if n > 1:
        lens[0], lens[1], tables[1, -1] = 0, 2 ** 31 - 1, 2 ** 31 - 1
    got = ops.kv_free_pages(tables, lens, n_pages)
    assert np.array_equal(got, free_by_hand(tables, lens, n_pages))


def test_a_search_keeps_to_its_pages():
    """Steps of plan, reordering and pages given back, over many borders of two pages, in a pool that has what the beams hold at any
    one time and no more: no page is lost, none is in use twice, nobody is refused.  Captured, with tables and lengths going to and
    fro, and replayed: two steps a replay."""
    import ctypes as C
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(8)
    stream = C.c_void_p(lib.cthip_stream())
    n, K, kv, dh, table, steps = 2, 4, 1, 32, 8, 400
    # full pages of a request: with random parents nearly all are shared; room for a bit more than one row of pages and K last ones
    n_pages = n * (steps // PAGE + 2 * K + 2)
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    a = {k: ops.DeviceArray.from_numpy(np.asarray(v, np.int32)) for k, v in dict(lens=[0] * n * K, one=[1] * n * K, per=[0] * n, parents=np.zeros((n, K)), free=np.zeros(n_pages), n=[0]).items()}
    tables = [ops.DeviceArray.from_numpy(np.full((n * K, table), -1, np.int32)) for _ in range(2)]
    o = {k: ops.DeviceArray((m,), np.int32) for k, m in dict(slots=n * K, starts=n * K + 1, refused=1).items()}

    def step(t, u):
        _lib.check(lib.cthip_kv_free_paged(a["free"].ptr, a["n"].ptr, t.ptr, table, a["lens"].ptr, n * K, n_pages))
        _lib.check(lib.cthip_kv_plan_paged(o["slots"].ptr, None, o["starts"].ptr, t.ptr, table, a["lens"].ptr, a["n"].ptr, o["refused"].ptr, a["lens"].ptr, a["one"].ptr, n * K,
                                           a["free"].ptr, a["n"].ptr, n * K))
        _lib.check(lib.cthip_beam_reorder_paged_q4(u.ptr, None, cache.k.ptr, cache.v.ptr, 1, n_pages, t.ptr, table, a["per"].ptr, a["parents"].ptr, n, K, kv, dh, None, 0, None, None))

    def upload(d, x):
        x = np.ascontiguousarray(x, np.int32)
        _lib.check(lib.cthip_h2d(d.ptr, x.ctypes.data, x.nbytes))

    def look(t, length):
        rows, lens, left, free = t.numpy(), a["lens"].numpy(), int(a["n"].numpy()[0]), a["free"].numpy()
        assert o["refused"].numpy()[0] == 0 and (lens == length).all()
        used = {int(p) for r in rows for p in r[:-(-length // PAGE)]}
        assert all(0 <= p < n_pages for p in used) and not used & set(free[:left].tolist())
        if length % PAGE:  # the last pages are one to a beam
            assert len({int(r[length // PAGE]) for r in rows}) == n * K
        return len(used) + left

    # eager: the step's lengths and parents come from the host
    lost = 0
    for s in range(200):
        upload(a["per"], [s + 1] * n)
        upload(a["parents"], rng.integers(0, K, (n, K)))
        step(*tables)
        tables = tables[::-1]
        lost = max(lost, n_pages - look(tables[0], s + 1))
    assert lost > 0  # (between a reordering and the next call they are in nobody's hands)
    assert np.array_equal(ops.kv_free_pages(tables[0].numpy(), a["lens"].numpy(), n_pages), free_by_hand(tables[0].numpy(), a["lens"].numpy(), n_pages))
    # captured: two steps, the second back into the first's tables; lengths as high as the second's (the same page but at a border, which these keep off)
    graph, run = C.c_void_p(), C.c_void_p()
    assert lib.hipStreamBeginCapture(stream, 1) == 0
    step(*tables)
    step(*tables[::-1])
    assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for s in range(200, steps, 2):
        if (s + 1) // PAGE != (s + 2) // PAGE:
            for k in range(2):  # (across a border step by step)
                upload(a["per"], [s + k + 1] * n)
                step(*tables)
                tables = tables[::-1]
        else:
            upload(a["per"], [s + 1] * n)
            upload(a["parents"], rng.integers(0, K, (n, K)))
            assert lib.hipGraphLaunch(run, stream) == 0
        look(tables[0], s + 2)
    lib.hipGraphExecDestroy(run)
    lib.hipGraphDestroy(graph)


def test_refusals_of_free_pages():
    from caten_amd import HipError, _lib, ops
    lib = _lib.init()
    p = ops.DeviceArray((4096,), np.int32).ptr
    args = lambda **k: [dict(dict(free=p, n=p, t=p, stride=4, lens=p, seqs=2, pages=3), **k)[x] for x in ("free", "n", "t", "stride", "lens", "seqs", "pages")]
    for code, change in ((_lib.E_BAD_ARG, dict(free=None)), (_lib.E_BAD_ARG, dict(n=None)), (_lib.E_BAD_ARG, dict(t=None)), (_lib.E_BAD_ARG, dict(lens=None)), (_lib.E_BAD_ARG, dict(stride=0)),
                         (_lib.E_BAD_ARG, dict(seqs=-1)), (_lib.E_BAD_ARG, dict(pages=-1)), (_lib.E_BAD_ARG, dict(pages=2 ** 31 - 1)), (_lib.E_UNSUPPORTED, dict(seqs=65536))):
        with pytest.raises(HipError) as e:
            _lib.check(lib.cthip_kv_free_paged(*args(**change)))
        assert e.value.code == code, change
    with pytest.raises(ValueError):
        ops.kv_free_pages(np.zeros((2, 3)), [1], 4)
