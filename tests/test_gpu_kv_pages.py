"""Sequences that go on from others, and the pages in use brought to the front of the pool, against their definitions (include/caten_hip.h)."""
import numpy as np
import pytest

from tests.test_gpu_paged_q4 import PAGE, plan_by_hand

pytestmark = pytest.mark.gpu


def fork_by_hand(tables, lens, parents, children, at, free, k, v):
    """cthip_kv_fork_paged_q4, fork after fork; k and v (layers, pages, bytes) are changed."""
    n, stride = tables.shape
    old, tables, out, k0, v0 = tables, tables.copy(), list(lens), k.copy(), v.copy()
    refused, wanted, taken = [], 0, 0
    for f, (p, c, t) in enumerate(zip(parents, children, at)):
        ok = 0 <= p < n and 0 <= c < n and 0 <= t and c not in children[:f] and c not in parents
        ok = ok and t <= min(lens[p], stride * PAGE)
        need = ok and t % PAGE > 0
        wanted += need
        if not ok or (need and wanted > len(free)):
            refused.append(1)
            continue
        refused.append(0)
        full = t // PAGE
        tables[c, :full], out[c] = old[p, :full], t
        if need:
            page = free[len(free) - wanted]
            tables[c, full] = page
            taken += 1
            if 0 <= page < k.shape[1] and 0 <= old[p, full] < k.shape[1]:
                k[:, page], v[:, page] = k0[:, old[p, full]], v0[:, old[p, full]]
    return dict(tables=tables, lens=np.array(out), n_free=len(free) - taken, refused=np.array(refused))


def filled(rng, n_pages, kv, dh, layers):
    from caten_amd import _lib, ops
    cache = ops.PagedCacheQ4(n_pages, kv, dh, layers)
    for pool in (cache.k, cache.v):
        x = rng.integers(0, 256, pool.shape, dtype=np.uint8)
        _lib.check(_lib.load().cthip_h2d(pool.ptr, x.ctypes.data, x.nbytes))
    return cache


def sequences(rng, lens, stride, n_pages):
    pages = list(rng.permutation(n_pages))
    tables = np.full((len(lens), stride), -1, np.int32)
    for i, n in enumerate(lens):
        tables[i, :-(-n // PAGE)] = [pages.pop() for _ in range(-(-n // PAGE))]
    return tables, pages


def fork_and_compare(rng, cache, tables, lens, parents, children, at, free, spare=3):
    k, v = cache.k.numpy(), cache.v.numpy()
    got = cache.fork(tables, lens, parents, children, at, np.concatenate([free, [12345] * spare]), n_free=len(free))
    want = fork_by_hand(tables, lens, list(parents), list(children), at, free, k, v)
    for key in want:
        assert np.array_equal(got[key], want[key]), (key, got[key], want[key])
    assert np.array_equal(cache.k.numpy(), k) and np.array_equal(cache.v.numpy(), v)
    return got


@pytest.mark.parametrize("kv,dh,layers", [(12, 64, 3), (1, 32, 1), (8, 128, 2)])
@pytest.mark.parametrize("parents,forks,longest", [(1, 1, 10), (1, 8, 700), (5, 23, 300), (3, 0, 100), (2, 300, 130)])
def test_forks(kv, dh, layers, parents, forks, longest):
    print(f"case: {forks} forks of {parents} sequences up to {longest}, {kv} heads of {dh}, {layers} layers", flush=True)
    rng = np.random.default_rng(kv + forks)
    n, stride = parents + forks + 3, 12
    lens = [int(rng.integers(1, longest + 1)) for _ in range(parents)] + [0] * (n - parents)
    n_pages = sum(-(-x // PAGE) for x in lens) + forks + 4
    cache = filled(rng, n_pages, kv, dh, layers)
    tables, free = sequences(rng, lens, stride, n_pages)
    who = rng.integers(0, parents, forks)
    at = [int(rng.choice([lens[p], lens[p] // PAGE * PAGE, rng.integers(0, lens[p] + 1)])) for p in who]
    fork_and_compare(rng, cache, tables, lens, who, rng.permutation(np.arange(parents, n))[:forks], at, free)


def test_forks_that_are_refused():
    """Indices outside, lengths outside, children twice, children that are parents, and too few pages; what a child's row held behind its pages stays."""
    rng = np.random.default_rng(1)
    lens = [200, 130, 64, 100, 0, 0, 0, 0, 500, 7, 0, 0]
    stride, n_pages = 4, 40
    cache = filled(rng, n_pages, 2, 32, 2)
    tables, free = sequences(rng, [min(x, stride * PAGE) for x in lens], stride, n_pages)
    tables[4:8] = rng.integers(0, n_pages, (4, stride))
    parents = [0, 0, -1, 12, 1, 1, 1, 2, 8, 9, 2, 3, 3, 0, 1, 0]
    children = [4, 4, 5, 5, -1, 12, 0, 7, 6, 9, 8, 11, 10, 5, 3, 4]
    at = [150, 150, 3, 3, 3, 3, 3, 64, 257, 7, -1, 101, 100, 0, 5, 10]
    got = fork_and_compare(rng, cache, tables, lens, parents, children, at, free)
    assert got["refused"].sum() == 13 and not got["refused"][[0, 7, 12]].any()
    # two pages for four forks that need one: the two that need none are made
    got = fork_and_compare(rng, cache, tables, lens, [0, 0, 0, 1, 1, 0], [4, 5, 6, 7, 10, 11], [150, 128, 10, 129, 64, 20], free[:2])
    assert list(got["refused"]) == [0, 0, 0, 1, 0, 1] and got["n_free"] == 0
    got = fork_and_compare(rng, cache, tables, lens, [0, 0], [4, 5], [150, 128], [])
    assert list(got["refused"]) == [1, 0] and got["n_free"] == 0


def test_forks_from_pages_outside_the_pool():
    """A page id outside holds no key, in the child as in the parent; nothing is copied from or to it."""
    rng = np.random.default_rng(2)
    cache = filled(rng, 9, 1, 32, 2)
    tables = np.array([[3, -1, 9], [2 ** 31 - 1, 4, 5], [-1, -1, -1], [-1, -1, -1], [-1, -1, -1]], np.int32)
    fork_and_compare(rng, cache, tables, [130, 190, 0, 0, 0], [0, 0, 1], [2, 3, 4], [100, 130, 70], [7, 9, -3, 8])


@pytest.mark.parametrize("spare", [0, 300])
def test_forks_that_end_in_a_page_outside_the_pool(spare):
    """It holds no key, so the child's entry is the parent's and no page is taken: one from the stack would show the child what its last owner left there.  spare: forks in
    front of these, more than a workgroup's threads."""
    from caten_amd import ops
    rng = np.random.default_rng(11)
    n_pages, n = 12 + spare, 9 + spare
    cache = filled(rng, n_pages, 1, 32, 2)
    k, v = cache.k.numpy(), cache.v.numpy()
    tables = np.full((n, 3), -1, np.int32)
    tables[0], tables[1], tables[2], tables[4] = [3, -1, n_pages], [2 ** 31 - 1, 4, 5], [6, 7, 1], [2, 2, 2]
    lens = np.zeros(n, np.int32)
    lens[:3] = 130, 190, 192
    free = list(range(12, n_pages)) + [8, 9, 10, 11]
    parents, children, at = [2] * spare + [0, 0, 1, 1, 0], list(range(9, n)) + [3, 4, 5, 6, 7], [1 + i % 63 for i in range(spare)] + [100, 130, 70, 20, 128]
    for _ in range(2):  # (the same call again gives the same)
        got = cache.fork(tables, lens, parents, children, at, free)
        want = tables.copy()
        want[9:, 0] = free[::-1][:spare]
        page = free[::-1][spare]  # for the one fork of these that ends in a page of the pool
        want[3, :2], want[4], want[5, :2], want[6, :1], want[7, :2] = [3, -1], [3, -1, n_pages], [2 ** 31 - 1, page], [2 ** 31 - 1], [3, -1]
        assert np.array_equal(got["tables"], want) and not got["refused"].any() and got["n_free"] == len(free) - spare - 1
        assert np.array_equal(got["lens"][children], at)
        for pool, now in ((k, cache.k.numpy()), (v, cache.v.numpy())):
            pool[:, page] = pool[:, 4]
            pool[:, want[9:, 0]] = pool[:, 6][:, None]
            assert np.array_equal(now, pool)
    # the plan takes pages from where the forks have left the stack, and the two that need none are made without any
    got = cache.fork(tables, lens, [0, 0], [3, 4], [100, 130], [])
    assert not got["refused"].any() and got["n_free"] == 0
    # attention: the parent's rows that there are
    from tests.test_gpu_paged_q4 import _fill
    cache = ops.PagedCacheQ4(n_pages, 1, 32)
    _fill(cache, 0xff)
    rows = rng.normal(0, 1, (64 * 2, 1, 32)).astype(np.float32)
    cache.append(rows, rows, np.concatenate([np.arange(64) + 3 * 64, np.arange(64) + 11 * 64]))  # page 11: of a sequence that has left
    got = cache.fork(tables, lens, [0], [3], [100], free)
    q = rng.normal(0, 1, (1, 2, 32)).astype(np.float32)
    one = lambda table, length: cache.attend(q, table, [length], [0, 1])
    assert np.array_equal(one(got["tables"][3:4], 100), one(tables[:1], 100))


def test_as_many_forks_as_there_can_be():
    rng = np.random.default_rng(3)
    n, forks, stride = 4096, 4000, 2
    lens = [100] * 90 + [0] * (n - 90)
    cache = filled(rng, 4500, 1, 32, 1)
    tables, free = sequences(rng, lens, stride, 4500)
    parents, children = rng.integers(0, 90, forks), rng.permutation(np.arange(90, n))[:forks]
    at = rng.integers(0, 101, forks)
    k, v = cache.k.numpy(), cache.v.numpy()
    got = cache.fork(tables, lens, parents, children, at, free)
    assert not got["refused"].any() and np.array_equal(got["lens"][children], at)
    need = at % PAGE > 0
    page = np.array(free)[len(free) - np.cumsum(need)]
    assert got["n_free"] == len(free) - need.sum()
    full = at // PAGE
    assert np.array_equal(got["tables"][children[need], full[need]], page[need])
    k[:, page[need]], v[:, page[need]] = k[:, tables[parents, full][need]], v[:, tables[parents, full][need]]
    assert np.array_equal(cache.k.numpy(), k) and np.array_equal(cache.v.numpy(), v)


def test_free_pages_in_place_and_apart():
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(4)
    cache = filled(rng, 12, 1, 32, 1)
    tables, free = sequences(rng, [100, 0, 0], 3, 12)
    d = {k: ops.DeviceArray.from_numpy(np.asarray(v, np.int32)) for k, v in dict(t=tables, lens=[100, 0, 0], p=[0, 0], c=[1, 2], at=[70, 99], free=free, n=[len(free)]).items()}
    out, refused = ops.DeviceArray((1,), np.int32), ops.DeviceArray((2,), np.int32)

    def call(to, n):
        _lib.check(lib.cthip_kv_fork_paged_q4(d["t"].ptr, 3, d["lens"].ptr, 3, to.ptr, refused.ptr, cache.k.ptr, cache.v.ptr, 1, 12, d["p"].ptr, d["c"].ptr, d["at"].ptr, n, d["free"].ptr, d["n"].ptr,
                                              1, 32))
    for _ in range(2):  # the same call again gives the same
        call(out, 2)
        assert out.numpy()[0] == len(free) - 2 and d["n"].numpy()[0] == len(free) and list(d["t"].numpy()[1:, 1]) == free[::-1][:2]
    call(d["n"], 2)
    assert d["n"].numpy()[0] == len(free) - 2
    call(d["n"], 0)
    call(out, 0)
    assert d["n"].numpy()[0] == len(free) - 2 and out.numpy()[0] == len(free) - 2


def compact_by_hand(tables, lens, n_pages, k, v):
    there = np.arange(tables.shape[1]) < -(-np.maximum(lens, 0) // PAGE)[:, None]
    there &= (tables >= 0) & (tables < n_pages)
    used = np.zeros(n_pages, bool)
    used[tables[there]] = True
    n = used.sum()
    src, dst = np.flatnonzero(used[n:]) + n, np.flatnonzero(~used[:n])
    to = np.arange(n_pages)
    to[src] = dst
    out = tables.copy()
    out[there] = to[tables[there]]
    k[:, dst], v[:, dst] = k[:, src], v[:, src]
    return out, np.arange(n_pages - 1, n - 1, -1)


@pytest.mark.parametrize("kv,dh,layers", [(3, 64, 2), (1, 32, 1), (2, 128, 3)])
@pytest.mark.parametrize("n,longest,spare,shared", [(1, 1, 0, 0), (5, 300, 20, 2), (40, 200, 100, 1), (7, 500, 0, 0), (3, 64, 700, 0), (300, 90, 900, 1)])
def test_compaction(kv, dh, layers, n, longest, spare, shared):
    print(f"case: {n} sequences up to {longest}, {spare} pages besides, {shared} shared, {kv} heads of {dh}, {layers} layers", flush=True)
    rng = np.random.default_rng(n + spare)
    lens = rng.integers(0, longest + 1, n)
    lens[0] = longest
    lens[3::7] = -5
    stride = -(-longest // PAGE) + 2
    n_pages = int(sum(-(-max(x, 0) // PAGE) for x in lens)) + spare
    cache = filled(rng, n_pages, kv, dh, layers)
    tables, _ = sequences(rng, np.maximum(lens, 0), stride, n_pages)
    tables[1:, :shared] = np.where(lens[1:, None] > PAGE * np.arange(shared), tables[0, :shared], tables[1:, :shared])
    tables[:, -1] = 3                                 # behind every sequence's pages
    if n > 20:
        tables[5, 0], tables[6, 0] = -7, n_pages + 2  # outside the pool
    k, v = cache.k.numpy(), cache.v.numpy()
    want, free = compact_by_hand(tables, lens, n_pages, k, v)
    got = cache.compact(tables, lens)
    assert np.array_equal(got["tables"], want) and np.array_equal(got["free_pages"], free)
    assert np.array_equal(cache.k.numpy(), k) and np.array_equal(cache.v.numpy(), v)
    again = cache.compact(want, lens)  # nothing left to move
    assert np.array_equal(again["tables"], want) and np.array_equal(again["free_pages"], free) and np.array_equal(cache.k.numpy(), k)


def test_compaction_of_a_large_pool():
    rng = np.random.default_rng(5)
    n, stride, n_pages = 500, 130, 70001
    lens = rng.integers(0, stride * PAGE + 1, n)
    tables, _ = sequences(rng, lens, stride, n_pages)
    cache = filled(rng, n_pages, 1, 32, 1)
    k, v = cache.k.numpy(), cache.v.numpy()
    want, free = compact_by_hand(tables, lens, n_pages, k, v)
    got = cache.compact(tables, lens)
    assert np.array_equal(got["tables"], want) and np.array_equal(got["free_pages"], free)
    assert np.array_equal(cache.k.numpy(), k) and np.array_equal(cache.v.numpy(), v)


@pytest.mark.parametrize("n_seqs,n_pages", [(0, 5), (2, 0), (0, 0)])
def test_compaction_of_nothing(n_seqs, n_pages):
    from caten_amd import _lib, ops
    lib = _lib.init()
    tables, lens = ops.DeviceArray.from_numpy(np.full((2, 3), 4, np.int32)), ops.DeviceArray.from_numpy(np.array([70, 3], np.int32))
    out, free, n, ws, pool = (ops.DeviceArray((m,), np.int32) for m in (6, 8, 1, 64, 8000))
    _lib.check(lib.cthip_kv_compact_paged_q4(out.ptr, free.ptr, n.ptr, pool.ptr, pool.ptr, 1, n_pages, tables.ptr, 3, lens.ptr, n_seqs, 1, 32, ws.ptr))
    assert n.numpy()[0] == n_pages and list(free.numpy()[:n_pages]) == list(range(n_pages))[::-1] and list(out.numpy()) == [4 * (n_seqs > 0)] * 6


def test_a_plan_behind_a_compaction_takes_the_lowest_pages():
    from caten_amd import ops
    rng = np.random.default_rng(6)
    cache = filled(rng, 30, 1, 32, 1)
    lens = [100, 64, 5]
    tables, _ = sequences(rng, lens, 4, 30)
    got = cache.compact(tables, lens)
    step = ops.kv_plan(lens, [60, 1, 1], got["tables"], got["free_pages"], 70)
    assert step["refused"] == 0 and step["tables"].max() == 5 and step["n_free"] == 24
    want = plan_by_hand(lens, [60, 1, 1], got["tables"], list(got["free_pages"]), 70)
    assert np.array_equal(step["tables"], want["tables"]) and np.array_equal(step["slots"], want["slots"])


def test_refusals():
    from caten_amd import _lib, ops
    lib, d = _lib.init(), ops.DeviceArray((1 << 16,), np.uint8)
    p = d.ptr

    def fork(**k):
        a = dict(t=p, stride=4, lens=p + 1024, n=2, nfo=p + 2048, ref=p + 3000, kp=p + 8192, vp=p + 8192 + 1152 * 4, layers=1, pages=4, par=p + 4096, ch=p + 4352, at=p + 4608, f=0, free=p + 5120,
                 nf=p + 6144, kv=1, dh=32)
        a.update(k)
        return lib.cthip_kv_fork_paged_q4(*a.values())

    def compact(**k):
        a = dict(to=p, free=p + 1024, nf=p + 2048, kp=p + 8192, vp=p + 8192 + 1152 * 4, layers=1, pages=4, t=p + 3000, stride=4, lens=p + 4096, n=0, kv=1, dh=32, ws=p + 5120)
        a.update(k)
        return lib.cthip_kv_compact_paged_q4(*a.values())

    for bad in (dict(n=-1), dict(f=-1), dict(layers=-1), dict(pages=-1), dict(stride=0), dict(nf=None), dict(nfo=None), dict(pages=1 << 26), dict(stride=1 << 26), dict(f=1, ref=None), dict(f=1, par=None),
                dict(f=1, ch=None), dict(f=1, at=None), dict(f=1, free=None), dict(f=1, t=None), dict(f=1, lens=None), dict(f=1, kp=None), dict(f=1, vp=p + 8200)):
        assert fork(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(kv=0), dict(dh=48), dict(n=4097), dict(f=4097), dict(layers=(1 << 20) + 1)):
        assert fork(**bad) == _lib.E_UNSUPPORTED, bad
    for bad in (dict(n=-1), dict(layers=-1), dict(pages=-1), dict(stride=0), dict(nf=None), dict(ws=None), dict(ws=p + 5124), dict(free=None), dict(n=1, t=None), dict(n=1, to=None), dict(n=1, lens=None),
                dict(kp=None), dict(vp=p + 8200), dict(pages=1 << 26)):
        assert compact(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(kv=0), dict(dh=48), dict(n=65536), dict(layers=65535)):
        assert compact(**bad) == _lib.E_UNSUPPORTED, bad
    assert not d.numpy().any()
    cache = ops.PagedCacheQ4(2, 1, 32)
    for call in (lambda: cache.fork(np.zeros((2, 2)), [1], [0], [1], [0], [1]), lambda: cache.fork(np.zeros((2, 2)), [1, 0], [0], [1, 1], [0], [1]),
                 lambda: cache.fork(np.zeros((2, 2)), [1, 0], [0], [1], [0], [1], n_free=2), lambda: cache.compact(np.zeros((2, 2)), [1])):
        with pytest.raises(ValueError):
            call()
