"""Attention of a batch whose sequences share their first pages: against its definition in 64 bits, with the tolerance of attention over the 4-bit cache
(derived in test_gpu_paged_q4.close; maxima and sums joined once more are two fp32 roundings, within what is left there)."""
import numpy as np
import pytest

from tests.test_gpu_paged_q4 import PAGE, _fill, attention, close

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=[2, 0], ids=["apart", "together"])
def way(request):
    """Shared pages in a launch of their own, or as every sequence's own: option "shared_prefix"."""
    from caten_amd import _lib
    _lib.check(_lib.init().cthip_set_option(b"shared_prefix", request.param))
    yield request.param
    _lib.check(_lib.load().cthip_set_option(b"shared_prefix", 1))


def answers(rng, groups, kv, dh, spare=3):
    """groups: (rows shared, [(rows held in all, query rows)]); pages in any order, what no row was written to is NaN.
    (cache, tables, lens, starts, borders, shared, [(k, v)])"""
    from caten_amd import ops
    seqs = [s for _, m in groups for s in m]
    stride = max(1, max(-(-t // PAGE) for t, _ in seqs))
    pages = list(rng.permutation(sum(p // PAGE + sum(-(-t // PAGE) for t, _ in m) for p, m in groups) + spare))
    cache = ops.PagedCacheQ4(len(pages), kv, dh)
    _fill(cache, 0xff)
    tables, held, i = np.full((len(seqs), stride), -1, np.int32), [], 0

    def rows(mine, first, n):
        if n <= 0:
            return np.zeros((0, kv, dh), np.float32), np.zeros((0, kv, dh), np.float32)
        k = (rng.normal(0, 1, (n, kv, dh)) * np.exp(0.5 * rng.normal(0, 1, (1, kv, dh)))).astype(np.float32)
        v = (rng.normal(0, 1, (n, kv, dh)) * np.exp(0.5 * rng.normal(0, 1, (1, kv, dh)))).astype(np.float32)
        slots = np.array([mine[t // PAGE] * PAGE + t % PAGE for t in range(first, first + n)], np.int32)
        cache.append(k, v, slots)
        return cache.rows(slots)
    for p, m in groups:
        common = [pages.pop() for _ in range(p // PAGE)]
        first = rows(common, 0, p // PAGE * PAGE)
        for t, _ in m:
            mine = common + [pages.pop() for _ in range(-(-t // PAGE) - p // PAGE)]
            tables[i, :len(mine)] = mine
            own = rows(mine, p // PAGE * PAGE, t - p // PAGE * PAGE)
            held.append([np.concatenate([a, b]) for a, b in zip(first, own)])
            i += 1
    return (cache, tables, np.array([t for t, _ in seqs]), np.concatenate([[0], np.cumsum([r for _, r in seqs])]), np.concatenate([[0], np.cumsum([len(m) for _, m in groups])]),
            np.array([p for p, _ in groups]), held)


def seen(q, k, v, whole):
    """`attention` of the last rows of a sequence whose first `whole` keys every row sees."""
    n, at = len(q), len(k) - len(q)
    if at + 1 >= whole:
        return attention(q, k, v)
    parts = [attention(q[r:r + 1], k[:max(at + r + 1, whole)], v[:max(at + r + 1, whole)]) for r in range(n)]
    return tuple(np.concatenate(x) for x in zip(*parts))


def compare(rng, H, kv, dh, groups, scale=1.0):
    cache, tables, lens, starts, borders, shared, held = answers(rng, groups, kv, dh)
    q = (scale * rng.normal(0, 1, (starts[-1], H, dh))).astype(np.float32)
    got = cache.attend_shared(q, tables, lens, starts, borders, shared)
    whole = np.concatenate([[p // PAGE * PAGE * (len(m) > 1)] * len(m) for p, m in groups]).astype(int)
    for i, (k, v) in enumerate(held):
        if starts[i + 1] > starts[i]:
            close(got[starts[i]:starts[i + 1]], *seen(q[starts[i]:starts[i + 1]], k, v, whole[i]))
    assert np.array_equal(got, cache.attend_shared(q, tables, lens, starts, borders, shared))  # two runs, the same bits
    return cache, tables, lens, starts, borders, shared, held, q, got


SHAPES = [(12, 12, 64), (32, 4, 64), (8, 1, 128), (4, 4, 128), (6, 2, 32), (16, 1, 32), (21, 3, 128), (17, 1, 64)]


@pytest.mark.parametrize("H,kv,dh", SHAPES)
@pytest.mark.parametrize("groups", [
    [(64, [(65, 1), (66, 1)])],
    [(200, [(201, 1), (264, 1), (330, 1), (193, 1), (500, 1)])],
    [(128, [(140, 5), (129, 1), (300, 0), (200, 17)]), (63, [(70, 3), (64, 1)]), (64, [(90, 2)]), (320, [(321, 1)] * 9)],
    [(1000, [(1001, 1)] * 20)]])
def test_groups(H, kv, dh, groups):
    print(f"case: {H} heads over {kv} of {dh}, groups {groups}", flush=True)
    compare(np.random.default_rng(H + dh + len(groups)), H, kv, dh, groups)


@pytest.mark.parametrize("H,kv,dh,groups", [
    (32, 32, 128, [(1000, [(1001 + 3 * i, 1) for i in range(64)])]),
    (64, 8, 128, [(700, [(800 + i, 5) for i in range(14)]), (320, [(330 + 60 * i, 4) for i in range(9)])]),
    (64, 1, 128, [(192, [(193 + i, 3) for i in range(7)])]),
    (8, 8, 64, [(450, [(460 + i, 1 + i % 40) for i in range(41)])]),
    (4, 2, 32, [(256, [(300 + i, 33) for i in range(9)])]),
    (6, 3, 128, [(128, [(128 + 200, 200), (128 + 150, 150)])])])
def test_many_rows(H, kv, dh, groups):
    print(f"case: many rows, {H} heads over {kv} of {dh}, {len(groups)} groups", flush=True)
    compare(np.random.default_rng(H + dh), H, kv, dh, groups)


@pytest.mark.parametrize("H,kv,dh,members", [(4, 1, 64, 3), (8, 8, 128, 40), (16, 1, 128, 9)])
def test_a_long_prefix(H, kv, dh, members):
    compare(np.random.default_rng(members), H, kv, dh, [(20000, [(20001 + i, 1) for i in range(members)])])


def test_many_groups():
    rng = np.random.default_rng(12)
    compare(rng, 4, 2, 64, [(64 * (i % 3), [(64 * (i % 3) + 1 + (i * 37 + j) % 100, (i + j) % 3) for j in range(i % 4 + 1)]) for i in range(150)])


# More jobs than workgroups that run at once, each of four rows of a head at most: a wavefront takes a job by itself (at 64 channels and fewer in one launch as well).  One
# sequence or two hold far more behind the shared pages, whose shares many wavefronts join.
@pytest.mark.parametrize("H,kv,dh,groups", [
    (12, 12, 64, [(300, [(301 + 9 * i, 1) for i in range(40)] + [(9000, 1)]), (330, [(331 + i % 70, 1) for i in range(50)]), (0, [(1 + 5 * i, 1) for i in range(30)])]),
    (4, 4, 32, [(320, [(321 + i, 1) for i in range(150)] + [(20000, 1)]), (290, [(300 + i % 300, i % 3 != 1) for i in range(160)])]),
    (8, 4, 64, [(260, [(270 + i % 40, 1 + i % 3) for i in range(270)] + [(6000, 2)])]),
    (32, 32, 128, [(200, [(201 + 4 * i, 1) for i in range(35)] + [(5000, 1)]), (64, [(65, 1), (3000, 1), (70, 4)])]),
    (16, 8, 128, [(450, [(451 + i % 100, 2) for i in range(110)] + [(4000, 1)])])])
def test_jobs_of_single_wavefronts(H, kv, dh, groups):
    print(f"case: jobs of single wavefronts, {H} heads over {kv} of {dh}, {len(groups)} groups", flush=True)
    compare(np.random.default_rng(26 + dh + H), H, kv, dh, groups)


def test_wavefronts_with_more_pages_than_lanes():
    """Parts of some 80 pages: a wavefront asks for page ids 64 at a time, of the group's table in one launch."""
    from caten_amd import ops
    rng = np.random.default_rng(27)
    n, kv, dh, pages = 520, 2, 32, 240
    cache = ops.PagedCacheQ4(pages + n + 3, kv, dh)
    _fill(cache, 0xff)
    ids = rng.permutation(cache.n_pages)
    tables = np.concatenate([np.full((n, pages), -1), ids[pages:pages + n, None]], 1).astype(np.int32)
    tables[0, :pages] = ids[:pages]  # (of what is shared the first sequence's entries are read)
    own = 1 + np.arange(n) % 60
    lens, starts = pages * PAGE + own, np.arange(n + 1)

    def rows(slots):
        k, v = (rng.normal(0, 1, (len(slots), kv, dh)).astype(np.float32) for _ in range(2))
        cache.append(k, v, slots)
        return cache.rows(slots)
    first = rows((tables[0, :pages, None] * PAGE + np.arange(PAGE)).ravel())
    behind = rows(np.concatenate([t * PAGE + np.arange(m) for t, m in zip(tables[:, -1], own)]))
    q = rng.normal(0, 1, (n, kv, dh)).astype(np.float32)
    got = cache.attend_shared(q, tables, lens, starts, [0, n], [pages * PAGE])
    at = np.concatenate([[0], np.cumsum(own)])
    for i in range(n):
        close(got[i:i + 1], *attention(q[i:i + 1], *(np.concatenate([a, b[at[i]:at[i + 1]]]) for a, b in zip(first, behind))))
    assert np.array_equal(got, cache.attend_shared(q, tables, lens, starts, [0, n], [pages * PAGE]))


def test_as_many_sequences_as_there_may_be():
    rng = np.random.default_rng(23)
    groups, left = [], 4096
    while left:
        m = min(left, 1 + len(groups) % 8)
        left -= m
        groups.append((64 * (len(groups) % 3), [(64 * (len(groups) % 3) + 1 + j, (j + len(groups)) % 4 != 0) for j in range(m)]))
    compare(rng, 2, 1, 32, groups)


def test_the_same_as_without_sharing():
    """Against the attention that reads every sequence's pages by itself: both are within the tolerance of the same numbers, with groups that share nothing or have one
    sequence too.  A batch without groups is the same bits."""
    rng = np.random.default_rng(13)
    cache, tables, lens, starts, borders, shared, held, q, got = compare(rng, 12, 4, 64, [(300, [(310, 2), (305, 1), (400, 7)]), (90, [(95, 1)])])
    plain = cache.attend(q, tables, lens, starts)
    assert np.array_equal(cache.attend_shared(q, tables, lens, starts, [0], []), plain)
    for some in [got] + [cache.attend_shared(q, tables, lens, starts, b, s)
                         for b, s in (([0, 3, 4], [0, 0]), ([0, 3, 4], [63, 64]), ([0, 0, 0, 1, 1], [640] * 4), ([2, 3], [300]), ([0, 3], [-5]))]:
        for i, (k, v) in enumerate(held):
            _, size, big = attention(q[starts[i]:starts[i + 1]], k, v)
            close(some[starts[i]:starts[i + 1]], plain[starts[i]:starts[i + 1]], 2 * size, 2 * big)
    # some sequences in front of the groups and behind them
    for b, s in (([1, 3], [300]), ([0, 2], [300]), ([0, 1, 3, 4], [300, 256, 90])):
        part = cache.attend_shared(q, tables, lens, starts, b, s)
        for i, (k, v) in enumerate(held):
            close(part[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


def test_rows_in_front_of_what_is_shared():
    """A row sees all of its group's shared pages, whatever its position, and of what is behind them what its own position reaches."""
    rng = np.random.default_rng(14)
    H, kv, dh = 6, 2, 64
    cache, tables, lens, starts, borders, shared, held = answers(rng, [(128, [(200, 1), (150, 1), (140, 3)])], kv, dh)
    q = rng.normal(0, 1, (5, H, dh)).astype(np.float32)
    short = np.array([200, 100, 130])  # the second ends inside the shared pages, the third's first rows lie in them
    got = cache.attend_shared(q, tables, short, starts, borders, shared)
    for row, (i, t) in enumerate([(0, 200), (1, 128), (2, 128), (2, 129), (2, 130)]):
        k, v = (x[:t] for x in held[i])
        close(got[row:row + 1], *attention(q[row:row + 1], k, v))


def test_pages_outside_the_pool():
    """Shared pages that are nowhere hold no key; where a sequence has none besides either, its rows are zero; a table's end."""
    rng = np.random.default_rng(15)
    H, kv, dh = 8, 2, 64
    cache, tables, lens, starts, borders, shared, held = answers(rng, [(192, [(193, 1), (200, 2), (192, 1)])], kv, dh)
    q = rng.normal(0, 1, (4, H, dh)).astype(np.float32)
    gone = tables.copy()
    gone[0, 1] = -1
    got = cache.attend_shared(q, gone, lens, starts, borders, shared)
    for row, (i, t) in enumerate([(0, 193), (1, 199), (1, 200), (2, 192)]):
        k, v = (np.concatenate([x[:64], x[128:t]]) for x in held[i])
        close(got[row:row + 1], *attention(q[row:row + 1], k, v))
    gone[0, :3] = cache.n_pages, -1, 2 ** 31 - 1
    got = cache.attend_shared(q, gone, lens, starts, borders, shared)
    for row, (i, t) in enumerate([(0, 193), (1, 199), (1, 200)]):
        k, v = (x[192:t] for x in held[i])
        close(got[row:row + 1], *attention(q[row:row + 1], k, v))
    assert not got[3].any()
    got = cache.attend_shared(q, tables[:, :2], lens, starts, borders, [10 ** 6])  # a table of two pages
    for row, i in enumerate([0, 1, 1, 2]):
        k, v = (x[:128] for x in held[i])
        close(got[row:row + 1], *attention(q[row:row + 1], k, v))


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("factors", [(1e-6, 1), (1, 1e-6), (30, 1), (1e5, 1), (1, 1e5), (1e3, 1e-3), (0, 1), (1, 0)])
def test_sizes_of_values(rows, factors):
    """Values of the shared pages and of the others of different sizes (a power of two goes with each part's sums)."""
    rng = np.random.default_rng(rows)
    H, kv, dh = 8, 2, 64
    cache, tables, lens, starts, borders, shared, held = answers(rng, [(192, [(220, rows), (300, rows), (193, 1)])], kv, dh)
    for i in range(3):
        for first, n, factor in ((0, 192, factors[0]), (192, lens[i] - 192, factors[1])):
            slots = np.array([tables[i, t // PAGE] * PAGE + t % PAGE for t in range(first, first + n)], np.int32)
            k, v = (x[first:first + n] for x in held[i])
            if first or i == 0:
                cache.append(k, np.float32(factor) * v, slots)
            got = cache.rows(slots)
            held[i][0][first:first + n], held[i][1][first:first + n] = got
    q = rng.normal(0, 1, (starts[-1], H, dh)).astype(np.float32)
    got = cache.attend_shared(q, tables, lens, starts, borders, shared)
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


@pytest.mark.parametrize("scale", [1e-30, 30.0, 3e3, 1e6])
def test_sizes_of_queries(scale):
    compare(np.random.default_rng(16), 8, 2, 64, [(256, [(270, 1), (300, 3), (257, 1)])], scale)


def test_infinities_and_nan():
    """A query row that is not finite is NaN and its neighbours are not; a key that is not, in the shared pages, is everybody's; behind them, its sequence's."""
    rng = np.random.default_rng(17)
    H, kv, dh = 4, 2, 64
    cache, tables, lens, starts, borders, shared, held, q, want = compare(rng, H, kv, dh, [(128, [(140, 1), (150, 2), (129, 1)])])
    for bad in (np.nan, np.inf, -np.inf):
        x = q.copy()
        x[1, 2, 5] = bad
        got = cache.attend_shared(x, tables, lens, starts, borders, shared)
        assert np.isnan(got[1, 2]).all()
        keep = np.ones((4, H), bool)
        keep[1, 2] = False
        assert np.array_equal(got[keep], want[keep])
    one = np.zeros((1, kv, dh), np.float32)
    one[0, 0, 3] = np.nan
    cache.append(one, one, np.array([tables[2, 2] * PAGE], np.int32))  # the last sequence's own row
    got = cache.attend_shared(q, tables, lens, starts, borders, shared)
    assert np.array_equal(got[:3], want[:3]) and np.isnan(got[3, :2]).any() and np.isfinite(got[3, 2:]).all()
    cache.append(one, one, np.array([tables[0, 0] * PAGE + 9], np.int32))
    got = cache.attend_shared(q, tables, lens, starts, borders, shared)
    assert np.isnan(got[:, :2]).any(-1).all() and np.isfinite(got[:, 2:]).all()


def test_rows_behind_the_last_and_a_workspace_of_other_shapes():
    """Rows behind the last sequence's stay; one workspace goes from shape to shape."""
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(18)
    ws = ops.DeviceArray((int(lib.cthip_sdpa_shared_paged_q4_workspace(200, 64, 128)),), np.uint8)
    for H, kv, dh, groups in ((64, 8, 128, [(400, [(500 + i, 3) for i in range(20)])]), (12, 12, 64, [(900, [(901 + i, 1) for i in range(8)])]), (6, 2, 32, [(64, [(65, 1), (700, 30)])]),
                              (64, 8, 128, [(5000, [(5001 + i, 1) for i in range(3)])]), (16, 1, 64, [(128, [(129, 2)] * 60)])):
        cache, tables, lens, starts, borders, shared, held = answers(rng, groups, kv, dh)
        n = int(starts[-1])
        q = rng.normal(0, 1, (n + 5, H, dh)).astype(np.float32)
        dq, dt, dl, ds, dg, dsh = (ops.DeviceArray.from_numpy(np.ascontiguousarray(a, t)) for a, t in ((q, np.float32), (tables, np.int32), (lens, np.int32), (starts, np.int32), (borders, np.int32),
                                                                                                        (shared, np.int32)))
        out = ops.DeviceArray.from_numpy(np.full(q.shape, 7.0, np.float32))
        for _ in range(2):
            _lib.check(lib.cthip_sdpa_shared_paged_q4(out.ptr, dq.ptr, H * dh, cache.k.ptr, cache.v.ptr, cache.n_pages, dt.ptr, tables.shape[1], dl.ptr, ds.ptr, len(lens), n + 5, dg.ptr, dsh.ptr,
                                                      len(shared), H, kv, dh, ws.ptr))
            got = out.numpy()
            assert (got[n:] == 7.0).all()
            for i, (k, v) in enumerate(held):
                close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))
        assert not ws.numpy()[:16384].any()


def test_a_caches_workspace_is_kept():
    """One for all calls, as large as the largest has asked for: its size does not depend on the batch but for its rows, and it is left ready for any."""
    rng = np.random.default_rng(25)
    cache, tables, lens, starts, borders, shared, held = answers(rng, [(192, [(200, 1), (230, 9), (193, 1)])], 2, 64)
    q = rng.normal(0, 1, (starts[-1], 8, 64)).astype(np.float32)
    few = cache.attend_shared(q[:1, :2], tables, lens, [0, 1, 1, 1], borders, shared)
    first = cache.shared_workspace
    got = cache.attend_shared(q, tables, lens, starts, borders, shared)
    larger = cache.shared_workspace
    assert larger.nbytes > first.nbytes and not larger.numpy()[:16384].any()
    assert np.array_equal(cache.attend_shared(q[:1, :2], tables, lens, [0, 1, 1, 1], borders, shared), few)
    assert np.array_equal(cache.attend_shared(q, tables, lens, starts, borders, shared), got) and cache.shared_workspace is larger
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


@pytest.mark.parametrize("fill", [0x7f, 0xff])
def test_whatever_the_workspace_holds(fill):
    """Behind its tickets: large numbers, NaN; the groups are one of many jobs, some of shares, and a batch by wavefronts."""
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(20)
    for H, kv, dh, groups in ((64, 8, 128, [(900, [(1000 + i, 3) for i in range(20)])]), (32, 32, 128, [(300, [(301 + i, 1) for i in range(40)])]), (6, 2, 64, [(640, [(650, 1), (700, 30)])])):
        cache, tables, lens, starts, borders, shared, held = answers(rng, groups, kv, dh)
        q = rng.normal(0, 1, (starts[-1], H, dh)).astype(np.float32)
        raw = np.full(int(lib.cthip_sdpa_shared_paged_q4_workspace(len(q), H, dh)), fill, np.uint8)
        raw[:16384] = 0
        ws, dq, dt, dl, ds, dg, dsh = (ops.DeviceArray.from_numpy(np.ascontiguousarray(a, t)) for a, t in ((raw, np.uint8), (q, np.float32), (tables, np.int32), (lens, np.int32),
                                                                                                            (starts, np.int32), (borders, np.int32), (shared, np.int32)))
        out = ops.DeviceArray(q.shape, np.float32)
        _lib.check(lib.cthip_sdpa_shared_paged_q4(out.ptr, dq.ptr, H * dh, cache.k.ptr, cache.v.ptr, cache.n_pages, dt.ptr, tables.shape[1], dl.ptr, ds.ptr, len(lens), len(q), dg.ptr, dsh.ptr,
                                                  len(shared), H, kv, dh, ws.ptr))
        got = out.numpy()
        for i, (k, v) in enumerate(held):
            close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))
        assert np.array_equal(got, cache.attend_shared(q, tables, lens, starts, borders, shared))


@pytest.mark.parametrize("borders", [[1, 3, 2, 3], [-4, 0, 9, 2, 4], [2 ** 31 - 1, -2 ** 31], [1, 3, 1, 3, 1, 3]])
def test_groups_out_of_order(borders):
    """Rows of groups that fall or leave the batch are anybody's guess; those of sequences in front of all groups and behind them are right."""
    from caten_amd import _lib, ops
    rng = np.random.default_rng(21)
    H, kv, dh = 8, 2, 64
    cache, tables, lens, starts, _, _, held = answers(rng, [(200, [(210, 1), (300, 3), (260, 2), (201, 1)]), (0, [(77, 2)])], kv, dh)
    q = rng.normal(0, 1, (starts[-1], H, dh)).astype(np.float32)
    lib = _lib.init()
    raw = np.full(int(lib.cthip_sdpa_shared_paged_q4_workspace(len(q), H, dh)), 0xff, np.uint8)  # (what rows left out find there)
    raw[:16384] = 0
    ws, dq, dt, dl, ds, dg, dsh = (ops.DeviceArray.from_numpy(np.ascontiguousarray(a, t)) for a, t in ((raw, np.uint8), (q, np.float32), (tables, np.int32), (lens, np.int32), (starts, np.int32),
                                                                                                        (borders, np.int32), ([192] * (len(borders) - 1), np.int32)))
    out = ops.DeviceArray(q.shape, np.float32)
    _lib.check(lib.cthip_sdpa_shared_paged_q4(out.ptr, dq.ptr, H * dh, cache.k.ptr, cache.v.ptr, cache.n_pages, dt.ptr, tables.shape[1], dl.ptr, ds.ptr, len(lens), len(q), dg.ptr, dsh.ptr,
                                              len(borders) - 1, H, kv, dh, ws.ptr))
    got = out.numpy()
    for i, (k, v) in enumerate(held):
        if i < min(max(min(borders), 0), 5) or i >= min(max(borders), 5) or borders[0] > 5:
            close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


def test_places_past_32_bits():
    """Shared pages at the end of a pool of more than 2^32 bytes."""
    from caten_amd import ops
    rng = np.random.default_rng(19)
    kv, dh, n_pages, H = 32, 128, 30000, 32
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    tables = np.array([[n_pages - 1, n_pages - 2, 3], [n_pages - 1, n_pages - 2, n_pages - 3], [n_pages - 1, n_pages - 2, n_pages - 4]], np.int32)
    lens, held = [130, 150, 192], []
    for i, t in enumerate(lens):
        slots = np.array([tables[i, j // PAGE] * PAGE + j % PAGE for j in range(t)], np.int32)
        new = slots if i == 0 else slots[128:]
        cache.append(*(rng.normal(0, 1, (len(new), kv, dh)).astype(np.float32) for _ in range(2)), new)
        held.append(cache.rows(slots))
    q = rng.normal(0, 1, (3, H, dh)).astype(np.float32)
    got = cache.attend_shared(q, tables, lens, [0, 1, 2, 3], [0, 3], [128])
    for i, (k, v) in enumerate(held):
        close(got[i:i + 1], *attention(q[i:i + 1], k, v))


def test_refusals():
    from caten_amd import _lib, ops
    lib, d = _lib.init(), ops.DeviceArray((1 << 16,), np.uint8)
    p = d.ptr

    def call(**k):
        a = dict(out=p, q=p + 4096, qs=128, kp=p + 8192, vp=p + 8192 + 2304, pages=1, t=p + 16384, stride=4, lens=p + 17408, starts=p + 18432, n=2, rows=2, groups=p + 19456, shared=p + 20480, g=1, H=2,
                 kv=1, dh=64, ws=p + 32768)
        a.update(k)
        return lib.cthip_sdpa_shared_paged_q4(*a.values())

    for bad in (dict(n=-1), dict(rows=-1), dict(pages=-1), dict(stride=0), dict(H=0), dict(kv=0), dict(H=3, kv=2, qs=300), dict(g=-1), dict(g=3), dict(groups=None), dict(shared=None), dict(out=None),
                dict(q=None), dict(q=p), dict(t=None), dict(lens=None), dict(starts=None), dict(ws=None), dict(ws=p + 32772), dict(kp=None), dict(vp=p + 8200), dict(qs=127)):
        assert call(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(dh=48), dict(H=65536, qs=1 << 30), dict(n=4097), dict(rows=(1 << 20) + 1)):
        assert call(**bad) == _lib.E_UNSUPPORTED, bad
    assert call(n=0, g=0, q=None) == 0 and call(rows=0, q=None) == 0
    cache = ops.PagedCacheQ4(2, 1, 64)
    for groups, shared, dh in (([0, 1], [64, 64], 64), ([0, 1], [64], 32)):
        with pytest.raises(ValueError):
            cache.attend_shared(np.zeros((1, 2, dh)), np.zeros((1, 1)), [1], [0, 1], groups, shared)


@pytest.mark.parametrize("H,kv,dh,groups,stride,want", [
    (12, 12, 64, [(600, [(601, 1)] * 4)], None, 0),                  # nothing to gain, known from the sizes
    (12, 12, 64, [(600, [(601, 1)] * 4)], 4096, 2),                  # longer tables: a launch over shared pages, which takes them if it gains anything
    (64, 8, 128, [(130, [(133 + 5, 5)] * 30)], 4096, None),          # and leaves them where it does not
    (32, 32, 128, [(64, [(65, 4)] * 40)], 4096, None),
    (32, 32, 128, [(1300, [(1301, 1)] * 40)], None, 2),
    (64, 8, 128, [(1300, [(1301, 6)] * 30)], None, 0),       # tiles as full without sharing
    (32, 32, 128, [(640, [(650, 1)] * 20), (1300, [(1301, 1)] * 12)], 100, 2)])
def test_the_rule(H, kv, dh, groups, stride, want, way):
    """By default the way is taken that is faster; either has its own roundings."""
    from caten_amd import _lib
    rng = np.random.default_rng(22)
    cache, tables, lens, starts, borders, shared, held = answers(rng, groups, kv, dh)
    if stride:
        tables = np.concatenate([tables, np.full((len(tables), stride - tables.shape[1]), -1, np.int32)], 1)
    q = rng.normal(0, 1, (starts[-1], H, dh)).astype(np.float32)
    forced = cache.attend_shared(q, tables, lens, starts, borders, shared)
    _lib.check(_lib.load().cthip_set_option(b"shared_prefix", 1))
    got = cache.attend_shared(q, tables, lens, starts, borders, shared)
    assert want is None or np.array_equal(got, forced) == (way == want)
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *seen(q[starts[i]:starts[i + 1]], k, v, next(p // PAGE * PAGE for p, e in zip(shared, borders[1:]) if i < e)))
    for bad in (-1, 3):
        assert _lib.load().cthip_set_option(b"shared_prefix", bad) == _lib.E_BAD_ARG


@pytest.mark.parametrize("H,kv,members,prefix,piece", [(32, 32, 40, 1300, 600), (16, 8, 64, 2500, 600)])
def test_the_rule_beside_rows_of_no_group(H, kv, members, prefix, piece, way):
    """A piece of another prompt in the same step takes nothing from what the samples of one save: their pages are taken apart as they are without it."""
    from caten_amd import _lib
    rng = np.random.default_rng(24)
    print(f"case: {members} samples over {prefix} rows beside a piece of {piece}, {H} heads over {kv}", flush=True)
    cache, tables, lens, starts, borders, shared, held = answers(rng, [(prefix, [(prefix + 1 + i % 3, 1) for i in range(members)]), (0, [(piece + 50, piece)])], kv, 128)
    borders, shared = borders[:2], shared[:1]
    q = rng.normal(0, 1, (starts[-1], H, 128)).astype(np.float32)
    forced = cache.attend_shared(q, tables, lens, starts, borders, shared)
    _lib.check(_lib.load().cthip_set_option(b"shared_prefix", 1))
    got = cache.attend_shared(q, tables, lens, starts, borders, shared)
    assert np.array_equal(got, forced) == (way == 2)
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))
