"""Many sequences over one pool of pages with rows in 4 bits: block tables and slot maps, rows in and out, attention of
ragged batches.  The reference has one sequence over a dense fp32 cache (external/llm/layers.lisp:19-33) and nothing to
compare with, so each is held against its definition (include/caten_hip.h) in NumPy, in 64 bits."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
PAGE = 64


# ---------------------------------------------------------------------------------------------------------- definitions


def plan_by_hand(lens, new, tables, free, max_rows):
    """cthip_kv_plan_paged, sequence after sequence."""
    lens, new, tables = [int(v) for v in lens], [int(v) for v in new], np.array(tables)
    starts, slots, positions, left, refused, want = [0], [-1] * max_rows, [-1] * max_rows, len(free), 0, 0
    out = list(lens)
    for i, (a, b) in enumerate(zip(lens, new)):
        starts.append(starts[-1] + max(b, 0))
        ok = a >= 0 and b >= 0 and a + b <= tables.shape[1] * PAGE and starts[-1] <= max_rows
        need = -(-(a + b) // PAGE) - -(-a // PAGE) if ok else 0
        first = want
        want += need
        if not ok or (need and want > len(free)):
            refused += 1
            continue
        for k in range(need):
            tables[i, -(-a // PAGE) + k] = free[len(free) - 1 - first - k]
            left -= 1
        for j in range(b):
            positions[starts[i] + j] = a + j
            page = tables[i, (a + j) // PAGE]
            slots[starts[i] + j] = page * PAGE + (a + j) % PAGE if page >= 0 else -1
        out[i] = a + b
    return dict(slots=slots, positions=positions, starts=starts, tables=tables, lens=out, n_free=left, refused=refused)


def quantised(x):
    """What the cache holds of rows (..., dh): per block of 32 the fp16 scale and the numbers, in 64 bits."""
    b = np.asarray(x, np.float64).reshape(-1, 32)
    out = np.empty_like(b)
    for r, row in enumerate(b):
        if not np.isfinite(row).all():
            out[r] = np.nan
            continue
        m = row.max() if row.max() >= -row.min() else row.min()
        d = float(np.float16(min(max(m / -8, -65504.0), 65504.0)))
        out[r] = 0.0 if d == 0 else d * (np.clip(np.floor(row / d + 8.5), 0, 15) - 8)
    return out.reshape(np.shape(x))


def attention(q, k, v):
    """q (rows, H, dh) the last rows of a sequence with keys k, values v (T, Hkv, dh), in 64 bits; and how large its scores'
    terms and its values are, for the tolerance."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rows, H, dh = q.shape
    T, G = k.shape[0], H // k.shape[1]
    out, size, big = np.zeros(q.shape), np.zeros((rows, H)), np.zeros((rows, H))
    for r in range(rows):
        t = T - rows + r + 1
        if t <= 0:
            continue
        for h in range(H):
            kk, vv = k[:t, h // G], v[:t, h // G]
            s = kk @ q[r, h] / np.sqrt(dh)
            p = np.exp(s - s.max())
            out[r, h] = p @ vv / p.sum()
            size[r, h] = (np.abs(kk) @ np.abs(q[r, h])).max() / np.sqrt(dh)
            big[r, h] = np.abs(vv).max()
    return out, size, big


def close(got, want, size, big):
    """Half a step of a 22-bit number is 2^-22 of the largest.  Of a page's 64 probabilities times scales, each off by that
    much of the largest of them and times a number up to 8: at most 2^-13 of the largest p d, 2^-16 of the largest p v, and
    the largest p of all pages sum to at most 1.  A score is off by 2^-22 of its terms' sum from q, and by at most four fp32
    roundings of it (2^-22); weights then by twice that.  The rest (fp32 sums over pages, exponentials) is
    below 2^-16 for the lengths here."""
    tol = big * (2.0 ** -15 + size * 2.0 ** -19)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol[..., None]).all(), float(np.max(np.abs(got - want) / np.maximum(tol[..., None], 1e-30)))


def batch(rng, lens, rows, kv, dh, spare=3, scale=1.0):
    """A cache with sequences of these lengths in pages in any order; (cache, tables, starts, [(k, v)])."""
    from caten_amd import ops
    stride = max(1, max(-(-n // PAGE) for n in lens))
    pages = list(rng.permutation(sum(-(-n // PAGE) for n in lens) + spare))
    cache = ops.PagedCacheQ4(len(pages), kv, dh)
    # what the pages hold where no row was written must not matter: NaN scales, any quants
    _fill(cache, 0xff)
    tables = np.full((len(lens), stride), -1, np.int32)
    held = []
    for i, n in enumerate(lens):
        mine = [pages.pop() for _ in range(-(-n // PAGE))]
        tables[i, :len(mine)] = mine
        k = (rng.normal(0, 1, (n, kv, dh)) * np.exp(0.5 * rng.normal(0, 1, (1, kv, dh))) * scale).astype(np.float32)
        v = (rng.normal(0, 1, (n, kv, dh)) * np.exp(0.5 * rng.normal(0, 1, (1, kv, dh)))).astype(np.float32)
        slots = np.array([mine[t // PAGE] * PAGE + t % PAGE for t in range(n)], np.int32)
        if n:
            cache.append(k, v, slots)
            k, v = cache.rows(slots)
        held.append((k, v))
    return cache, tables, np.concatenate([[0], np.cumsum(rows)]).astype(np.int32), held


def _fill(cache, byte):
    from caten_amd import _lib
    for pool in (cache.k, cache.v):
        _lib.check(_lib.load().cthip_memset(pool.ptr, byte, pool.nbytes))


def attend_over(value, cache, q, tables, lens, starts):
    """PagedCacheQ4.attend into an array that holds `value`."""
    from caten_amd import _lib, ops
    n, H, dh = q.shape
    dq, dt, dl, ds = (ops.DeviceArray.from_numpy(np.ascontiguousarray(a, t)) for a, t in ((q, np.float32), (tables, np.int32), (lens, np.int32), (starts, np.int32)))
    out = ops.DeviceArray.from_numpy(np.full(q.shape, value, np.float32))
    _lib.check(_lib.load().cthip_sdpa_paged_q4(out.ptr, dq.ptr, H * dh, cache.k.ptr, cache.v.ptr, cache.n_pages, dt.ptr, tables.shape[1], dl.ptr, ds.ptr, len(lens), n, H, cache.kv_heads, dh,
                                               cache.workspace.ptr))
    return out.numpy()


# ------------------------------------------------------------------------------------------------------------- planning


@pytest.mark.parametrize("n,new,table,spare,max_rows", [
    (1, 1, 4, 5, 1), (1, 0, 4, 0, 0), (3, 1, 4, 3, 10), (64, 1, 32, 64, 64), (64, 1, 32, 3, 64), (7, 200, 8, 40, 900), (7, 200, 8, 4, 900), (9, 100, 16, 40, 300),
    (500, 70, 16, 2000, 20000), (500, 70, 16, 300, 20000), (1025, 3, 4, 900, 3000), (4096, 5, 8, 3000, 9000), (2000, 40, 8, 9000, 40000)])
def test_plan(n, new, table, spare, max_rows):
    print(f"case: plan {n} sequences, up to {new} new, {table} pages a row, {spare} free, {max_rows} rows", flush=True)
    from caten_amd import ops
    rng = np.random.default_rng(n + new)
    lens = rng.integers(0, table * PAGE + 1, n)
    lens[:: 5] = lens[:: 5] // PAGE * PAGE  # on a border of two pages
    add = rng.integers(0, new + 1, n) if new > 1 else np.full(n, new)
    add[3::11] = 0
    lens[4::13] = np.minimum(lens[4::13], 3)
    if n > 20:
        add[17], lens[18] = -2, -1
    ids = rng.permutation(n * table + spare)
    tables = np.full((n, table), -1, np.int32)
    at = 0
    for i, v in enumerate(lens):
        c = -(-max(v, 0) // PAGE)
        tables[i, :c] = ids[at:at + c]
        at += c
    free = ids[at:at + spare].astype(np.int32)
    want = plan_by_hand(lens, add, tables, free, max_rows)
    got = ops.kv_plan(lens, add, tables, np.concatenate([free, [12345] * 3]), max_rows, n_free=spare)  # (behind the stack's end)
    for key in want:
        assert np.array_equal(got[key], want[key]), key


def test_plan_of_nothing():
    from caten_amd import ops
    got = ops.kv_plan(np.zeros(0), np.zeros(0), np.zeros((0, 4)), [7, 8], 5)
    assert (got["slots"] == -1).all() and (got["positions"] == -1).all() and got["starts"][0] == 0 and got["n_free"] == 2 and got["refused"] == 0
    got = ops.kv_plan([64, 0, 3], [0, 0, 0], -np.ones((3, 4)), [], 0)
    assert not got["starts"].any() and list(got["lens"]) == [64, 0, 3] and got["refused"] == 0
    got = ops.kv_plan([64, 0, 3], [1, 0, 1], np.array([[5, -1], [-1, -1], [6, -1]]), [], 2)  # no page left for the first
    assert list(got["slots"]) == [-1, 6 * PAGE + 3] and list(got["lens"]) == [64, 0, 4] and got["refused"] == 1


def test_plan_out_of_place_leaves_its_inputs():
    from caten_amd import _lib
    from caten_amd.ops import DeviceArray
    lib = _lib.init()
    lens, new, free = np.array([64, 0, 130, 5], np.int32), np.array([3, 70, 1, 0], np.int32), np.arange(50, 60, dtype=np.int32)
    tables = np.full((4, 6), -1, np.int32)
    tables[0, 0], tables[2, :3], tables[3, 0] = 1, (2, 3, 4), 5
    d = {k: DeviceArray.from_numpy(v) for k, v in dict(lens=lens, new=new, free=free, tables=tables, n=np.array([10], np.int32)).items()}
    o = {k: DeviceArray((m,), np.int32) for k, m in dict(slots=80, starts=5, lens=4, n=1, refused=1).items()}
    for _ in range(2):  # the same call again gives the same
        _lib.check(lib.cthip_kv_plan_paged(o["slots"].ptr, None, o["starts"].ptr, d["tables"].ptr, 6, o["lens"].ptr, o["n"].ptr, o["refused"].ptr, d["lens"].ptr, d["new"].ptr,
                                           4, d["free"].ptr, d["n"].ptr, 80))
        want = plan_by_hand(lens, new, tables, list(free), 80)
        assert np.array_equal(o["slots"].numpy(), want["slots"]) and np.array_equal(d["tables"].numpy(), want["tables"])
        assert np.array_equal(o["lens"].numpy(), want["lens"]) and o["n"].numpy()[0] == want["n_free"] and o["refused"].numpy()[0] == 0
        assert np.array_equal(d["lens"].numpy(), lens) and d["n"].numpy()[0] == 10 and np.array_equal(d["free"].numpy(), free)


# ------------------------------------------------------------------------------------------------------- rows in and out


@pytest.mark.parametrize("kv,dh,rows", [(1, 32, 1), (12, 64, 48), (3, 32, 200), (8, 128, 130), (32, 128, 3), (5, 64, 1000), (17, 64, 1100), (32, 32, 1024), (8, 128, 1025)])
def test_rows_in_and_out(kv, dh, rows):
    print(f"case: rows {kv} heads of {dh}, {rows} rows", flush=True)
    from caten_amd import ops
    rng = np.random.default_rng(kv * dh + rows)
    k, v = (rng.normal(0, 1, (rows, kv, dh)).astype(np.float32) * np.exp(rng.normal(0, 2, (rows, kv, 1))).astype(np.float32) for _ in range(2))
    r = rows // 2
    k[r, 0, :32] = 0.0                                     # a block of zeros
    v[r, 0, :32] = np.tile([1.0, -1.0], 16)                # two values of the largest magnitude
    k[rows - 1, kv - 1, -32:] = np.linspace(-8, 7, 32)     # with d = 1: values on the borders between two numbers
    k[rows - 1, kv - 1, -1], k[rows - 1, kv - 1, -2] = -8.0, -7.5
    cache = ops.PagedCacheQ4(-(-rows // PAGE) + 4, kv, dh)
    slots = rng.permutation(cache.n_pages * PAGE)[:rows].astype(np.int32)
    cache.append(k, v, slots)
    got_k, got_v = cache.rows(slots)
    assert np.array_equal(got_k, quantised(k)) and np.array_equal(got_v, quantised(v))
    # half a step of the block's scale, or a whole one at the end of the range that has seven steps: |m| - 7 d there, and d, rounded
    # to 11 bits, is |m| / 8 (1 - 2^-11) at least: |m| / 8 (1 + 7 * 2^-11) < |m| / 8 (1 + 2^-8)
    for x, got in ((k, got_k), (v, got_v)):
        b, top = x.reshape(-1, 32).astype(np.float64), np.abs(x.reshape(-1, 32)).max(1, keepdims=True)
        assert (np.abs(got.reshape(-1, 32) - b) <= top / 8 * (1 + 2.0 ** -8)).all()


def test_values_at_the_ends_of_the_range():
    from caten_amd import ops
    tiny, big = np.float32(1e-45), np.float32(3e38)
    rows = np.zeros((8, 1, 32), np.float32)
    rows[0] = np.linspace(-1, 1, 32)
    rows[1, 0, 3], rows[2, 0, 4] = np.inf, np.nan
    rows[3, 0, 5], rows[4, 0, 6] = big, -big               # scales held within fp16
    rows[5, 0, 7], rows[5, 0, 8] = tiny, -tiny
    rows[6, 0, :] = np.linspace(-5e-7, 4e-7, 32)           # subnormal scales
    rows[7, 0, :] = np.linspace(-6e4, 5e5, 32)
    cache = ops.PagedCacheQ4(1, 1, 32)
    slots = np.arange(8, dtype=np.int32)
    cache.append(rows, -rows, slots)
    k, v = cache.rows(slots)
    assert np.array_equal(k, quantised(rows), equal_nan=True) and np.array_equal(v, quantised(-rows), equal_nan=True)
    assert np.isnan(k[1]).all() and np.isnan(k[2]).all() and np.isfinite(np.delete(k, [1, 2], 0)).all()


def test_strided_rows_and_slots_outside_the_pool():
    from caten_amd import _lib, ops
    rng = np.random.default_rng(5)
    lib, kv, dh, rows, width = _lib.init(), 2, 64, 37, 5 * 128 + 3
    fused = rng.normal(0, 1, (rows, width)).astype(np.float32)
    cache = ops.PagedCacheQ4(2, kv, dh)
    _fill(cache, 0x5a)
    before = cache.k.numpy(), cache.v.numpy()
    slots = rng.permutation(2 * PAGE)[:rows].astype(np.int32)
    slots[[3, 5, 9]] = -1, 2 * PAGE, 2 ** 31 - 1
    src, ds = ops.DeviceArray.from_numpy(fused), ops.DeviceArray.from_numpy(slots)
    # slices that begin at addresses of 4 bytes' alignment
    _lib.check(lib.cthip_kv_append_paged_q4(cache.k.ptr, cache.v.ptr, src.ptr + 4 * 129, src.ptr + 4 * 259, width, width, ds.ptr, rows, 2, kv, dh))
    fine = (slots >= 0) & (slots < 2 * PAGE)
    k, v = cache.rows(slots[fine])
    assert np.array_equal(k, quantised(fused[fine, 129:257]).reshape(-1, kv, dh)) and np.array_equal(v, quantised(fused[fine, 259:387]).reshape(-1, kv, dh))
    # every byte outside those rows is as it was
    for pool, old in zip((cache.k, cache.v), before):
        same = (pool.numpy() == old).reshape(2, kv, 36 * dh)
        assert (~same).sum() <= fine.sum() * kv * 36 * dh // PAGE
    untouched = np.setdiff1d(np.arange(2 * PAGE), slots)
    k2, v2 = cache.rows(untouched)
    _fill(cache, 0x5a)
    k3, v3 = cache.rows(untouched)
    assert np.array_equal(k2, k3) and np.array_equal(v2, v3)
    # reading back: rows outside the pool stay as they were, either output may be left out
    out = ops.DeviceArray.from_numpy(np.full((rows, kv * dh), 7.0, np.float32))
    _lib.check(lib.cthip_kv_rows_paged_q4(None, out.ptr, None, cache.v.ptr, ds.ptr, rows, 2, kv, dh))
    got = out.numpy()
    assert (got[~fine] == 7.0).all() and not (got[fine] == 7.0).any()


@pytest.mark.parametrize("kv,dh,offset,rows", [(3, 64, 17, 200), (40, 32, 0, 900), (17, 64, 17, 1000), (9, 128, 63, 1000), (33, 64, 1, 513), (64, 32, 61, 640), (8, 128, 0, 64 * 16 + 3)])
def test_rows_of_a_prompt(kv, dh, offset, rows):
    """Slots that follow one another, from anywhere in a page on, pages in any order; one row of the third 64 is left out."""
    print(f"case: prompt of {rows} rows from row {offset} on, {kv} heads of {dh}", flush=True)
    from caten_amd import ops
    rng = np.random.default_rng(offset + rows)
    cache = ops.PagedCacheQ4(-(-(offset + rows) // PAGE) + 2, kv, dh)
    _fill(cache, 0x5a)
    pages = rng.permutation(cache.n_pages)
    at = offset + np.arange(rows)
    slots = (pages[at // PAGE] * PAGE + at % PAGE).astype(np.int32)
    left_out = 140 if rows > 180 else rows - 1
    there = np.arange(rows) != left_out
    others = np.setdiff1d(np.arange(cache.n_pages * PAGE), slots[there]).astype(np.int32)
    before = cache.rows(others)
    k, v = (rng.normal(0, 1, (rows, kv, dh)).astype(np.float32) for _ in range(2))
    given = np.where(there, slots, -1)
    cache.append(k, v, given)
    got_k, got_v = cache.rows(given)
    assert np.array_equal(got_k[there], quantised(k[there])) and np.array_equal(got_v[there], quantised(v[there]))
    assert not got_k[left_out].any() and not got_v[left_out].any()
    one_by_one = [cache.rows(given[i:i + 1]) for i in range(0, rows, 37)]  # (a few rows take another kernel)
    assert all(np.array_equal(a[0], got_k[i]) and np.array_equal(b[0], got_v[i]) for i, (a, b) in zip(range(0, rows, 37), one_by_one))
    assert all(np.array_equal(a, b) for a, b in zip(before, cache.rows(others)))
    # the same rows, one at a time, are the same bytes
    whole = cache.k.numpy(), cache.v.numpy()
    _fill(cache, 0x5a)
    for i in range(0, rows, 100):
        cache.append(k[i:i + 100], v[i:i + 100], given[i:i + 100])
    assert np.array_equal(whole[0], cache.k.numpy()) and np.array_equal(whole[1], cache.v.numpy())


def test_places_past_32_bits():
    """A pool of more than 2^32 bytes, its last pages in use."""
    from caten_amd import ops
    rng = np.random.default_rng(21)
    kv, dh, n_pages = 32, 128, 30000  # 4.4 GB a pool
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    lens, H = [130, 200], 32
    tables = np.array([[n_pages - 1, 3, n_pages - 2, -1], [n_pages - 3, n_pages - 4, 5, n_pages - 5]], np.int32)
    held = []
    for i, n in enumerate(lens):
        slots = np.array([tables[i, t // PAGE] * PAGE + t % PAGE for t in range(n)], np.int32)
        k, v = (rng.normal(0, 1, (n, kv, dh)).astype(np.float32) for _ in range(2))
        cache.append(k, v, slots)
        held.append(cache.rows(slots))
        assert np.array_equal(held[-1][0], quantised(k)) and np.array_equal(held[-1][1], quantised(v))
    q = rng.normal(0, 1, (2, H, dh)).astype(np.float32)
    got = cache.attend(q, tables, lens, [0, 1, 2])
    for i, (k, v) in enumerate(held):
        close(got[i:i + 1], *attention(q[i:i + 1], k, v))


# ------------------------------------------------------------------------------------------------------------ attention

SHAPES = [(12, 12, 64), (32, 4, 64), (8, 1, 128), (4, 4, 128), (6, 2, 32), (16, 1, 32), (21, 3, 128), (10, 5, 64), (17, 1, 64)]


@pytest.mark.parametrize("H,kv,dh", SHAPES)
@pytest.mark.parametrize("lens", [[1], [2], [63, 64, 65], [0, 128, 1, 0, 300, 129], [700]])
def test_single_rows(H, kv, dh, lens):
    print(f"case: one row each, {H} heads over {kv} of {dh}, lengths {lens}", flush=True)
    rng = np.random.default_rng(H + dh + len(lens))
    rows = [min(n, 1) for n in lens]
    cache, tables, starts, held = batch(rng, lens, rows, kv, dh)
    q = rng.normal(0, 1, (sum(rows), H, dh)).astype(np.float32)
    got = cache.attend(q, tables, lens, starts)
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


@pytest.mark.parametrize("H,kv,dh", SHAPES)
@pytest.mark.parametrize("lens,rows", [([2], [2]), ([5, 70, 3], [5, 3, 1]), ([200, 64, 65, 0, 90], [17, 64, 2, 0, 33]), ([150], [150]), ([131, 333], [67, 16])])
def test_several_rows(H, kv, dh, lens, rows):
    print(f"case: {rows} rows, {H} heads over {kv} of {dh}, lengths {lens}", flush=True)
    rng = np.random.default_rng(H * dh + sum(rows))
    cache, tables, starts, held = batch(rng, lens, rows, kv, dh)
    q = rng.normal(0, 1, (sum(rows), H, dh)).astype(np.float32)
    got = cache.attend(q, tables, lens, starts)
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


@pytest.mark.parametrize("H,kv,dh,lens,rows", [(8, 8, 128, [9000, 40], [1, 1]), (8, 2, 64, [12345], [1]), (8, 1, 32, [4100, 4099, 77], [3, 1, 20]), (4, 1, 128, [6000], [40]), (4, 1, 64, [100000], [2]),
                                               (17, 1, 128, [60000], [1]), (6, 2, 32, [90000, 5], [1, 1])])
def test_long_sequences(H, kv, dh, lens, rows):
    """Split over workgroups and joined; the sequences' lengths far apart."""
    print(f"case: long {lens} {rows}, {H} heads over {kv} of {dh}", flush=True)
    rng = np.random.default_rng(sum(lens))
    cache, tables, starts, held = batch(rng, lens, rows, kv, dh)
    q = rng.normal(0, 1, (sum(rows), H, dh)).astype(np.float32)
    got = cache.attend(q, tables, lens, starts)
    again = cache.attend(q, tables, lens, starts)
    assert np.array_equal(got, again)  # joined in an order of its own, whichever workgroup comes last
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


@pytest.mark.parametrize("H,kv", [(4, 4), (16, 2), (40, 2)])
def test_many_sequences(H, kv):
    rng = np.random.default_rng(H)
    lens = rng.integers(0, 150, 130)
    rows = np.minimum(lens, rng.choice([0, 1, 1, 1, 5], 130))
    cache, tables, starts, held = batch(rng, list(lens), list(rows), kv, 64)
    q = rng.normal(0, 1, (rows.sum(), H, 64)).astype(np.float32)
    got = cache.attend(q, tables, lens, starts)
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


@pytest.mark.parametrize("H,kv,rows", [(4, 4, 1), (8, 1, 1), (8, 2, 20)])
def test_rows_that_see_nothing_and_rows_behind_the_last(H, kv, rows):
    """A table entry outside the pool is a page without keys; a row without any key is zero; rows behind starts[n] stay."""
    from caten_amd import _lib, ops
    rng = np.random.default_rng(H * rows)
    lib, dh, lens = _lib.init(), 64, [200, 64, 130]
    cache, tables, starts, held = batch(rng, lens, [rows] * 3, kv, dh)
    tables[0, 1], tables[1, 0], tables[2, 0] = -1, cache.n_pages, 2 ** 31 - 1
    lens[2] = 64  # (its only page is outside the pool)
    n = 3 * rows + 5
    q = rng.normal(0, 1, (n, H, dh)).astype(np.float32)
    q[3 * rows:] = np.nan
    dq, dt, dl, ds = (ops.DeviceArray.from_numpy(np.asarray(a, t)) for a, t in ((q, np.float32), (tables, np.int32), (lens, np.int32), (starts, np.int32)))
    out = ops.DeviceArray.from_numpy(np.full(q.shape, 7.0, np.float32))
    _lib.check(lib.cthip_sdpa_paged_q4(out.ptr, dq.ptr, H * dh, cache.k.ptr, cache.v.ptr, cache.n_pages, dt.ptr, tables.shape[1], dl.ptr, ds.ptr, 3, n, H, kv, dh, cache.workspace.ptr))
    got = out.numpy()
    assert (got[3 * rows:] == 7.0).all() and (got[rows:3 * rows] == 0.0).all()
    k, v = held[0]
    for r in range(rows):
        t = 200 - rows + r + 1
        keep = [x for x in range(t) if x // PAGE != 1]
        close(got[r:r + 1], *attention(q[r:r + 1], k[keep], v[keep]))


def test_a_very_long_sequence():
    """More pages than a wavefront holds the ids of: over a million keys of one narrow head."""
    from caten_amd import ops
    rng = np.random.default_rng(22)
    T, kv, dh, H = 1100000, 1, 32, 3
    n_pages = -(-T // PAGE)
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    tables = rng.permutation(n_pages).astype(np.int32)[None]
    slots = (tables[0].astype(np.int64)[np.arange(T) // PAGE] * PAGE + np.arange(T) % PAGE).astype(np.int32)
    k, v = (rng.standard_normal((T, kv, dh), np.float32) for _ in range(2))
    k[::, 0] *= (1 + np.arange(T) % 3)[:, None]
    cache.append(k, v, slots)
    k, v = cache.rows(slots)
    q = rng.normal(0, 1, (2, H, dh)).astype(np.float32)
    got = cache.attend(q, tables, [T], [0, 2])
    want, size, big = attention(q, k, v)
    # sums of 1.1e6 positive terms in 63 x 4 pieces of some 70 pages: off by a few hundred roundings of 2^-24 at most, against 2^-16 allowed for
    close(got, want, size, big)


@pytest.mark.parametrize("H,kv,dh", [(4, 2, 64), (16, 1, 128), (3, 3, 32)])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("factors", [(1e-6,), (1e-3,), (30,), (1e5,), (1e-4, 1, 1e3), (1e3, 1, 1e-2), (0, 1), (1, 0, 50)])
def test_sizes_of_values(H, kv, dh, rows, factors):
    """Values from where a block's scale is subnormal to where it is the largest there is, alike or different page by page."""
    from caten_amd import ops
    rng = np.random.default_rng(dh + rows)
    T = 40 * PAGE + 30
    cache, tables, starts, held = batch(rng, [T], [rows], kv, dh)
    slots = np.array([tables[0, t // PAGE] * PAGE + t % PAGE for t in range(T)], np.int32)
    factor = np.array(factors)[np.arange(T) // PAGE * len(factors) // (T // PAGE + 1)].astype(np.float32)
    k, v = held[0][0], held[0][1] * factor[:, None, None]
    cache.append(k, v, slots)
    k, v = cache.rows(slots)
    q = rng.normal(0, 1, (rows, H, dh)).astype(np.float32)
    close(cache.attend(q, tables, [T], starts), *attention(q, k, v))


@pytest.mark.parametrize("factor", [1e-30, 1e-4, 3e3, 1e6, 1e9, 1e25])
def test_sizes_of_queries(factor):
    """Scores that are all alike, and scores of which the largest alone counts, up to where fp32 does not tell neighbours apart."""
    rng = np.random.default_rng(24)
    for H, kv, dh, rows in ((4, 2, 64, 1), (8, 1, 32, 20)):
        T = 500
        cache, tables, starts, held = batch(rng, [T], [rows], kv, dh)
        q = (rng.normal(0, 1, (rows, H, dh)) * factor).astype(np.float32)
        got = cache.attend(q, tables, [T], starts)
        want, size, big = attention(q, *held[0])
        if factor < 1e5:
            close(got, want, size, big)
            continue
        # a score is off by what 2^-22 of its terms' sum is: keys that near the largest may have any share, others none
        for r in range(rows):
            for h in range(H):
                k, v = (a[:T - rows + r + 1, h // (H // kv)].astype(np.float64) for a in held[0])
                s = k @ q[r, h].astype(np.float64) / np.sqrt(dh)
                near = s >= s.max() - size[r, h] * 2.0 ** -19 - 20
                assert np.isfinite(got[r, h]).all()
                slack = big[r, h] * 2.0 ** -15
                assert (got[r, h] >= v[near].min(0) - slack).all() and (got[r, h] <= v[near].max(0) + slack).all()


def test_starts_in_any_order():
    """Rows in front of an earlier sequence's are nobody's; a negative length is none.  The workspace stays as it was."""
    rng = np.random.default_rng(25)
    kv, dh, H = 2, 64, 4
    lens = [5000, 300, 200, 100] + [40] * 100
    cache, tables, _, held = batch(rng, lens, [0] * len(lens), kv, dh)
    n = 12
    q = rng.normal(0, 1, (n, H, dh)).astype(np.float32)

    def call(starts, lens):
        return attend_over(7.0, cache, q, tables, lens, starts)

    def whose(got, rows, i):
        close(got[rows], *attention(q[rows], *held[i]))

    got = call([0, 2, 1, 3, 4] + [4] * 100, lens)  # sequence 1 ends in front of its start, sequence 2's row 1 is sequence 0's
    whose(got, slice(0, 2), 0)
    whose(got, slice(3, 4), 3)
    assert (got[2] == 7.0).all() and (got[4:] == 7.0).all()
    got = call([-3, 2, 4, 2 ** 31 - 1, 5] + [0] * 99 + [3], lens)
    whose(got, slice(2, 4), 1)
    whose(got, slice(4, 12), 2)
    assert (got[:2] == 7.0).all()
    many = [0] * 70 + [9] + [1, 9, 10] * 10 + [4, 12, 11]  # behind the first 64
    got = call(many + [11], lens)
    whose(got, slice(0, 9), 69)
    owner = [i for i in range(len(lens)) if many[i] == 9 and (many + [11])[i + 1] == 10][0]
    whose(got, slice(9, 10), owner)
    starts = np.minimum(np.arange(len(lens) + 1), 4)
    got = call(starts, [5000, -1, -2 ** 31, 100] + [40] * 100)
    whose(got, slice(0, 1), 0)
    whose(got, slice(3, 4), 3)
    assert not got[1:3].any()
    assert not cache.workspace.numpy()[:4 * 2048].any()


@pytest.mark.parametrize("H,kv,dh", [(4, 4, 32), (20, 1, 64), (8, 2, 128)])
def test_sequences_without_keys(H, kv, dh):
    """Their rows are zero, wherever they lie between the others."""
    rng = np.random.default_rng(H)
    for n, share in ((1, 1.0), (5, 0.5), (700, 0.5), (700, 1.0)):
        lens = np.where(rng.uniform(0, 1, n) < share, 0, rng.integers(1, 300, n))
        rows = np.where(lens == 0, rng.integers(1, 4, n), np.minimum(lens, rng.integers(0, 3, n)))
        cache, tables, starts, held = batch(rng, list(lens), list(rows), kv, dh)
        q = rng.normal(0, 1, (rows.sum(), H, dh)).astype(np.float32)
        got = attend_over(7.0, cache, q, tables, lens, starts)
        for i, (k, v) in enumerate(held):
            mine = slice(starts[i], starts[i + 1])
            if lens[i] == 0:
                assert not got[mine].any()
            else:
                close(got[mine], *attention(q[mine], k, v))


def test_nothing_in_the_pool():
    from caten_amd import _lib, ops
    lib, out = _lib.init(), ops.DeviceArray.from_numpy(np.full((3, 2, 32), 7.0, np.float32))
    ws = ops.DeviceArray((int(lib.cthip_sdpa_paged_q4_workspace(32)),), np.uint8)
    q, t, lens, starts = (ops.DeviceArray.from_numpy(a) for a in (np.ones((3, 2, 32), np.float32), np.zeros((2, 4), np.int32), np.array([9, 0], np.int32), np.array([0, 1, 2], np.int32)))
    _lib.check(lib.cthip_sdpa_paged_q4(out.ptr, q.ptr, 64, None, None, 0, t.ptr, 4, lens.ptr, starts.ptr, 2, 3, 2, 1, 32, ws.ptr))
    got = out.numpy()
    assert not got[:2].any() and (got[2] == 7.0).all()


def test_more_rows_than_keys_and_a_table_that_is_too_short():
    rng = np.random.default_rng(11)
    cache, tables, starts, held = batch(rng, [3, 200], [8, 1], 2, 64)
    q = rng.normal(0, 1, (9, 4, 64)).astype(np.float32)
    got = cache.attend(q, np.ascontiguousarray(tables[:, :2]), [3, 200], starts)
    want = attention(q[:8], *held[0])
    assert (got[:5] == 0).all()
    close(got[:8], *want)
    close(got[8:], *attention(q[8:], held[1][0][:128], held[1][1][:128]))  # keys past the table's end are not there


def test_infinities_and_nan():
    """In a row that is masked they change nothing; in one that is seen the result is NaN: everywhere with a key, in its
    block's channels with a value."""
    from caten_amd import ops
    rng = np.random.default_rng(12)
    for H, rows in ((2, 10), (16, 10), (2, 1)):
        kv, dh, T = 2, 64, 100
        cache, tables, starts, held = batch(rng, [T], [rows], kv, dh)
        q = rng.normal(0, 1, (rows, H, dh)).astype(np.float32)
        k, v = (a.copy() for a in held[0])
        clean, size, big = attention(q, k, v)
        slot = [tables[0, (T - 1) // PAGE] * PAGE + (T - 1) % PAGE]
        v[T - 1, 1, 40] = np.inf
        cache.append(k[T - 1:], v[T - 1:], slot)
        got = cache.attend(q, tables, [T], starts)
        close(got[:-1], clean[:-1], size[:-1], big[:-1])  # the last row alone sees the last key
        bad = np.isnan(got[-1])
        assert bad[H // 2:, 32:].all() and not bad[:H // 2].any() and not bad[:, :32].any()
        close(got[-1:, :, :32], clean[-1:, :, :32], size[-1:], big[-1:])
        v[T - 1], k[T - 1, 0, 3] = held[0][1][T - 1], np.nan
        cache.append(k[T - 1:], v[T - 1:], slot)
        got = cache.attend(q, tables, [T], starts)
        close(got[:-1], clean[:-1], size[:-1], big[:-1])
        assert np.isnan(got[-1, :H // 2]).all()
        close(got[-1:, H // 2:], clean[-1:, H // 2:], size[-1:, H // 2:], big[-1:, H // 2:])
        cache.append(held[0][0][T - 1:], held[0][1][T - 1:], slot)
        q[0, 0, 5] = np.nan if rows > 1 else np.inf
        got = cache.attend(q, tables, [T], starts)
        assert np.isnan(got[0, 0]).all()
        got[0, 0], clean[0, 0] = 0, 0
        close(got, clean, size, big)


@pytest.mark.parametrize("H,kv", [(4, 4), (16, 2)])
@pytest.mark.parametrize("rows", [1, 30])
def test_scores_far_apart(H, kv, rows):
    """Softmax where one key has nearly all the weight, scores in the hundreds, and values of very different sizes: a key with a
    large weight and a small value beside many with small weights and large values."""
    rng = np.random.default_rng(13 + H)
    T, dh = 500, 64
    cache, tables, starts, held = batch(rng, [T], [rows], kv, dh)
    slots = np.array([tables[0, t // PAGE] * PAGE + t % PAGE for t in range(T)], np.int32)
    q = rng.normal(0, 1, (rows, H, dh)).astype(np.float32)
    k, v = held[0]
    got = cache.attend(q * 100, tables, [T], starts)
    close(got, *attention(q * 100, k, v))
    k, v = k.copy(), v.copy()
    direction = rng.normal(0, 1, (1, kv, dh))
    q = (0.3 * q + np.repeat(direction, H // kv, 1)).astype(np.float32)
    k[70] = 6 * direction[0] / np.sqrt(dh) * 2
    v[70] *= 0.001
    cache.append(k, v, slots)
    k, v = cache.rows(slots)
    got = cache.attend(q, tables, [T], starts)
    want, size, big = attention(q, k, v)
    close(got, want, size, big)
    # and as near as fp32 sums are, whatever the largest weight's value is: 2^-16 of the weighted values' sizes
    spread = np.zeros_like(want)
    for r in range(rows):
        for h in range(H):
            s = k[:T - rows + r + 1, h // (H // kv)].astype(np.float64) @ q[r, h] / np.sqrt(dh)
            p = np.exp(s - s.max())
            spread[r, h] = p @ np.abs(v[:T - rows + r + 1, h // (H // kv)]) / p.sum()
    assert (np.abs(got - want) <= spread.max(-1, keepdims=True) * (2.0 ** -15 + size[..., None] * 2.0 ** -19)).all()


def test_strided_queries():
    from caten_amd import _lib, ops
    rng = np.random.default_rng(14)
    H, kv, dh, lens = 8, 4, 64, [130, 70]
    cache, tables, starts, held = batch(rng, lens, [1, 3], kv, dh)
    fused = rng.normal(0, 1, (4, H * dh + 2 * kv * dh + 1)).astype(np.float32)
    src, dt, dl, ds = (ops.DeviceArray.from_numpy(np.asarray(a)) for a in (fused, tables, np.array(lens, np.int32), starts))
    out = ops.DeviceArray((4, H, dh), np.float32)
    _lib.check(_lib.load().cthip_sdpa_paged_q4(out.ptr, src.ptr + 4, fused.shape[1], cache.k.ptr, cache.v.ptr, cache.n_pages, dt.ptr, tables.shape[1], dl.ptr, ds.ptr, 2, 4, H, kv, dh,
                                               cache.workspace.ptr))
    q = fused[:, 1:1 + H * dh].reshape(4, H, dh)
    got = out.numpy()
    for i, (k, v) in enumerate(held):
        close(got[starts[i]:starts[i + 1]], *attention(q[starts[i]:starts[i + 1]], k, v))


# ----------------------------------------------------------------------------------------------------- a step as a whole


def test_steps_of_a_batch():
    """Prompts, then tokens one by one: every step planned, appended and attended with what the step before left on the
    device, sequences joining late and leaving; against a cache kept by hand."""
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(15)
    n, H, kv, dh, table, n_pages, max_rows = 5, 6, 3, 64, 6, 40, 400
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    _fill(cache, 0xff)
    d = {k: ops.DeviceArray.from_numpy(np.asarray(v, np.int32)) for k, v in dict(lens=[0] * n, tables=np.full((n, table), -1), free=rng.permutation(n_pages), n=[n_pages]).items()}
    o = {k: ops.DeviceArray((m,), np.int32) for k, m in dict(slots=max_rows, starts=n + 1, refused=1).items()}
    out = ops.DeviceArray((max_rows, H, dh), np.float32)
    hist = [(np.zeros((0, kv, dh), np.float32), np.zeros((0, kv, dh), np.float32)) for _ in range(n)]
    for step, new in enumerate([[130, 1, 0, 64, 70]] + [[1, 1, 0, 1, 1]] * 3 + [[1, 90, 63, 1, 0]] + [[1, 1, 1, 1, 0]] * 4):
        rows = sum(new)
        dnew = ops.DeviceArray.from_numpy(np.array(new, np.int32))
        _lib.check(lib.cthip_kv_plan_paged(o["slots"].ptr, None, o["starts"].ptr, d["tables"].ptr, table, d["lens"].ptr, d["n"].ptr, o["refused"].ptr, d["lens"].ptr, dnew.ptr, n,
                                           d["free"].ptr, d["n"].ptr, max_rows))
        qkv = rng.normal(0, 1, (max_rows, (H + 2 * kv) * dh)).astype(np.float32)
        src = ops.DeviceArray.from_numpy(qkv)
        w = qkv.shape[1]
        _lib.check(lib.cthip_kv_append_paged_q4(cache.k.ptr, cache.v.ptr, src.ptr + 4 * H * dh, src.ptr + 4 * (H + kv) * dh, w, w, o["slots"].ptr, max_rows, n_pages, kv, dh))
        _lib.check(lib.cthip_sdpa_paged_q4(out.ptr, src.ptr, w, cache.k.ptr, cache.v.ptr, n_pages, d["tables"].ptr, table, d["lens"].ptr, o["starts"].ptr, n, max_rows, H, kv, dh,
                                           cache.workspace.ptr))
        got = out.numpy()[:rows]
        assert o["refused"].numpy()[0] == 0
        at = 0
        for i, m in enumerate(new):
            k, v = (quantised(qkv[at:at + m, (H + a) * dh:(H + a + kv) * dh].reshape(m, kv, dh)).astype(np.float32) for a in (0, kv))
            hist[i] = tuple(np.concatenate([a, b]) for a, b in zip(hist[i], (k, v)))
            if m:
                close(got[at:at + m], *attention(qkv[at:at + m, :H * dh].reshape(m, H, dh), *hist[i]))
            at += m
    assert np.array_equal(d["lens"].numpy(), [len(k) for k, _ in hist])


def test_captured_steps():
    """A decode step as a graph: what it reads of lengths and tables lies on the device, so a replay is the next step.  Two
    graphs with a workspace each, eager work between the replays."""
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(16)
    stream = C.c_void_p(lib.cthip_stream())
    n, H, kv, dh, table, n_pages = 3, 8, 2, 64, 8, 24
    lens0 = [190, 62, 127]

    def fresh():
        cache = ops.PagedCacheQ4(n_pages, kv, dh)
        r = np.random.default_rng(17)
        d = {k: ops.DeviceArray.from_numpy(np.asarray(v, np.int32)) for k, v in dict(lens=[0] * n, tables=np.full((n, table), -1), free=r.permutation(n_pages), n=[n_pages], new=lens0,
                                                                                     one=[1] * n).items()}
        o = {k: ops.DeviceArray((m,), np.int32) for k, m in dict(slots=400, starts=n + 1, refused=1).items()}
        qkv = ops.DeviceArray.from_numpy(r.normal(0, 1, (400, (H + 2 * kv) * dh)).astype(np.float32))
        out = ops.DeviceArray((400, H, dh), np.float32)

        def step(new, rows):
            w = (H + 2 * kv) * dh
            _lib.check(lib.cthip_kv_plan_paged(o["slots"].ptr, None, o["starts"].ptr, d["tables"].ptr, table, d["lens"].ptr, d["n"].ptr, o["refused"].ptr, d["lens"].ptr, new.ptr, n,
                                               d["free"].ptr, d["n"].ptr, rows))
            _lib.check(lib.cthip_kv_append_paged_q4(cache.k.ptr, cache.v.ptr, qkv.ptr + 4 * H * dh, qkv.ptr + 4 * (H + kv) * dh, w, w, o["slots"].ptr, rows, n_pages, kv, dh))
            _lib.check(lib.cthip_sdpa_paged_q4(out.ptr, qkv.ptr, w, cache.k.ptr, cache.v.ptr, n_pages, d["tables"].ptr, table, d["lens"].ptr, o["starts"].ptr, n, rows, H, kv, dh,
                                               cache.workspace.ptr))

        step(d["new"], 400)
        _lib.check(lib.cthip_sync())
        return cache, d, o, qkv, out, step

    eager, graphed = fresh(), [fresh(), fresh()]
    runs = []
    for f in graphed:
        graph, run = C.c_void_p(), C.c_void_p()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        f[5](f[1]["one"], n)
        assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        runs.append((graph, run))
    for _ in range(5):
        eager[5](eager[1]["one"], n)
        want = eager[4].numpy()[:n]
        for f, (_, run) in zip(graphed, runs):
            assert lib.hipGraphLaunch(run, stream) == 0
        for f in graphed:
            assert np.array_equal(f[4].numpy()[:n], want)
            assert np.array_equal(f[1]["lens"].numpy(), eager[1]["lens"].numpy())
    for graph, run in runs:
        lib.hipGraphExecDestroy(run)
        lib.hipGraphDestroy(graph)


# ------------------------------------------------------------------------------------------------------------- refusals


def test_refusals():
    from caten_amd import HipError, _lib, ops
    lib = _lib.init()
    a = ops.DeviceArray((4096,), np.int32)
    p = a.ptr

    def refused(code, fn, *args):
        with pytest.raises(HipError) as e:
            _lib.check(fn(*args))
        assert e.value.code == code, e.value

    bad, no = _lib.E_BAD_ARG, _lib.E_UNSUPPORTED
    plan = lambda **k: [dict(dict(slots=p, pos=p, starts=p, tables=p, stride=4, lens_out=p, free_out=p, refused=p, lens=p, new=p, n=2, free=p, n_free=p, rows=8), **k)[x] for x in
                        ("slots", "pos", "starts", "tables", "stride", "lens_out", "free_out", "refused", "lens", "new", "n", "free", "n_free", "rows")]
    for change in (dict(n=-1), dict(rows=-1), dict(stride=0), dict(stride=2 ** 31 - 1), dict(slots=None), dict(starts=None), dict(tables=None), dict(lens=None), dict(new=None), dict(free=None),
                   dict(n_free=None), dict(lens_out=None), dict(free_out=None), dict(refused=None), dict(rows=2 ** 31 - 1)):
        refused(bad, lib.cthip_kv_plan_paged, *plan(**change))
    refused(no, lib.cthip_kv_plan_paged, *plan(n=4097))
    append = lambda **k: [dict(dict(k=p, v=p, kr=p, vr=p, ks=64, vs=64, slots=p, rows=1, pages=1, kv=2, dh=32), **k)[x] for x in
                          ("k", "v", "kr", "vr", "ks", "vs", "slots", "rows", "pages", "kv", "dh")]
    for change in (dict(k=None), dict(v=None), dict(kr=None), dict(vr=None), dict(slots=None), dict(ks=63), dict(vs=63), dict(rows=-1), dict(pages=-1), dict(pages=2 ** 31 - 1), dict(k=p + 8)):
        refused(bad, lib.cthip_kv_append_paged_q4, *append(**change))
    for change in (dict(dh=48), dict(dh=256), dict(kv=0), dict(kv=-3), dict(kv=70000)):
        refused(no, lib.cthip_kv_append_paged_q4, *append(**change))
    rows = lambda **k: [dict(dict(kr=p, vr=p, k=p, v=p, slots=p, rows=1, pages=1, kv=2, dh=32), **k)[x] for x in ("kr", "vr", "k", "v", "slots", "rows", "pages", "kv", "dh")]
    for change in (dict(k=None), dict(v=None), dict(slots=None), dict(rows=-1), dict(v=p + 4)):
        refused(bad, lib.cthip_kv_rows_paged_q4, *rows(**change))
    refused(no, lib.cthip_kv_rows_paged_q4, *rows(dh=40))
    attend = lambda **k: [dict(dict(out=p, q=p + 8192, qs=128, k=p, v=p, pages=1, tables=p, stride=1, lens=p, starts=p, n=1, rows=1, H=4, kv=2, dh=32, ws=p), **k)[x] for x in
                          ("out", "q", "qs", "k", "v", "pages", "tables", "stride", "lens", "starts", "n", "rows", "H", "kv", "dh", "ws")]
    for change in (dict(out=None), dict(q=None), dict(q=p), dict(k=None), dict(v=None), dict(tables=None), dict(lens=None), dict(starts=None), dict(ws=None), dict(ws=p + 4), dict(k=p + 8), dict(qs=127), dict(n=-1),
                   dict(rows=-1), dict(stride=0), dict(H=3), dict(H=0), dict(pages=-1)):
        refused(bad, lib.cthip_sdpa_paged_q4, *attend(**change))
    refused(no, lib.cthip_kv_append_paged_q4, *append(rows=2 ** 28 + 1))
    refused(no, lib.cthip_kv_rows_paged_q4, *rows(rows=2 ** 28 + 1))
    for change in (dict(dh=96, qs=1000), dict(n=4097), dict(rows=2 ** 20 + 1), dict(rows=2 ** 20, H=128, kv=1, qs=4096), dict(H=65536, kv=65536, qs=2 ** 21)):
        refused(no, lib.cthip_sdpa_paged_q4, *attend(**change))
    # nothing to do
    _lib.check(lib.cthip_kv_append_paged_q4(*append(rows=0, k=None)))
    _lib.check(lib.cthip_sdpa_paged_q4(*attend(rows=0, q=None)))
    _lib.check(lib.cthip_sdpa_paged_q4(*attend(n=0)))
    _lib.check(lib.cthip_sync())
    with pytest.raises(HipError):
        ops.PagedCacheQ4(4, 2, 48)
    with pytest.raises(ValueError):
        ops.kv_plan([1, 2], [1], np.zeros((2, 2)), [], 3)
