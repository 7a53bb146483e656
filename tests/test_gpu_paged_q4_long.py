"""Attention over the 4-bit paged cache where a call is so long, or might be, that its parts are cut in other ways: more pages a
wavefront than it holds the ids of, and pages shared out in pieces of more than four.  Tables name a few pages many times over, so that
the definition, in 64 bits, sums each page once and counts it."""
import numpy as np
import pytest

from tests.test_gpu_paged_q4 import PAGE, close

pytestmark = pytest.mark.gpu


def few_pages(rng, n_pages, kv, dh):
    from caten_amd import ops
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    slots = np.arange(n_pages * PAGE, dtype=np.int32)
    k, v = (rng.standard_normal((slots.size, kv, dh), np.float32) for _ in range(2))
    k *= (1 + np.arange(slots.size) % 3)[:, None, None] * np.float32(0.5)
    for at in range(0, slots.size, 256):
        cache.append(k[at:at + 256], v[at:at + 256], slots[at:at + 256])
    k, v = cache.rows(slots)
    return cache, k.astype(np.float64), v.astype(np.float64)


def attention_by_counts(q, k, v, table, T):
    """The last rows of a sequence of T keys in the pages of `table` (entries outside the pool: none)."""
    q = q.astype(np.float64)
    rows, H, dh = q.shape
    n_pages, kv = k.shape[0] // PAGE, k.shape[1]
    out, size, big = np.zeros(q.shape), np.zeros((rows, H)), np.zeros((rows, H))
    for r in range(rows):
        t = T - rows + r + 1
        if t <= 0:
            continue
        full = table[:t // PAGE]
        count = np.repeat(np.bincount(full[(full >= 0) & (full < n_pages)], minlength=n_pages), PAGE).astype(np.float64)
        if t % PAGE and 0 <= table[t // PAGE] < n_pages:
            count[table[t // PAGE] * PAGE:][:t % PAGE] += 1
        there = count > 0
        if not there.any():
            continue
        for h in range(H):
            kk, vv = k[there, h // (H // kv)], v[there, h // (H // kv)]
            s = kk @ q[r, h] / np.sqrt(dh)
            p = np.exp(s - s.max()) * count[there]
            out[r, h] = p @ vv / p.sum()
            size[r, h] = (np.abs(kk) @ np.abs(q[r, h])).max() / np.sqrt(dh)
            big[r, h] = np.abs(vv).max()
    return out, size, big


@pytest.mark.parametrize("H,kv,dh,shares", [(3, 1, 32, 128), (16, 1, 64, 256), (2, 1, 128, 256)])
def test_more_pages_than_a_wavefront_holds_ids_of(H, kv, dh, shares):
    """At most `shares` workgroups have a part of a tile; with 70 pieces of four pages each, a wavefront has 70 pages, and the ids of 64."""
    rng = np.random.default_rng(41 + dh)
    pages = (shares - 1) * 70 * 4 - 9
    T = pages * PAGE - 23
    pieces = -(-pages // 4) + 1
    assert -(-pieces // (shares - 1)) > 64  # of a part, and so pages of a wavefront
    print(f"case: {T} keys, {H} heads over {kv} of {dh}", flush=True)
    cache, k, v = few_pages(rng, 37, kv, dh)
    table = rng.integers(0, 37, pages).astype(np.int32)
    table[rng.integers(0, pages, pages // 50)] = -1
    table[5000:5300] = 37  # (a stretch without keys)
    q = rng.normal(0, 1, (2, H, dh)).astype(np.float32)
    got = cache.attend(q, table[None], [T], [0, 2])
    assert np.array_equal(got, cache.attend(q, table[None], [T], [0, 2]))
    # (sums of some 2^12 keys a wavefront and 2^8 shares are off by less than 2^-16, as for the shorter ones)
    close(got, *attention_by_counts(q, k, v, table, T))


@pytest.mark.parametrize("stride,rows", [(2 ** 20 + 5, [1, 1]), (2 ** 22 + 3, [1, 1]), (2 ** 21, [20, 3]), (2 ** 24, [0, 1])])
def test_larger_pieces(stride, rows):
    """Tables so wide that the line of all costs would pass 2^30 in pieces of four pages."""
    rng = np.random.default_rng(stride % 1000 + rows[0])
    kv, dh, n_pages, lens = 4096, 32, 7, [20000, 333]
    tiles = sum(rows) // 16 + min(2, sum(rows))
    piece = 2
    while tiles * kv * ((stride >> piece) + 2) > 2 ** 30 - 1:
        piece += 1
    assert piece > 2
    print(f"case: tables of {stride}, rows {rows}, pieces of {1 << piece} pages", flush=True)
    cache, k, v = few_pages(rng, n_pages, kv, dh)
    tables = np.full((2, stride), -1, np.int32)
    for i, n in enumerate(lens):
        tables[i, :-(-n // PAGE)] = rng.integers(0, n_pages, -(-n // PAGE))
    tables[0, 100:104] = -1
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    q = rng.normal(0, 1, (sum(rows), kv, dh)).astype(np.float32)
    got = cache.attend(q, tables, lens, starts)
    some = np.concatenate([[0, 1, kv - 1], rng.integers(0, kv, 60)])
    for i, n in enumerate(lens):
        mine = slice(starts[i], starts[i + 1])
        close(got[mine][:, some], *attention_by_counts(q[mine][:, some], k[:, some], v[:, some], tables[i], n))
    # all heads against a narrower table's result, cut in pieces of four pages: both are within the bound of the definition
    again = cache.attend(q, np.ascontiguousarray(tables[:, :400]), lens, starts)
    size = np.stack([np.einsum("thc,hc->th", np.abs(k), np.abs(x)).max(0) for x in q.astype(np.float64)]) / np.sqrt(dh)
    close(got, again, 2 * size, 2 * np.broadcast_to(np.abs(v).max((0, 2)), size.shape))
