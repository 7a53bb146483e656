"""Attention over the 4-bit paged cache where every rounding can be counted: few keys have a weight at all, so sums have few
terms and the bound is near what the products themselves lose.  Held against the definition in NumPy, in 64 bits, channel by
channel: a channel's error is measured by its own weighted values, not by the largest of the head."""
import numpy as np
import pytest

from tests.test_gpu_paged_q4 import PAGE, batch

pytestmark = pytest.mark.gpu


def sparse_keys(rng, T, kv, dh, live):
    """Keys of which all but `live` score some hundreds below the others for queries from `gated_queries` (their weights are
    exactly zero in fp32), the live ones with two channels a block that are not zero."""
    k = np.zeros((T, kv, dh), np.float32)
    k[:, :, 0] = -4000.0
    for t in live:
        k[t] = 0.0
        for h in range(kv):
            for b in range(dh // 32):
                k[t, h, 32 * b + 1 + rng.permutation(31)[:2]] = rng.normal(0, 2.0, 2)
    return k


def gated_queries(rng, rows, H, dh):
    q = rng.normal(0, 1, (rows, H, dh)).astype(np.float32)
    q[:, :, 0] = 2.0
    return q


def channels(q, k, v, p_of=None, q_of=None):
    """(out, tolerance) of the last rows of a sequence, channel by channel; p_of / q_of: what a poorer kernel would make of
    weights (of the largest) times scales and of queries.

    Of one live key, per unit of its weighted value:
      q     two fp16 terms of the row's largest: off by 2^-23 of it; times the key's channels: q_err
      score a sum of 2 channels a block in two terms (4 additions a block), a scale and an addition a block, a weight: 6 NB + 2 roundings of
            2^-23 (a matrix instruction may cut off) of the terms' sum
      exponential  the argument, below 16 for weights above 2^-30, rounded: ln 2 * 16 * 2^-24 < 2^-20; itself 2^-22
      p d   p as two terms 2^-22, the products' second term 2^-22; the fp32 form less.  Half a step of fp16's grid of 2^-24 in 2^10 p,
            times a value below 512 (pages with larger scales take the fp32 form): 2^-35 of that; in 2^10 p d, times a number up to 8: 2^-32
      sums  of L live keys and their terms over wavefronts and shares: 2 L + 8 roundings of 2^-23
    An error of a weight counts twice: above and below the line."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    rows, H, dh = q.shape
    T, G, NB = k.shape[0], H // k.shape[1], dh // 32
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    used = q if q_of is None else q_of(q)
    for r in range(rows):
        t = T - rows + r + 1
        for h in range(H):
            kk, vv = k[:t, h // G], v[:t, h // G]
            s = kk @ used[r, h] / np.sqrt(dh)
            live = s > s.max() - 100
            p = np.exp(s - s.max())
            if p_of is None:
                out[r, h] = p[live] @ vv[live] / p[live].sum()
            else:  # a block's scale is its largest value's size / 8, within a rounding: of values that are whole multiples of it
                d = np.repeat(np.abs(vv[live]).reshape(-1, NB, 32).max(-1) / 8, 32, 1)
                out[r, h] = (p_of(p[live][:, None], d) * (vv[live] / np.where(d > 0, d, 1))).sum(0) / p[live].sum()
            size = (np.abs(kk[live]) @ np.abs(q[r, h])).max() / np.sqrt(dh)
            q_err = np.abs(kk[live]).sum(1).max() * np.abs(q[r, h]).max() * 2.0 ** -23 / np.sqrt(dh)
            one = q_err + size * (6 * NB + 2) * 2.0 ** -23 + 2.0 ** -20 + 2.0 ** -22 + 2.0 ** -21
            L = live.sum()
            tol[r, h] = p[live] @ np.abs(vv[live]) / p[live].sum() * (2 * one + (2 * L + 8) * 2.0 ** -23 + 2.0 ** -24) + L * (2.0 ** -32 + 2.0 ** -35 * np.minimum(np.abs(vv[live]).max(0), 512))
    return out, tol


def check(got, q, k, v):
    want, tol = channels(q, k, v)
    assert np.isfinite(got).all()
    worst = np.abs(got - want) / tol
    print("share of the tolerance:", float(worst.max()), flush=True)
    assert (worst <= 1).all(), float(worst.max())
    return want, tol


def sequence(rng, T, rows, kv, dh, live, sizes):
    """A sequence with sparse keys and values of `sizes` (T, kv, dh); (cache, tables, starts, keys, values as held)."""
    cache, tables, starts, _ = batch(rng, [T], [rows], kv, dh)
    slots = np.array([tables[0, t // PAGE] * PAGE + t % PAGE for t in range(T)], np.int32)
    v = (rng.normal(0, 1, (T, kv, dh)) * sizes).astype(np.float32)
    cache.append(sparse_keys(rng, T, kv, dh, live), v, slots)
    k, v = cache.rows(slots)
    return cache, tables, starts, k, v


LIVE = [3, 40, 70, 100, 130, 200, 260, 290]


def half(x):
    return np.float16(x).astype(np.float64)


POORER = dict(
    one_term_of_p=dict(p_of=lambda p, d: half(p * 2.0 ** 14) * d / 2.0 ** 14),
    one_term_of_p_d=dict(p_of=lambda p, d: half(p * d * 2.0 ** 14) / 2.0 ** 14),
    no_second_term_times_d=dict(p_of=lambda p, d: (half(half(p * 2.0 ** 14) * d) + half(half(p * 2.0 ** 14) * d - half(half(p * 2.0 ** 14) * d))) / 2.0 ** 14),
    one_term_of_q=dict(q_of=lambda q: half(q * 256) / 256),
    bfloat16_of_q=dict(q_of=lambda q: (np.float32(q).view(np.uint32) + 0x8000 & 0xFFFF0000).view(np.float32).astype(np.float64)))


@pytest.mark.parametrize("H,kv,dh", [(4, 2, 64), (16, 1, 128), (3, 3, 32), (12, 12, 64), (32, 4, 128), (17, 1, 64)])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("T,live", [(340, LIVE), (64, [0, 1, 20, 35]), (3000, list(range(7, 2960, 301)))])
def test_every_term_counts(H, kv, dh, rows, T, live):
    """Within the bound, which a kernel that lost the second term of a product would not be: that is asked of the definition
    with the term left out."""
    rng = np.random.default_rng(H * rows + T)
    cache, tables, starts, k, v = sequence(rng, T, rows, kv, dh, live, np.ones((T, kv, dh)))
    q = gated_queries(rng, rows, H, dh)
    want, tol = check(cache.attend(q, tables, [T], starts), q, k, v)
    for name, poorer in POORER.items():
        lost = np.abs(channels(q, k, v, **poorer)[0] - want) / tol
        print(name, float(lost.max()), flush=True)
        assert lost.max() > 4, name


@pytest.mark.parametrize("H,kv,dh", [(4, 2, 64), (16, 1, 128), (3, 3, 64), (32, 4, 128)])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("large,small", [(100, 0.01), (1000, 0.01), (1e4, 0.05), (1.8e4, 1.0), (4e5, 0.05), (30, 3e-3)])
def test_a_block_of_large_values_beside_small_ones(H, kv, dh, rows, large, small):
    """Channels 32 .. 63 large, the others small: in all pages, or in one of them."""
    rng = np.random.default_rng(int(large) + dh + rows)
    T = 340
    for pages in (range(6), [0], [3]):
        sizes = np.full((T, kv, dh), small)
        for page in pages:
            sizes[PAGE * page:PAGE * (page + 1), :, 32:64] = large
        cache, tables, starts, k, v = sequence(rng, T, rows, kv, dh, LIVE, sizes)
        q = gated_queries(rng, rows, H, dh)
        check(cache.attend(q, tables, [T], starts), q, k, v)


@pytest.mark.parametrize("H,kv,dh", [(6, 2, 32), (4, 2, 64), (16, 1, 128), (3, 3, 128)])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("size", [20, 4.7e3, 2.4e4, 3.9e5])
def test_a_large_row_without_weight(H, kv, dh, rows, size):
    """One row of large values that no query has a weight for, in the first page, in a later one, in the last: the others' results
    do not depend on it."""
    rng = np.random.default_rng(int(size) + dh + rows)
    T = 340
    for row in (5, 150, 310):
        sizes = np.full((T, kv, dh), 0.05)
        sizes[row] = size
        cache, tables, starts, k, v = sequence(rng, T, rows, kv, dh, LIVE, sizes)
        q = gated_queries(rng, rows, H, dh)
        check(cache.attend(q, tables, [T], starts), q, k, v)


@pytest.mark.parametrize("H,kv,dh", [(6, 2, 32), (16, 1, 128), (4, 4, 64)])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("size,nats", [(4e5, 18), (4e5, 20.5), (300, 15), (600, 20), (30, 12), (17, 0.5), (200, 3)])
def test_a_large_row_of_little_weight(H, kv, dh, rows, size, nats):
    """Its score lies `nats` below that of a key of zeros."""
    rng = np.random.default_rng(int(size + nats) + dh + rows)
    T = 340
    for row in (5, 150, 310):
        sizes = np.full((T, kv, dh), 0.05)
        sizes[row] = size
        cache, tables, starts, k, v = sequence(rng, T, rows, kv, dh, LIVE, sizes)
        slot = [tables[0, row // PAGE] * PAGE + row % PAGE]
        k[row] = 0.0
        k[row, :, 0] = -nats * np.sqrt(dh) / 2.0
        cache.append(k[row:row + 1], v[row:row + 1], slot)
        k[row:row + 1], v[row:row + 1] = cache.rows(slot)
        q = gated_queries(rng, rows, H, dh)
        check(cache.attend(q, tables, [T], starts), q, k, v)


@pytest.mark.parametrize("H,kv,dh", [(2, 2, 32), (8, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("factors", [(1e-5, 1, 1e3), (1e3, 1e-3, 1), (1e-4, 1e4, 1e-4), (1, 1e5, 1e-2)])
def test_sizes_page_by_page(H, kv, dh, rows, factors):
    rng = np.random.default_rng(dh * rows)
    T = 40 * PAGE + 30
    live = list(range(7, T, 211))
    sizes = np.array(factors)[np.arange(T) // PAGE * len(factors) // (T // PAGE + 1)][:, None, None] * np.ones((1, kv, dh))
    cache, tables, starts, k, v = sequence(rng, T, rows, kv, dh, live, sizes)
    q = gated_queries(rng, rows, H, dh)
    check(cache.attend(q, tables, [T], starts), q, k, v)


@pytest.mark.parametrize("H,kv,dh", [(2, 2, 64), (16, 2, 32), (4, 1, 128)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_a_query_that_is_not_finite_and_sees_no_key(H, kv, dh, what):
    """Its row is zero like any other without keys, next to rows that see some; one that sees a key is NaN."""
    rng = np.random.default_rng(H + dh)
    lens, rows = [3, 100, 70], [8, 1, 1]
    cache, tables, starts, held = batch(rng, lens, rows, kv, dh)
    q = rng.normal(0, 1, (10, H, dh)).astype(np.float32)
    clean = cache.attend(q, tables, lens, starts)
    q[1, :, 5], q[4, 0, 0], q[8, :, dh - 1] = what, what, what
    tables[1] = -1, cache.n_pages  # (all of the second sequence's pages are outside the pool)
    got = cache.attend(q, tables, lens, starts)
    assert not got[:5].any() and not got[8].any()
    assert np.array_equal(got[5:8], clean[5:8]) and np.array_equal(got[9], clean[9])
    q[6, 0, 1] = what
    got = cache.attend(q, tables, lens, starts)
    assert np.isnan(got[6, 0]).all() and np.array_equal(got[6, 1:], clean[6, 1:]) and not got[:5].any()
    assert np.array_equal(got[[5, 7, 9]], clean[[5, 7, 9]])
