"""Beam search: the selection over beams and vocabulary, and what the beams hold following them (the reference decodes
greedily, apps/gpt2/gpt2.lisp:97-113): against the definitions of include/caten_hip.h in NumPy, in 64 bits."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
PAGE = 64


def select_by_hand(logits, scores, finished, eos):
    """All candidates in order: the higher score, then the lower beam, then the higher logit, then the lower token."""
    n, K, V = logits.shape
    tokens, parents, best = np.zeros((n, K), int), np.zeros((n, K), int), np.zeros((n, K))
    for i in range(n):
        x = logits[i].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        s = np.where(np.isnan(scores[i]), -np.inf, scores[i].astype(np.float64))
        y = np.full((K, V), -np.inf)
        for k in range(K):
            top = x[k].max()
            if s[k] == -np.inf:
                x[k] = 0  # (all alike)
            elif finished is not None and finished[i, k]:
                y[k, eos] = s[k]
                x[k] = 0
            elif top > -np.inf:
                with np.errstate(invalid="ignore"):
                    rel = np.where(x[k] == top, 0.0, x[k] - top)
                y[k] = s[k] + rel - np.log(np.exp(rel).sum())
        flat = np.lexsort((np.tile(np.arange(V), K), -x.ravel(), np.repeat(np.arange(K), V), -y.ravel()))[:K]
        parents[i], tokens[i], best[i] = flat // V, flat % V, y.ravel()[flat]
    return tokens, parents, best


def check(logits, scores, finished=None, eos=-1):
    from caten_amd import ops
    got = ops.beam_select(logits, scores, finished, eos)
    tokens, parents, best = select_by_hand(logits, scores, finished, eos)
    assert np.array_equal(got["tokens"], tokens) and np.array_equal(got["parents"], parents)
    fine = np.isfinite(best)
    assert np.array_equal(got["scores"][~fine], best[~fine].astype(np.float32))
    # a rounding of the score, and a sum of exponentials each off by a few roundings: 2^-21 of it, and of its logarithm
    assert (np.abs(got["scores"][fine] - best[fine]) <= np.abs(best[fine]) * 2.0 ** -24 + 2.0 ** -21).all()
    was = np.zeros(scores.shape, int) if finished is None else np.asarray(finished)
    assert np.array_equal(got["finished"], (np.take_along_axis(was, parents, 1) != 0) | (tokens == eos))
    return got


@pytest.mark.parametrize("n,K,V", [(1, 1, 1), (1, 1, 50257), (1, 4, 50257), (2, 3, 7), (3, 5, 5), (5, 8, 1000), (2, 32, 4099), (40, 4, 3001), (1, 16, 131072), (7, 2, 64), (3, 32, 32), (2, 6, 65537)])
def test_select(n, K, V):
    print(f"case: select {n} x {K} beams of {V}", flush=True)
    rng = np.random.default_rng(n * K + V)
    logits = rng.normal(0, 3, (n, K, V)).astype(np.float32)
    scores = -np.sort(rng.uniform(0, 12, (n, K)).astype(np.float32), 1)
    check(logits, scores)
    done = (rng.uniform(0, 1, (n, K)) < 0.3).astype(np.int32)
    check(logits, scores, done, eos=V // 2)
    logits[rng.uniform(0, 1, logits.shape) < 0.3] = -np.inf
    check(logits, scores, done, eos=0)


@pytest.mark.parametrize("n,K,V", [(1, 32, 131072), (1, 14, 250001), (2, 2, 300007), (1, 3, 600000)])
def test_long_rows(n, K, V):
    """More lists than the merge keeps by it, rows of more than 32 slices' registers."""
    print(f"case: long rows, {n} x {K} beams of {V}", flush=True)
    rng = np.random.default_rng(V)
    logits = rng.standard_normal((n, K, V), np.float32)
    logits[:, :, -3:] += 4
    scores = -np.sort(rng.uniform(0, 2, (n, K)).astype(np.float32), 1)
    check(logits, scores)
    check(np.round(logits), scores, (rng.uniform(0, 1, (n, K)) < 0.4).astype(np.int32), eos=V - 1)


def test_more_equal_candidates_than_the_merge_holds():
    """32 beams, each with 32 tokens of one logit, all scores alike: 1024 equal candidates."""
    logits = np.zeros((2, 32, 4000), np.float32)
    logits[0, :, 100:140] = 9.0
    logits[1, 5:, 7:3000:90] = 9.0
    check(logits, np.zeros((2, 32), np.float32))


def test_first_step():
    """Beams that all hold the prompt: only the first counts."""
    rng = np.random.default_rng(1)
    logits = np.repeat(rng.normal(0, 3, (4, 1, 5000)).astype(np.float32), 5, 1)
    scores = np.full((4, 5), -np.inf, np.float32)
    scores[:, 0] = 0
    got = check(logits, scores)
    assert (got["parents"] == 0).all()


def test_ties():
    rng = np.random.default_rng(2)
    V = 30011
    logits = rng.normal(0, 1, (3, 4, V)).astype(np.float32)
    logits[0, :, rng.permutation(V)[:50]] = 8.0                    # equal logits in a beam: the lower token
    logits[1] = logits[1, :1]                                       # equal beams: the lower beam
    logits[2] = 0.25                                                # everything equal
    scores = np.zeros((3, 4), np.float32)
    check(logits, scores)
    check(np.round(logits * 2) / 2, scores)                         # few levels: more equal ones than any list holds
    one = np.full((1, 8, 70000), -5.0, np.float32)
    one[0, :, 69990:] = 1.0
    check(one, np.zeros((1, 8), np.float32))


def test_what_is_not_finite():
    rng = np.random.default_rng(3)
    inf, nan = np.inf, np.nan
    logits = rng.normal(0, 2, (8, 3, 2000)).astype(np.float32)
    scores = np.tile(np.array([-1, -2, -3], np.float32), (8, 1))
    done = np.zeros((8, 3), np.int32)
    logits[0, :, 1:] = -inf                                        # one candidate a beam
    logits[1, 0] = -inf                                            # a beam without candidates
    logits[2] = -inf                                               # none at all
    logits[3, 1, 5:800] = nan
    logits[3, 2] = nan
    logits[4, 0, 7], logits[4, 0, 1900] = inf, inf                 # all weight on two
    scores[5] = -inf, nan, -4
    scores[6] = nan
    done[7] = 1, 1, 0
    logits[7, 2, 1:] = -inf
    check(logits, scores)
    check(logits, scores, done, eos=11)
    check(np.float32(3e38) * np.sign(logits), scores, done, eos=11)  # differences past fp32's range
    only = np.full((1, 2, 100), np.finfo(np.float32).min, np.float32)  # a mask of the lowest value
    only[0, 0, 40] = 0
    check(only, np.zeros((1, 2), np.float32))


def test_strided_logits_and_a_call_again():
    from caten_amd import _lib, ops
    rng = np.random.default_rng(4)
    lib, n, K, V, stride = _lib.init(), 3, 4, 20001, 20011
    wide = rng.normal(0, 2, (n * K, stride)).astype(np.float32)
    wide[:, V:] = 100.0                                             # behind a row's end
    scores = -np.sort(rng.uniform(0, 9, (n, K)).astype(np.float32), 1)
    ws = ops.DeviceArray((int(lib.cthip_beam_select_workspace(n, K)),), np.uint8)
    d, s = ops.DeviceArray.from_numpy(np.concatenate([np.zeros(1, np.float32), wide.ravel()])), ops.DeviceArray.from_numpy(scores)
    tokens, parents = (ops.DeviceArray((n, K), np.int32) for _ in range(2))
    best = ops.DeviceArray((n, K), np.float32)
    want = select_by_hand(wide[:, :V].reshape(n, K, V), scores, None, -1)
    for _ in range(3):
        _lib.check(lib.cthip_beam_select(tokens.ptr, parents.ptr, best.ptr, None, d.ptr + 4, stride, s.ptr, None, n, K, V, -1, ws.ptr))
        assert np.array_equal(tokens.numpy(), want[0]) and np.array_equal(parents.numpy(), want[1])


def test_captured_selection():
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(5)
    stream = C.c_void_p(lib.cthip_stream())
    n, K, V = 2, 5, 50257
    ws = ops.DeviceArray((int(lib.cthip_beam_select_workspace(n, K)),), np.uint8)
    logits, scores = ops.DeviceArray((n, K, V), np.float32), ops.DeviceArray((n, K), np.float32)
    tokens, parents, done = (ops.DeviceArray((n, K), np.int32) for _ in range(3))
    best = ops.DeviceArray((n, K), np.float32)
    call = lambda: _lib.check(lib.cthip_beam_select(tokens.ptr, parents.ptr, best.ptr, done.ptr, logits.ptr, V, scores.ptr, None, n, K, V, 3, ws.ptr))
    graph, run = C.c_void_p(), C.c_void_p()
    assert lib.hipStreamBeginCapture(stream, 1) == 0
    call()
    assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(4):
        x, s = rng.normal(0, 2, (n, K, V)).astype(np.float32), -np.sort(rng.uniform(0, 9, (n, K)).astype(np.float32), 1)
        _lib.check(lib.cthip_h2d(logits.ptr, x.ctypes.data, x.nbytes))
        _lib.check(lib.cthip_h2d(scores.ptr, s.ctypes.data, s.nbytes))
        assert lib.hipGraphLaunch(run, stream) == 0
        got = tokens.numpy(), parents.numpy()
        want = select_by_hand(x, s, None, 3)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        call()
        assert np.array_equal(tokens.numpy(), got[0])
    lib.hipGraphExecDestroy(run)
    lib.hipGraphDestroy(graph)


# ------------------------------------------------------------------------------------------------------------ reordering


def reorder_by_hand(tables, lens, parents, k_pool, v_pool):
    """(tables, pools) after the reordering, request by request, from the pools as they were."""
    n, K = parents.shape
    out, pools = tables.copy(), [k_pool.copy(), v_pool.copy()]
    for i in range(n):
        par = [p if 0 <= p < K else j for j, p in enumerate(parents[i])]
        dead = [j for j in range(K) if j not in par]
        last, part = lens[i] // PAGE, lens[i] % PAGE
        seen = set()
        for j, p in enumerate(par):
            row, old = i * K + j, tables[i * K + p]
            out[row, :last] = old[:last]
            if part and last < tables.shape[1]:
                if p not in seen:
                    out[row, last] = old[last]
                else:
                    page = tables[i * K + dead.pop(0), last]
                    out[row, last] = page
                    if 0 <= old[last] < k_pool.shape[1] and 0 <= page < k_pool.shape[1]:
                        for new, was in zip(pools, (k_pool, v_pool)):
                            new[:, page] = was[:, old[last]]
            seen.add(p)
    return out, pools


@pytest.mark.parametrize("n,K,layers,kv,dh", [(1, 1, 1, 1, 32), (1, 4, 12, 12, 64), (6, 5, 3, 4, 64), (4, 32, 2, 1, 32), (3, 8, 1, 8, 128)])
def test_reorder(n, K, layers, kv, dh):
    print(f"case: reorder {n} x {K} beams, {layers} layers, {kv} heads of {dh}", flush=True)
    from caten_amd import _lib, ops
    rng = np.random.default_rng(n * K + dh)
    table = 5
    lens = rng.integers(0, table * PAGE + 1, n)
    lens[0] = 100
    if n > 2:
        lens[1], lens[2] = 128, table * PAGE
    pages = list(rng.permutation(n * (table + K) + 2))
    cache = ops.PagedCacheQ4(len(pages), kv, dh, layers)
    tables = rng.integers(-5, len(pages), (n * K, table)).astype(np.int32)  # (entries behind the last page: any)
    for i, t in enumerate(lens):
        tables[i * K:(i + 1) * K, :t // PAGE] = [pages.pop() for _ in range(t // PAGE)]
        if t % PAGE:
            tables[i * K:(i + 1) * K, t // PAGE] = [pages.pop() for _ in range(K)]
    for round_ in range(4):
        parents = rng.integers(0, K, (n, K)).astype(np.int32)
        if round_ == 1:
            parents[:] = K - 1
        if round_ == 2:
            parents[:, 0], parents[:, -1] = -1, K
        fill = [rng.integers(0, 256, p.shape).astype(np.uint8) for p in (cache.k, cache.v)]
        for pool, f in zip((cache.k, cache.v), fill):
            _lib.check(_lib.load().cthip_h2d(pool.ptr, f.ctypes.data, f.nbytes))
        want, pools = reorder_by_hand(tables, lens, parents, *fill)
        history, tokens, step = rng.integers(0, 1000, (n * K, 9)).astype(np.int32), rng.integers(0, 1000, (n, K)).astype(np.int32), [0, 8, 4, 9][round_]
        for _ in range(2):  # a call repeated writes the same bytes
            got, hist = cache.reorder(tables, lens, parents, history, tokens, step)
            assert np.array_equal(got, want)
            assert np.array_equal(cache.k.numpy(), pools[0]) and np.array_equal(cache.v.numpy(), pools[1])
        source = np.where((parents < 0) | (parents >= K), np.arange(K), parents) + np.arange(n)[:, None] * K
        expect = history[source.ravel()]
        if step < 9:
            expect[:, step] = tokens.ravel()
        assert np.array_equal(hist, expect)
        assert np.array_equal(cache.reorder(tables, lens, parents), want)
        # the last pages are still one to a beam
        for i, t in enumerate(lens):
            if t % PAGE:
                assert len(set(want[i * K:(i + 1) * K, t // PAGE])) == K


def test_captured_reordering():
    """A replay with other parents and lengths is that call; tables go to and fro."""
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(7)
    stream = C.c_void_p(lib.cthip_stream())
    n, K, layers, kv, dh, table = 2, 4, 3, 2, 32, 3
    n_pages = n * K * table
    cache = ops.PagedCacheQ4(n_pages, kv, dh, layers)
    tables = rng.permutation(n_pages).reshape(n * K, table).astype(np.int32)
    for i in range(n):
        tables[i * K:(i + 1) * K, 0] = tables[i * K, 0]
    dt, dl, dp = ops.DeviceArray.from_numpy(tables), ops.DeviceArray((n,), np.int32), ops.DeviceArray((n, K), np.int32)
    out, hist, dh_out = ops.DeviceArray(tables.shape, np.int32), ops.DeviceArray.from_numpy(rng.integers(0, 99, (n * K, 5)).astype(np.int32)), ops.DeviceArray((n * K, 5), np.int32)
    tokens, step = ops.DeviceArray.from_numpy(np.arange(n * K, dtype=np.int32)), ops.DeviceArray.from_numpy(np.array([2], np.int32))
    call = lambda: _lib.check(lib.cthip_beam_reorder_paged_q4(out.ptr, dh_out.ptr, cache.k.ptr, cache.v.ptr, layers, n_pages, dt.ptr, table, dl.ptr, dp.ptr, n, K, kv, dh, hist.ptr, 5,
                                                              tokens.ptr, step.ptr))
    graph, run = C.c_void_p(), C.c_void_p()
    assert lib.hipStreamBeginCapture(stream, 1) == 0
    call()
    assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(4):
        parents, lens = rng.integers(0, K, (n, K)).astype(np.int32), rng.integers(65, 128, n).astype(np.int32)
        fill = [rng.integers(0, 256, p.shape).astype(np.uint8) for p in (cache.k, cache.v)]
        for to, x in zip((cache.k, cache.v, dp, dl), fill + [parents, lens]):
            _lib.check(lib.cthip_h2d(to.ptr, x.ctypes.data, x.nbytes))
        want, pools = reorder_by_hand(tables, lens, parents, *fill)
        assert lib.hipGraphLaunch(run, stream) == 0
        assert np.array_equal(out.numpy(), want) and np.array_equal(cache.k.numpy(), pools[0]) and np.array_equal(cache.v.numpy(), pools[1])
        got = dh_out.numpy()
        call()
        assert np.array_equal(out.numpy(), want) and np.array_equal(dh_out.numpy(), got) and np.array_equal(got[:, 2], np.arange(n * K))
    lib.hipGraphExecDestroy(run)
    lib.hipGraphDestroy(graph)


def test_a_search_as_a_whole():
    """plan, append, attention, select, reorder, step after step on the device; against a search that keeps every hypothesis's
    own dense cache: the same tokens and scores, across a border of two pages."""
    from caten_amd import _lib, ops
    from tests.test_gpu_paged_q4 import attention, quantised
    lib, rng = _lib.init(), np.random.default_rng(6)
    n, K, H, kv, dh, V, steps, table, n_pages, cols = 2, 4, 4, 2, 32, 300, 40, 4, 60, 64
    prompts = [50, 30]
    emb = rng.normal(0, 1, (V, (H + 2 * kv) * dh)).astype(np.float32)  # a token's q, k and v
    head = rng.normal(0, 0.4, (V, H * dh)).astype(np.float32)
    prompt = [rng.integers(0, V, p) for p in prompts]
    # by hand
    beams = [[(0.0 if k == 0 else -np.inf, list(p)) for k in range(K)] for p in prompt]

    def logits_of(tokens):
        rows = emb[tokens]
        k, v = (quantised(rows[:, (H + a) * dh:(H + a + kv) * dh].reshape(-1, kv, dh)) for a in (0, kv))
        out, _, _ = attention(rows[-1:, :H * dh].reshape(1, H, dh), k, v)
        return head.astype(np.float64) @ out.ravel()

    # on the device
    cache = ops.PagedCacheQ4(n_pages, kv, dh)
    d = {k: ops.DeviceArray.from_numpy(np.asarray(v, np.int32)) for k, v in dict(lens=[0] * n * K, free=rng.permutation(n_pages), n=[n_pages], one=[1] * n * K).items()}
    tables = [ops.DeviceArray.from_numpy(np.full((n * K, table), -1, np.int32)) for _ in range(2)]
    hist = [ops.DeviceArray((n * K, cols), np.int32) for _ in range(2)]
    o = {k: ops.DeviceArray((m,), np.int32) for k, m in dict(slots=400, starts=n * K + 1, refused=1, tokens=n * K, parents=n * K, done=n * K, step=1).items()}
    scores = [ops.DeviceArray.from_numpy(np.tile(np.array([0] + [-np.inf] * (K - 1), np.float32), n)), ops.DeviceArray((n * K,), np.float32)]
    ws = ops.DeviceArray((int(lib.cthip_beam_select_workspace(n, K)),), np.uint8)
    out, wide = ops.DeviceArray((400, H * dh), np.float32), (H + 2 * kv) * dh
    feed = np.concatenate([p for p in prompt for _ in range(K)])  # every beam its own copy of the prompt: pages of its own
    new = ops.DeviceArray.from_numpy(np.repeat(prompts, K).astype(np.int32))
    for step in range(steps):
        rows = feed.size
        src = ops.DeviceArray.from_numpy(emb[feed])
        _lib.check(lib.cthip_kv_plan_paged(o["slots"].ptr, None, o["starts"].ptr, tables[0].ptr, table, d["lens"].ptr, d["n"].ptr, o["refused"].ptr, d["lens"].ptr,
                                           (new if step == 0 else d["one"]).ptr, n * K, d["free"].ptr, d["n"].ptr, rows))
        _lib.check(lib.cthip_kv_append_paged_q4(cache.k.ptr, cache.v.ptr, src.ptr + 4 * H * dh, src.ptr + 4 * (H + kv) * dh, wide, wide, o["slots"].ptr, rows, n_pages, kv, dh))
        _lib.check(lib.cthip_sdpa_paged_q4(out.ptr, src.ptr, wide, cache.k.ptr, cache.v.ptr, n_pages, tables[0].ptr, table, d["lens"].ptr, o["starts"].ptr, n * K, rows, H, kv, dh,
                                           cache.workspace.ptr))
        assert o["refused"].numpy()[0] == 0
        last = out.numpy()[o["starts"].numpy()[1:] - 1]
        logits = ops.DeviceArray.from_numpy((last.astype(np.float64) @ head.T.astype(np.float64)).astype(np.float32))
        _lib.check(lib.cthip_beam_select(o["tokens"].ptr, o["parents"].ptr, scores[1].ptr, o["done"].ptr, logits.ptr, V, scores[0].ptr, None, n, K, V, -1, ws.ptr))
        at, lens = ops.DeviceArray.from_numpy(np.array([step], np.int32)), ops.DeviceArray.from_numpy(d["lens"].numpy()[::K].copy())
        _lib.check(lib.cthip_beam_reorder_paged_q4(tables[1].ptr, hist[1].ptr, cache.k.ptr, cache.v.ptr, 1, n_pages, tables[0].ptr, table, lens.ptr, o["parents"].ptr, n, K, kv, dh, hist[0].ptr,
                                                   cols, o["tokens"].ptr, at.ptr))
        tables, hist, scores = tables[::-1], hist[::-1], scores[::-1]
        feed = o["tokens"].numpy()
        for i in range(n):
            table_of = []
            for k, (s, t) in enumerate(beams[i]):
                x = logits_of(t) if s > -np.inf else np.zeros(V)
                x = x - x.max()
                lp = s + x - np.log(np.exp(x).sum())
                table_of += [(-lp[v], k, v) for v in np.argsort(-lp)[:K]]
            table_of.sort()
            beams[i] = [(-y, beams[i][k][1] + [int(v)]) for y, k, v in table_of[:K]]
            got = hist[0].numpy()[i * K:(i + 1) * K, :step + 1]
            assert np.array_equal(got, [t[prompts[i]:] for _, t in beams[i]]), (step, i)
            assert np.allclose(scores[0].numpy()[i * K:(i + 1) * K], [s for s, _ in beams[i]], rtol=1e-4, atol=1e-3)


def test_refusals():
    from caten_amd import HipError, _lib, ops
    lib = _lib.init()
    a, b = ops.DeviceArray((4096,), np.int32), ops.DeviceArray((4096,), np.int32)
    p, r = a.ptr, b.ptr

    def refused(code, fn, *args):
        with pytest.raises(HipError) as e:
            _lib.check(fn(*args))
        assert e.value.code == code, e.value

    bad, no = _lib.E_BAD_ARG, _lib.E_UNSUPPORTED
    select = lambda **k: [dict(dict(t=p, par=p, s_out=p, f_out=p, x=p, stride=10, s=r, f=r, n=1, K=2, V=10, eos=1, ws=p), **k)[x] for x in
                          ("t", "par", "s_out", "f_out", "x", "stride", "s", "f", "n", "K", "V", "eos", "ws")]
    for change in (dict(t=None), dict(par=None), dict(s_out=None), dict(x=None), dict(s=None), dict(ws=None), dict(ws=p + 4), dict(stride=9), dict(n=-1), dict(K=0), dict(V=1), dict(V=0), dict(eos=10),
                   dict(eos=-2), dict(eos=-1), dict(s=p), dict(f=p)):
        refused(bad, lib.cthip_beam_select, *select(**change))
    for change in (dict(K=33, V=100, stride=100), dict(n=(1 << 17) + 1)):
        refused(no, lib.cthip_beam_select, *select(**change))
    reorder = lambda **k: [dict(dict(to=p, ho=p, k=p, v=p, layers=1, pages=1, t=r, stride=1, lens=p, par=p, n=1, K=2, kv=1, dh=32, h=r, cols=4, tok=p, step=p), **k)[x] for x in
                           ("to", "ho", "k", "v", "layers", "pages", "t", "stride", "lens", "par", "n", "K", "kv", "dh", "h", "cols", "tok", "step")]
    for change in (dict(to=None), dict(t=None), dict(t=p), dict(h=p), dict(h=None), dict(tok=None), dict(step=None), dict(k=None), dict(v=None), dict(k=p + 4), dict(lens=None), dict(par=None), dict(n=-1),
                   dict(K=0), dict(layers=-1), dict(pages=-1), dict(stride=0), dict(cols=-1)):
        refused(bad, lib.cthip_beam_reorder_paged_q4, *reorder(**change))
    for change in (dict(K=33), dict(n=40000), dict(dh=16), dict(kv=0)):
        refused(no, lib.cthip_beam_reorder_paged_q4, *reorder(**change))
    _lib.check(lib.cthip_beam_select(*select(n=0)))
    _lib.check(lib.cthip_beam_reorder_paged_q4(*reorder(n=0)))
    _lib.check(lib.cthip_sync())
    with pytest.raises(ValueError):
        ops.beam_select(np.zeros((2, 3, 4)), np.zeros((2, 2)))
