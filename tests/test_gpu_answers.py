"""Several answers to one prompt, drafted and verified, as a server would run them: prompt, fork, then steps of plan, rotary rows, append, attention over the
shared pages, probabilities and verification, with pages freed and the pool packed between steps.  Each step against a simulation in 64 bits; a captured step
against the eager one."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_draft import softmax, verified
from tests.test_gpu_paged_q4 import PAGE, quantised
from tests.test_gpu_rope_rows import turned
from tests.test_gpu_shared_prefix import close, seen

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[1, 2], ids=["as it pays", "apart"])
def way(request):
    """Shared pages in a launch of their own where that pays (nowhere here), and always."""
    from caten_amd import _lib
    _lib.check(_lib.init().cthip_set_option(b"shared_prefix", request.param))
    yield
    _lib.check(_lib.load().cthip_set_option(b"shared_prefix", 1))


def test_answers_to_a_prompt(way):
    from caten_amd import ops
    rng = np.random.default_rng(41)
    H, kv, dh, vocab, n, layers, table, n_pages = 8, 2, 64, 301, 6, 2, 12, 60
    prompt, at = 300, 290  # the answers branch off ten rows before the prompt's end: a page is copied
    w = (H + 2 * kv) * dh
    embed, head = (rng.normal(0, 1, (layers, vocab, w))).astype(np.float32), rng.normal(0, 0.2, (H * dh, vocab)).astype(np.float32)
    f = ops.rope_frequencies(dh, 10000.0, 4.0, 256)
    cache = ops.PagedCacheQ4(n_pages, kv, dh, layers)
    tables, lens, free = np.full((n, table), -1, np.int32), np.zeros(n, np.int32), rng.permutation(n_pages).astype(np.int32)
    tokens = [list(rng.integers(0, vocab, prompt))] + [[] for _ in range(n - 1)]
    held = [[(np.zeros((0, kv, dh)), np.zeros((0, kv, dh))) for _ in range(layers)] for _ in range(n)]

    def step(new, feed, groups, shared):
        """Rows of new tokens through both layers; what the last one gives."""
        nonlocal tables, lens, free
        plan = ops.kv_plan(lens, new, tables, free, int(sum(new)))
        assert plan["refused"] == 0
        tables, free = plan["tables"], free[:plan["n_free"]]
        starts, whole = plan["starts"], np.zeros(n, int)
        for g, s in enumerate(shared):
            if groups[g + 1] - groups[g] > 1:
                whole[groups[g]:groups[g + 1]] = s // PAGE * PAGE
        for layer in range(layers):
            qkv = embed[layer][feed].reshape(len(feed), -1, dh)
            q, k = ops.rope_rows(qkv[:, :H], qkv[:, H:H + kv], plan["positions"], f, "halves")
            for got, x in ((q, qkv[:, :H]), (k, qkv[:, H:H + kv])):
                want, size = turned(x, plan["positions"], f, "halves", 1.0)
                assert (np.abs(got - want) <= 2.0 ** -21 * size).all()
            cache.append(k, qkv[:, H + kv:], plan["slots"], layer)
            out = cache.attend_shared(q, tables, plan["lens"], starts, groups, shared, layer)
            for i in range(n):
                r = slice(starts[i], starts[i + 1])
                held[i][layer] = tuple(np.concatenate([a, quantised(b[r])]) for a, b in zip(held[i][layer], (k, qkv[:, H + kv:])))
                if new[i]:
                    close(out[r], *seen(q[r], *held[i][layer], whole[i]))
        lens = plan["lens"]
        return out, starts, plan["positions"]

    step([prompt] + [0] * (n - 1), tokens[0], [0], [])
    got = cache.fork(tables, lens, [0] * (n - 1), range(1, n), [at] * (n - 1), free)
    assert not got["refused"].any()
    tables, lens, free = got["tables"], got["lens"], free[:got["n_free"]]
    for i in range(1, n):
        tokens[i] = tokens[0][:at]
        held[i] = [(k[:at], v[:at]) for k, v in held[0]]
    last = [t.pop() for t in tokens]  # the token that goes in next; its row is not in the cache
    for i in range(n):
        lens[i] -= 1
        held[i] = [(k[:-1], v[:-1]) for k, v in held[i]]
    assert (np.array(lens) > at // PAGE * PAGE).all()
    for turn in range(5):
        drafts = [int(rng.integers(0, 5)) if i != turn else 0 for i in range(n)]
        starts = np.concatenate([[0], np.cumsum([d + 1 for d in drafts])])
        feed = np.zeros(starts[-1], int)
        for i in range(n):
            feed[starts[i]:starts[i + 1]] = [last[i]] + list(rng.integers(0, vocab, drafts[i]))
        out, _, positions = step([d + 1 for d in drafts], feed, [0, n], [at])
        target = ops.softmax(0.1 * (out.reshape(len(feed), -1) @ head))
        draft = softmax(rng.normal(0, 1, target.shape))
        uniforms = rng.random(len(feed)).astype(np.float32)
        got = ops.draft_verify(target, draft, feed, uniforms, starts, lens, positions)
        want = verified(target, draft, feed, uniforms, starts, lens, positions)
        for key in want:
            assert np.array_equal(got[key], want[key]), key
        lens = got["lens"]
        for i in range(n):
            out_tokens = [t for t in got["tokens"][starts[i]:starts[i + 1]] if t >= 0]
            tokens[i] += [last[i]] + out_tokens[:-1]
            last[i] = out_tokens[-1]
            held[i] = [(k[:lens[i]], v[:lens[i]]) for k, v in held[i]]
            assert len(tokens[i]) == lens[i] == len(held[i][0][0])
        if turn == 2:
            got = cache.compact(tables, lens)
            tables, free = got["tables"], got["free_pages"]
            assert tables[tables >= 0].size and free.min() == n_pages - free.size
        else:
            free = ops.kv_free_pages(tables, lens, n_pages)
        for i in range(n):
            for layer in range(layers):
                k, v = cache.rows([tables[i, t // PAGE] * PAGE + t % PAGE for t in range(lens[i])], layer)
                assert np.array_equal(k, held[i][layer][0]) and np.array_equal(v, held[i][layer][1])


def test_a_captured_step(way):
    """Rotary rows, append, shared attention, probabilities and verification of a step, recorded: replays give the next steps.  Two graphs with workspaces of their own,
    eager work between the replays."""
    from caten_amd import _lib, ops
    lib = _lib.init()
    stream = C.c_void_p(lib.cthip_stream())
    H, kv, dh, n, table, n_pages, drafts, prefix = 16, 4, 128, 5, 16, 60, 3, 448
    rows, w, vocab = n * (drafts + 1), (H + 2 * kv) * dh, H * dh
    r = np.random.default_rng(43)
    common = r.permutation(n_pages)[:prefix // PAGE]
    rest = np.setdiff1d(np.arange(n_pages), common)
    tables0 = np.full((n, table), -1)
    tables0[:, :len(common)] = common
    f = ops.rope_frequencies(dh)
    qkv0, draft0, uniforms0 = r.normal(0, 1, (8, rows, w)), softmax(r.normal(0, 1, (rows, vocab))), r.random((8, rows))
    tokens0 = r.integers(0, vocab, (8, rows))

    def fresh():
        cache = ops.PagedCacheQ4(n_pages, kv, dh)
        q = np.random.default_rng(44)
        cache.append(q.normal(0, 1, (prefix, kv, dh)), q.normal(0, 1, (prefix, kv, dh)), [common[t // PAGE] * PAGE + t % PAGE for t in range(prefix)])
        d = {k: ops.DeviceArray.from_numpy(np.asarray(v, np.int32)) for k, v in dict(lens=[prefix] * n, tables=tables0, free=rest, n=[rest.size], new=[drafts + 1] * n, groups=[0, n], shared=[prefix + 5],
                                                                                     tokens=tokens0[0]).items()}
        o = {k: ops.DeviceArray((m,), np.int32) for k, m in dict(slots=rows, positions=rows, starts=n + 1, refused=1, tokens=rows, accepted=n).items()}
        x = {k: ops.DeviceArray(s, np.float32) for k, s in dict(qkv=(rows, w), out=(rows, H * dh), target=(rows, vocab), u=(rows,)).items()}
        x["draft"], x["f"] = ops.DeviceArray.from_numpy(draft0), ops.DeviceArray.from_numpy(f)
        ws = ops.DeviceArray((int(lib.cthip_sdpa_shared_paged_q4_workspace(rows, H, dh)),), np.uint8), ops.DeviceArray((2048 * n,), np.uint8)

        def feed(k):
            for to, a, t in ((x["qkv"], qkv0[k], np.float32), (x["u"], uniforms0[k], np.float32), (d["tokens"], tokens0[k], np.int32)):
                a = np.ascontiguousarray(a, t)
                _lib.check(lib.cthip_h2d(to.ptr, a.ctypes.data, a.nbytes))

        def step():
            k_at, v_at = x["qkv"].ptr + 4 * H * dh, x["qkv"].ptr + 4 * (H + kv) * dh
            _lib.check(lib.cthip_kv_plan_paged(o["slots"].ptr, o["positions"].ptr, o["starts"].ptr, d["tables"].ptr, table, d["lens"].ptr, d["n"].ptr, o["refused"].ptr, d["lens"].ptr, d["new"].ptr, n,
                                               d["free"].ptr, d["n"].ptr, rows))
            _lib.check(lib.cthip_rope_rows(x["qkv"].ptr, w, k_at, w, x["qkv"].ptr, w, k_at, w, o["positions"].ptr, rows, H, kv, dh, dh, 0, x["f"].ptr, 1.0))
            _lib.check(lib.cthip_kv_append_paged_q4(cache.k.ptr, cache.v.ptr, k_at, v_at, w, w, o["slots"].ptr, rows, n_pages, kv, dh))
            _lib.check(lib.cthip_sdpa_shared_paged_q4(x["out"].ptr, x["qkv"].ptr, w, cache.k.ptr, cache.v.ptr, n_pages, d["tables"].ptr, table, d["lens"].ptr, o["starts"].ptr, n, rows,
                                                      d["groups"].ptr, d["shared"].ptr, 1, H, kv, dh, ws[0].ptr))
            _lib.check(lib.cthip_softmax(x["target"].ptr, x["out"].ptr, rows, vocab))
            _lib.check(lib.cthip_draft_verify(o["tokens"].ptr, o["accepted"].ptr, d["lens"].ptr, x["target"].ptr, vocab, x["draft"].ptr, vocab, d["tokens"].ptr, x["u"].ptr, o["starts"].ptr,
                                              o["positions"].ptr, d["lens"].ptr, n, rows, vocab, ws[1].ptr))
            # (rejected rows' pages come back)
            _lib.check(lib.cthip_kv_free_paged(d["free"].ptr, d["n"].ptr, d["tables"].ptr, table, d["lens"].ptr, n, n_pages))
        d["free"] = ops.DeviceArray.from_numpy(np.concatenate([rest, np.full(n_pages - rest.size, -1)]).astype(np.int32))
        return d, o, x, feed, step, cache, ws

    eager, graphed = fresh(), [fresh(), fresh()]
    runs = []
    for g in graphed:
        g[3](0)
        graph, run = C.c_void_p(), C.c_void_p()
        assert lib.hipStreamBeginCapture(stream, 1) == 0
        g[4]()
        assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        runs.append((graph, run))
    moved = 0
    for turn in range(6):
        eager[3](turn)
        eager[4]()
        want = {**{k: eager[1][k].numpy() for k in ("tokens", "accepted", "positions", "slots")}, "out": eager[2]["out"].numpy(), "lens": eager[0]["lens"].numpy(), "tables": eager[0]["tables"].numpy()}
        moved += want["accepted"].sum()
        for g, (_, run) in zip(graphed, runs):
            g[3](turn)
            assert lib.hipGraphLaunch(run, stream) == 0
        for g in graphed:
            for k, v in want.items():
                got = (g[1] if k in ("tokens", "accepted", "positions", "slots") else g[2] if k == "out" else g[0])[k].numpy()
                assert np.array_equal(got, v), (turn, k)
            assert g[1]["refused"].numpy()[0] == 0
    assert (want["lens"] >= prefix + 6).all() and (want["lens"] <= prefix + 6 * (drafts + 1)).all()
    for graph, run in runs:
        lib.hipGraphExecDestroy(run)
        lib.hipGraphDestroy(graph)


def test_captured_forks_and_packing():
    """Forks (the number of free pages in place) and a packed pool behind them, recorded once, replayed over other tables and pages: as eager calls."""
    from caten_amd import _lib, ops
    lib = _lib.init()
    stream = C.c_void_p(lib.cthip_stream())
    n, table, n_pages, layers, kv, dh, forks = 9, 6, 60, 3, 2, 64, 4
    page = int(lib.cthip_kv_page_bytes_q4(kv, dh))
    r = np.random.default_rng(45)

    def some():
        lens = r.integers(0, table * PAGE + 1, n)
        ids, tables = r.permutation(n_pages), np.full((n, table), -1)
        used = 0
        for i in range(n):
            c = -(-int(lens[i]) // PAGE)
            tables[i, :c] = ids[used:used + c]
            used += c
        who = r.permutation(n)
        parents, children = r.choice(who[:n - forks], forks), who[n - forks:]
        return dict(tables=tables, lens=lens, free=np.concatenate([ids[used:], np.full(used, -1)]), n=[n_pages - used], parents=parents, children=children, at=[r.integers(0, lens[p] + 1) for p in parents],
                    pools=r.integers(0, 256, (2, layers, n_pages, page), np.uint8))

    def fresh():
        d = {k: ops.DeviceArray((m,), np.int32) for k, m in dict(tables=n * table, lens=n, free=n_pages, n=1, parents=forks, children=forks, at=forks, refused=forks).items()}
        d["pools"], d["ws"] = ops.DeviceArray((2 * layers * n_pages * page,), np.uint8), ops.DeviceArray((64 + 8 * n_pages,), np.uint8)

        def feed(case):
            for k, v in case.items():
                a = np.ascontiguousarray(v, np.uint8 if k == "pools" else np.int32)
                _lib.check(lib.cthip_h2d(d[k].ptr, a.ctypes.data, a.nbytes))

        def step():
            kp, vp = d["pools"].ptr, d["pools"].ptr + layers * n_pages * page
            _lib.check(lib.cthip_kv_fork_paged_q4(d["tables"].ptr, table, d["lens"].ptr, n, d["n"].ptr, d["refused"].ptr, kp, vp, layers, n_pages, d["parents"].ptr, d["children"].ptr, d["at"].ptr, forks,
                                                  d["free"].ptr, d["n"].ptr, kv, dh))
            _lib.check(lib.cthip_kv_compact_paged_q4(d["tables"].ptr, d["free"].ptr, d["n"].ptr, kp, vp, layers, n_pages, d["tables"].ptr, table, d["lens"].ptr, n, kv, dh, d["ws"].ptr))
        return d, feed, step

    eager, graphed = fresh(), fresh()
    graph, run = C.c_void_p(), C.c_void_p()
    assert lib.hipStreamBeginCapture(stream, 1) == 0
    graphed[2]()
    assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert lib.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    moved = 0
    for _ in range(5):
        case = some()
        eager[1](case)
        eager[2]()
        graphed[1](case)
        assert lib.hipGraphLaunch(run, stream) == 0
        for k in ("tables", "lens", "free", "n", "refused"):
            assert np.array_equal(graphed[0][k].numpy(), eager[0][k].numpy()), k
        used = n_pages - int(eager[0]["n"].numpy()[0])
        a, b = (x[0]["pools"].numpy().reshape(2, layers, n_pages, page) for x in (eager, graphed))
        assert np.array_equal(a, b) and used < n_pages
        moved += (a[:, :, :used] != case["pools"][:, :, :used]).any(-1).sum()
    assert moved > 0
    lib.hipGraphExecDestroy(run)
    lib.hipGraphDestroy(graph)
