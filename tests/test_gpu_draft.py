"""Drafted tokens against the target's probabilities, against the definition (include/caten_hip.h) step by step in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def verified(target, draft, tokens, uniforms, starts, lens, positions=None):
    vocab = target.shape[1]
    out, accepted, left = np.full(len(tokens), -1), [], list(lens)
    for i in range(len(starts) - 1):
        r0, r1 = int(starts[i]), int(starts[i + 1])
        if not (0 <= r0 < r1 <= len(tokens)) or (positions is not None and positions[r0] < 0):
            accepted.append(0)
            continue
        n, p, q = r1 - r0 - 1, target.astype(np.float64), None if draft is None else draft.astype(np.float64)
        stay = 0
        while stay < n:
            r, x = r0 + stay, tokens[r0 + stay + 1]
            if not (0 <= x < vocab) or not float(uniforms[r]) * (1.0 if q is None else q[r, x]) < p[r, x]:
                break
            stay += 1
        r = r0 + stay
        own = np.where(p[r] > 0, p[r], 0.0)
        w = own
        if stay < n:
            if q is None:
                w = own.copy()
                if 0 <= tokens[r + 1] < vocab:
                    w[tokens[r + 1]] = 0.0
            else:
                w = p[r] - q[r]
                w = np.where(w > 0, w, 0.0)
        if not w.sum() > 0:
            w = own
        token = -1
        if w.sum() > 0:
            upto = np.cumsum(w)
            past = np.flatnonzero((upto > float(uniforms[r1 - 1]) * upto[-1]) & (w > 0))
            token = past[0] if len(past) else np.flatnonzero(w > 0)[-1]
        out[r0:r1] = np.concatenate([tokens[r0 + 1:r + 1], [token], np.full(n - stay, -1)])
        accepted.append(stay)
        left[i] -= n - stay
    return dict(tokens=out, accepted=np.array(accepted), lens=np.array(left))


def same(got, want):
    for key in want:
        assert np.array_equal(got[key], want[key]), (key, got[key], want[key])


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def some(rng, drafts, vocab, near=0.7):
    """Drafts of a model near the target; tokens drawn from the draft's probabilities."""
    starts = np.concatenate([[0], np.cumsum([d + 1 for d in drafts])])
    rows = starts[-1]
    x = 2.5 * rng.normal(0, 1, (rows, vocab))
    draft, target = softmax(x), softmax(x + near * rng.normal(0, 1, x.shape))
    tokens = np.zeros(rows, np.int64)
    for r in range(rows - 1):
        tokens[r + 1] = min(np.searchsorted(np.cumsum(draft[r].astype(np.float64)), rng.random(), side="right"), vocab - 1)
    lens = np.array([d + 1 + rng.integers(0, 500) for d in drafts])
    return target, draft, tokens, rng.random(rows).astype(np.float32), starts, lens


@pytest.mark.parametrize("drafts,vocab", [(d, v) for d in ([0], [1], [4], [3, 0, 5, 1, 0, 7]) for v in (1, 2, 63, 64, 257, 1024, 1025, 4099, 65537)] + [([70, 2, 130, 64, 63], v) for v in (2, 64, 1025)])
@pytest.mark.parametrize("sure", [False, True])
def test_drafts(drafts, vocab, sure):
    print(f"case: drafts {drafts}, vocabulary {vocab}, {'certain' if sure else 'drawn'}", flush=True)
    from caten_amd import ops
    rng = np.random.default_rng(vocab + len(drafts))
    for near in (0.0, 0.5, 3.0):
        target, draft, tokens, uniforms, starts, lens = some(rng, drafts, vocab, near)
        draft = None if sure else draft
        same(ops.draft_verify(target, draft, tokens, uniforms, starts, lens), verified(target, draft, tokens, uniforms, starts, lens))


def test_a_large_vocabulary_and_many_sequences():
    from caten_amd import ops
    rng = np.random.default_rng(2)
    for drafts, vocab in (([3] * 5, 200003), (rng.integers(0, 4, 700), 300)):
        args = some(rng, list(drafts), vocab)
        same(ops.draft_verify(*args), verified(*args))


@pytest.mark.parametrize("n,vocab,draft", [(150, 17003, False), (70, 16 * 1024 + 1, True), (450, 4099, False)])
def test_workgroups_of_several_slices(n, vocab, draft):
    from caten_amd import ops
    rng = np.random.default_rng(n)
    args = list(some(rng, [1 if draft else 0] * n, vocab))
    same(ops.draft_verify(*args), verified(*args))


def test_borders():
    """Weights that are whole steps of 1/256: sums and products are exact in any order, and a number on a border belongs to the token behind it."""
    from caten_amd import ops
    vocab, n = 4096 + 17, 200
    rng = np.random.default_rng(4)
    target = np.zeros((n, vocab), np.float32)
    for r in range(n):
        at = rng.choice(vocab, 64, replace=False)
        target[r, at] = 4 / 256
    uniforms = (rng.integers(0, 64, n) / 64).astype(np.float32)
    uniforms[:4] = 0.0, 1 - 2.0 ** -24, 63 / 64, 1 / 64
    starts = np.arange(n + 1)
    args = (target, None, np.zeros(n, np.int64), uniforms, starts, np.ones(n, np.int64))
    want = verified(*args)
    got = ops.draft_verify(*args)
    same(got, want)
    for r in (0, 1, 2, 3):  # by hand
        at = np.flatnonzero(target[r])
        assert got["tokens"][r] == at[int(uniforms[r] * 64)]


def test_comparisons_at_equality():
    """u q = p exactly is a rejection; the next number below stays.  p = q everywhere: rejected by u = 1 only, and then from the target itself."""
    from caten_amd import ops
    target, draft = np.full((3, 8), 0.125, np.float32), np.full((3, 8), 0.25, np.float32)
    draft[:, 4:] = 0.0
    for u, stays in ((0.5, 0), (np.nextafter(np.float32(0.5), np.float32(0)), 1)):
        args = (target, draft, np.array([0, 2, 0]), np.array([u, 0.3, 0.9], np.float32), np.array([0, 2, 3]), np.array([10, 20]))
        got = ops.draft_verify(*args)
        same(got, verified(*args))
        assert got["accepted"][0] == stays and got["tokens"][0] == (2 if stays else 5)  # max(p - q, 0) is even over 4 .. 7
    args = (target, target, np.array([0, 2, 0]), np.array([1.0, 0.3, 0.9], np.float32), np.array([0, 2, 3]), np.array([10, 20]))
    got = ops.draft_verify(*args)
    same(got, verified(*args))
    assert got["accepted"][0] == 0 and got["tokens"][0] == 2


def test_numbers_that_are_none():
    from caten_amd import ops
    rng = np.random.default_rng(7)
    target, draft, tokens, uniforms, starts, lens = some(rng, [2, 2, 2, 2, 0, 0, 0, 1, 1], 900)
    target[0, tokens[1]] = np.nan
    draft[3, tokens[4]] = np.nan
    uniforms[6], uniforms[8] = np.nan, np.nan
    uniforms[9], uniforms[11] = -1.0, 2.0
    target[12], target[13] = np.nan, 0.0
    target[14, ::3] = -target[14, ::3]
    target[15] = 0.0                        # the draft is rejected, and nothing is left of the target
    tokens[18] = 900                        # outside the vocabulary
    args = (target, draft, tokens, uniforms, starts, lens)
    got, want = ops.draft_verify(*args), verified(*args)
    same(got, want)
    assert got["tokens"][12] == -1 and got["tokens"][13] == -1 and got["tokens"][15] == -1 and got["accepted"][8] == 0


def test_probabilities_below_nothing():
    """They count as 0, the draft's too: its token is not accepted where the target excludes it, and the difference is not more than the target."""
    from caten_amd import ops
    target = np.zeros((8, 6), np.float32)
    target[:, 2:] = [0.5, 0.25, 0.25, 0.0]
    draft = np.zeros((8, 6), np.float32)
    draft[:, 3] = 1.0
    tokens, uniforms, starts = np.zeros(8, np.int64), np.full(8, 0.9, np.float32), np.array([0, 2, 4, 6, 8])
    draft[0, 1], tokens[1] = -0.5, 1                           # the target has nothing for the draft: rejected
    draft[2, 2], draft[2, 0], tokens[3] = -7.0, -1.0, 3        # rejected; left are 2 (0.5) and 4 (0.25)
    target[4, 5], draft[4, 5], tokens[5] = -0.25, -1.0, 5      # both below nothing: rejected, and 5 has no weight
    draft[6, 4], tokens[7] = -np.inf, 4                        # the target has something for it: accepted
    uniforms[[1, 3, 5]] = 0.1, 0.6, 0.999
    want = dict(tokens=[2, -1, 2, -1, 4, -1, 4, 4], accepted=[0, 0, 0, 1], lens=[9, 9, 9, 10])
    same(ops.draft_verify(target, draft, tokens, uniforms, starts, [10] * 4), {k: np.array(v) for k, v in want.items()})
    # over a vocabulary of several slices: the definition with such a draft's zeros
    rng = np.random.default_rng(13)
    target, draft, tokens, uniforms, starts, lens = some(rng, [3, 0, 5, 1, 1, 2], 4099)
    clean = np.where(rng.random(draft.shape) < 0.3, 0.0, draft).astype(np.float32)
    for below in (-1.0, -1e-30, -np.inf):
        draft = np.where(clean == 0, np.float32(below), clean)
        same(ops.draft_verify(target, draft, tokens, uniforms, starts, lens), verified(target, clean, tokens, uniforms, starts, lens))


def test_sequences_that_sit_out():
    """No rows, rows refused by the plan, rows outside; lengths may be left out, in place or apart."""
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(9)
    target, draft, tokens, uniforms, starts, lens = some(rng, [2, 1, 3, 0], 500)
    starts = np.array([0, 3, 3, 5, 9, 10])
    lens = np.array([50, 7, 60, 70, 80])
    positions = np.arange(10)
    positions[3:5] = -1
    args = (target, draft, tokens, uniforms, starts, lens, positions)
    want = verified(*args)
    same(ops.draft_verify(*args), want)
    assert list(want["tokens"][3:5]) == [-1, -1] and want["lens"][2] == 60
    got = ops.draft_verify(target, draft, tokens, uniforms, starts)
    same(got, {k: v for k, v in verified(target, draft, tokens, uniforms, starts, lens).items() if k != "lens"})
    # the last sequence's row is outside
    d = {k: ops.DeviceArray.from_numpy(np.ascontiguousarray(v, t)) for k, v, t in (("target", target, np.float32), ("draft", draft, np.float32), ("tokens", tokens, np.int32),
                                                                                 ("u", uniforms, np.float32), ("starts", starts, np.int32), ("lens", lens, np.int32))}
    out, accepted, left, ws = ops.DeviceArray.from_numpy(np.full(10, 77, np.int32)), ops.DeviceArray((5,), np.int32), ops.DeviceArray((5,), np.int32), ops.DeviceArray((5 * 2048,), np.uint8)
    for to in (left, d["lens"]):
        _lib.check(lib.cthip_draft_verify(out.ptr, accepted.ptr, to.ptr, d["target"].ptr, 500, d["draft"].ptr, 500, d["tokens"].ptr, d["u"].ptr, d["starts"].ptr, None, d["lens"].ptr, 5, 9, 500,
                                          ws.ptr))
        want = verified(target[:9], draft[:9], tokens[:9], uniforms[:9], starts, lens)
        assert np.array_equal(out.numpy()[:9], want["tokens"]) and out.numpy()[9] == 77
        assert np.array_equal(accepted.numpy(), want["accepted"]) and np.array_equal(to.numpy(), want["lens"])


@pytest.mark.parametrize("starts", [[1, -2 ** 31], [5, -2 ** 31 + 3, 4], [-2 ** 31, 2 ** 31 - 1, -1], [-1, 3, 2 ** 31 - 1, 0], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]])
def test_starts_far_outside(starts):
    """Differences of starts that 32 bits do not hold are no rows."""
    from caten_amd import ops
    target, draft, tokens, uniforms, _, _ = some(np.random.default_rng(12), [3, 2], 100)
    got = ops.draft_verify(target, draft, tokens, uniforms, starts, np.arange(len(starts) - 1) + 10)
    same(got, verified(target, draft, tokens, uniforms, starts, np.arange(len(starts) - 1) + 10))


def test_strides():
    from caten_amd import _lib, ops
    lib, rng = _lib.init(), np.random.default_rng(10)
    target, draft, tokens, uniforms, starts, lens = some(rng, [3, 2, 0], 1203)
    wide_t, wide_d = np.full((len(tokens), 1300), 9.0, np.float32), np.full((len(tokens), 1211), np.nan, np.float32)
    wide_t[:, 1:1204], wide_d[:, 3:1206] = target, draft
    d = [ops.DeviceArray.from_numpy(a) for a in (wide_t, wide_d, tokens.astype(np.int32), uniforms, starts.astype(np.int32), lens.astype(np.int32))]
    out, accepted, left, ws = (ops.DeviceArray((n,), np.int32) for n in (len(tokens), 3, 3, 3 * 512))
    _lib.check(lib.cthip_draft_verify(out.ptr, accepted.ptr, left.ptr, d[0].ptr + 4, 1300, d[1].ptr + 12, 1211, d[2].ptr, d[3].ptr, d[4].ptr, None, d[5].ptr, 3, len(tokens), 1203, ws.ptr))
    same(dict(tokens=out.numpy(), accepted=accepted.numpy(), lens=left.numpy()), verified(target, draft, tokens, uniforms, starts, lens))


def test_what_comes_out_is_the_targets_distribution():
    """20000 sequences of one draft each, drawn from the draft's probabilities: the first token out has the target's.  A count's standard deviation is
    sqrt(n p (1 - p)); six of them are exceeded once in 10^9."""
    from caten_amd import ops
    rng = np.random.default_rng(11)
    n, vocab = 20000, 12
    p, q = softmax(rng.normal(0, 1, vocab)), softmax(rng.normal(0, 1, vocab))
    tokens = np.zeros(2 * n, np.int64)
    tokens[1::2] = rng.choice(vocab, n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    got = ops.draft_verify(np.tile(p, (2 * n, 1)), np.tile(q, (2 * n, 1)), tokens, rng.random(2 * n).astype(np.float32), np.arange(0, 2 * n + 1, 2))
    count = np.bincount(got["tokens"][::2], minlength=vocab)
    assert (np.abs(count - n * p) <= 6 * np.sqrt(n * p * (1 - p)) + 1).all()
    assert 0.2 * n < got["accepted"].sum() < n


def test_refusals():
    from caten_amd import _lib, ops
    lib, d = _lib.init(), ops.DeviceArray((1 << 16,), np.uint8)
    p = d.ptr

    def call(**k):
        a = dict(out=p, acc=p + 1024, lens_out=p + 2048, t=p + 4096, ts=16, d=p + 8192, ds=16, tok=p + 12288, u=p + 13312, starts=p + 14336, pos=None, lens=p + 15360, n=2, rows=4, vocab=16,
                 ws=p + 16384)
        a.update(k)
        return lib.cthip_draft_verify(*a.values())

    for bad in (dict(n=-1), dict(rows=-1), dict(vocab=0), dict(ts=15), dict(ds=15), dict(acc=None), dict(starts=None), dict(ws=None), dict(ws=p + 16388), dict(lens=None), dict(out=None),
                dict(t=None), dict(tok=None), dict(u=None), dict(out=p + 12288), dict(vocab=(1 << 30) + 1, ts=1 << 31, ds=1 << 31)):
        assert call(**bad) == _lib.E_BAD_ARG, bad
    assert call(n=65536) == _lib.E_UNSUPPORTED
    assert call(n=0, acc=None, starts=None) == 0 and call(d=None, ds=0, lens_out=None, lens=None) == 0
    with pytest.raises(_lib.HipError):
        _lib.check(call(ts=15))
