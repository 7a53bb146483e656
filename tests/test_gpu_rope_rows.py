"""Query and key rows turned by positions of their own, against the definition in 64 bits.  The reference turns neighbouring channels of whole heads
at consecutive positions (nn/positional-encoding.lisp:3-64)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def turned(x, positions, frequencies, layout, magnitude):
    """And what the pair of each channel comes to, for the tolerance."""
    x = np.asarray(x, np.float64)
    out, size, half = x.copy(), np.zeros(x.shape), len(frequencies)
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if layout == "pairs" else (i, i + half)
    angle = np.asarray(positions, np.float64)[:, None, None] * frequencies
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = magnitude * (a * np.cos(angle) - b * np.sin(angle)), magnitude * (a * np.sin(angle) + b * np.cos(angle))
    size[..., first] = size[..., second] = abs(magnitude) * (np.abs(a) + np.abs(b))
    stay = np.asarray(positions) < 0
    out[stay], size[stay] = x[stay], 0.0
    return out, size


def close(got, want, size):
    """Sine and cosine off by 2^-23, times the magnitude (2^-24 of it), a product's rounding and the sum's (2^-24 each): below 2^-21 of |a| + |b|.  What does not turn is the same."""
    assert (np.abs(got - want) <= 2.0 ** -21 * size).all(), float(np.max(np.abs(got - want) / np.maximum(size, 1e-30)))


CASES = [(12, 12, 64, 64), (32, 4, 64, 64), (64, 8, 128, 128), (32, 32, 128, 32), (6, 2, 32, 8), (10, 5, 80, 40), (21, 3, 96, 24), (1, 0, 64, 64), (3, 1, 6, 6), (5, 2, 10, 4), (2, 1, 2, 2),
         (7, 7, 36, 18), (300, 1, 4, 4), (3, 2, 1024, 1024), (2, 1, 2100, 2052), (4, 4, 64, 0), (1, 1, 256, 2)]


@pytest.mark.parametrize("H,kv,dh,rotary", CASES)
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("rows", [1, 5, 130])
def test_rows(H, kv, dh, rotary, layout, rows):
    print(f"case: rope {rows} rows, {H} + {kv} heads of {dh}, {rotary} of them, {layout}", flush=True)
    from caten_amd import ops
    rng = np.random.default_rng(H + dh + rows)
    q, k = (rng.normal(0, 1, (rows, n, dh)).astype(np.float32) for n in (H, kv))
    positions = rng.integers(0, 5000, rows)
    positions[rows // 3] = -1 if rows > 1 else 0
    f = ops.rope_frequencies(rotary)
    got_q, got_k = ops.rope_rows(q, k, positions, f, layout, 1.25)
    close(got_q, *turned(q, positions, f, layout, 1.25))
    close(got_k, *turned(k, positions, f, layout, 1.25))


@pytest.mark.parametrize("layout", ["pairs", "halves"])
def test_far_positions(layout):
    """Angles of up to 2^31 radians: the same product of 64 bits on both sides."""
    from caten_amd import ops
    rng = np.random.default_rng(3)
    positions = np.array([0, 1, 2, 8191, 131071, 10 ** 6, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31 - 2, 77777777])
    q, k = (rng.normal(0, 1, (len(positions), n, 128)).astype(np.float32) for n in (5, 2))
    for f in (ops.rope_frequencies(128), ops.rope_frequencies(128, 500000.0, 8.0, 8192), ops.rope_frequencies(128, factor=4.0), -ops.rope_frequencies(128)):
        got_q, got_k = ops.rope_rows(q, k, positions, f, layout)
        close(got_q, *turned(q, positions, f, layout, 1.0))
        close(got_k, *turned(k, positions, f, layout, 1.0))


def test_quarter_turns():
    """Angles around every eighth of a turn."""
    from caten_amd import ops
    n = 400
    f = np.concatenate([np.pi / 4 * j + np.array([-1e-7, 0.0, 1e-12, 1e-4]) for j in range(-8, 24)])
    q = np.random.default_rng(5).normal(0, 1, (n, 1, 2 * f.size)).astype(np.float32)
    positions = np.arange(n)
    got, _ = ops.rope_rows(q, None, positions, f, "halves")
    close(got, *turned(q, positions, f, "halves", 1.0))


def test_the_layout_of_the_reference():
    """Consecutive positions, whole heads: cthip_rope, which rounds its angles to 32 bits (2^-24 of a position at the first pair)."""
    from caten_amd import ops
    rng = np.random.default_rng(6)
    x = rng.normal(0, 1, (1, 300, 4, 64)).astype(np.float32)
    want = ops.rope(x, 10000.0, 40)[0]
    got, _ = ops.rope_rows(x[0], None, np.arange(40, 340), ops.rope_frequencies(64))
    # theta is off by some 2^-21 of itself there (a power by logarithms in 32 bits), the angle below 340 by 340 * 2^-21 and its own 2^-24
    assert (np.abs(got - want) <= 8 * 340 * 2.0 ** -21).all()


@pytest.mark.parametrize("dh,rotary,layout", [(64, 64, 0), (64, 48, 1), (10, 6, 1), (10, 6, 0)])
def test_strided_out_of_place_and_untouched(dh, rotary, layout):
    """Slices of fused rows into rows of another stride, at addresses of 4 bytes' alignment; what lies between stays, and so do rows at -1."""
    from caten_amd import _lib, ops
    lib, rng, rows, H, kv = _lib.init(), np.random.default_rng(8), 70, 5, 2
    w, wq, wk = (H + 2 * kv) * dh + 3, H * dh + 5, kv * dh + 1
    fused = rng.normal(0, 1, (rows, w)).astype(np.float32)
    positions = rng.integers(-1, 300, rows).astype(np.int32)
    positions[[3, 60]] = -1, -2 ** 31
    f = ops.rope_frequencies(rotary)
    src, dp, df = (ops.DeviceArray.from_numpy(a) for a in (fused, positions, f))
    oq, ok = (ops.DeviceArray.from_numpy(np.full((rows, n), 7.0, np.float32)) for n in (wq, wk))
    _lib.check(lib.cthip_rope_rows(oq.ptr + 4, wq, ok.ptr, wk, src.ptr + 4, w, src.ptr + 4 * (1 + H * dh), w, dp.ptr, rows, H, kv, dh, rotary, layout, df.ptr, 1.0))
    name = ("pairs", "halves")[layout]
    q, k = fused[:, 1:1 + H * dh].reshape(rows, H, dh), fused[:, 1 + H * dh:1 + (H + kv) * dh].reshape(rows, kv, dh)
    there = positions >= 0
    for x, got, first, width in ((q, oq.numpy(), 1, H * dh), (k, ok.numpy(), 0, kv * dh)):
        want, size = turned(x, positions, f, name, 1.0)
        close(got[there, first:first + width].reshape(-1, x.shape[1], dh), want[there], size[there])
        assert (got[~there] == 7.0).all() and (np.delete(got, np.s_[first:first + width], 1) == 7.0).all()
    assert np.array_equal(src.numpy(), fused)


def test_refusals():
    from caten_amd import _lib, ops
    lib = _lib.init()
    d = ops.DeviceArray((4096,), np.float32)
    p = d.ptr

    def call(**k):
        a = dict(qo=p, qos=128, ko=p + 4096, kos=64, q=p, qs=128, k=p + 4096, ks=64, pos=p + 8192, n=2, H=2, kv=1, dh=64, rotary=64, layout=0, f=p + 12288, m=1.0)
        a.update(k)
        return lib.cthip_rope_rows(*a.values())

    for bad in (dict(n=-1), dict(H=-1), dict(kv=-1), dict(dh=-1), dict(rotary=3), dict(rotary=66), dict(rotary=-2), dict(layout=2), dict(layout=-1), dict(q=None), dict(qo=None), dict(k=None),
                dict(ko=None), dict(qs=127), dict(qos=127), dict(ks=63), dict(kos=63), dict(pos=None), dict(f=None), dict(qos=200), dict(kos=65)):
        assert call(**bad) == _lib.E_BAD_ARG, bad
    for bad in (dict(n=(1 << 23) + 1), dict(H=65536, qs=1 << 30, qos=1 << 30), dict(kv=65536, ks=1 << 30, kos=1 << 30), dict(dh=65536, qs=1 << 30, qos=1 << 30, ks=1 << 30, kos=1 << 30),
                dict(dh=33, rotary=32)):
        assert call(**bad) == _lib.E_UNSUPPORTED, bad
    assert call(n=0, q=None, pos=None) == 0 and call(H=0, kv=0, q=None, k=None, pos=None) == 0 and call(dh=0, rotary=0, q=None) == 0
    assert not d.numpy().any()
