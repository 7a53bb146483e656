"""NumPy-in / NumPy-out front-ends of the hand-written fused items.

Each function uploads its operands, calls the C ABI (include/caten_hip.h) and
downloads the result; they exist so that tests and examples read like the
reference's own (`(proceed (!softmax x))` ...).  The hot path itself (the decoder
session, `caten_amd.llm`) keeps everything resident on the device.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import numpy as np

from . import _lib
from .quant import packed_nbytes


class DeviceArray:
    """A flat device allocation from the caching allocator holding a NumPy-typed array."""

    def __init__(self, shape, dtype=np.float32):
        self.shape = tuple(int(s) for s in np.atleast_1d(shape)) if not isinstance(shape, tuple) else shape
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        p = C.c_void_p()
        _lib.check(_lib.init().cthip_alloc(C.byref(p), self.nbytes))
        self.ptr = p.value

    @classmethod
    def from_numpy(cls, a) -> "DeviceArray":
        a = np.ascontiguousarray(a)
        d = cls(a.shape, a.dtype)
        if a.nbytes:
            _lib.check(_lib.load().cthip_h2d(d.ptr, a.ctypes.data, a.nbytes))
        return d

    def numpy(self) -> np.ndarray:
        out = np.empty(self.shape, self.dtype)
        _lib.check(_lib.load().cthip_d2h(out.ctypes.data if out.nbytes else None, self.ptr, out.nbytes))
        return out

    def free(self):
        if self.ptr:
            _lib.check(_lib.load().cthip_free(self.ptr))
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def _dev(a, dtype=np.float32) -> Optional[DeviceArray]:
    return None if a is None else DeviceArray.from_numpy(np.asarray(a, dtype=dtype))


def _p(d: Optional[DeviceArray]):
    return None if d is None else d.ptr


def dequantize(kind: str, raw, n: int) -> np.ndarray:
    """caten/gguf:dequantize (external/gguf/dequantize.lisp:14-53) on the device."""
    raw = np.ascontiguousarray(np.asarray(raw).view(np.uint8).ravel())
    d_raw = DeviceArray.from_numpy(raw)
    out = DeviceArray((n,), np.float32)
    _lib.check(_lib.load().cthip_dequant(_lib.GGML_TYPE[kind], d_raw.ptr, n, out.ptr))
    return out.numpy()


class WeightMatrix:
    """A Linear weight (rows=out, cols=in) kept packed in HBM (cthip_wmat_*)."""

    def __init__(self, kind: str, raw, rows: int, cols: int):
        raw = np.ascontiguousarray(np.asarray(raw).view(np.uint8).ravel())
        want = packed_nbytes(kind, rows * cols)
        if raw.size != want:
            raise ValueError(f"WeightMatrix: {raw.size} bytes given, a {kind} ({rows},{cols}) matrix has {want}")
        self.kind, self.rows, self.cols = kind, rows, cols
        d_raw = DeviceArray.from_numpy(raw)
        h = C.c_void_p()
        _lib.check(_lib.init().cthip_wmat_create(C.byref(h), _lib.GGML_TYPE[kind], d_raw.ptr, rows, cols))
        self.handle = h
        d_raw.free()

    @property
    def nbytes(self) -> int:
        return int(_lib.load().cthip_wmat_nbytes(self.handle))

    def dequantize(self) -> np.ndarray:
        out = DeviceArray((self.rows, self.cols), np.float32)
        _lib.check(_lib.load().cthip_wmat_dequant(self.handle, out.ptr))
        return out.numpy()

    def fold_layernorm(self, gamma, beta, bias=None) -> None:
        """cthip_wmat_fold_layernorm: keeps device copies of gamma / beta / bias (the fold is keyed on their
        addresses) and prepares LayerNorm(gamma, beta) in front of this Linear to go through the product."""
        self._fold = (_dev(np.ascontiguousarray(gamma, np.float32)), _dev(np.ascontiguousarray(beta, np.float32)),
                      _dev(None if bias is None else np.ascontiguousarray(bias, np.float32)))
        dg, db, dbias = self._fold
        _lib.check(_lib.load().cthip_wmat_fold_layernorm(self.handle, dg.ptr, db.ptr, _p(dbias)))

    def linear_folded(self, x, act=None, eps: float = 1e-5) -> np.ndarray:
        """act(LayerNorm(x) @ W^T + bias) with the vectors given to fold_layernorm (fewer than 8 input rows)."""
        dg, db, dbias = self._fold
        x = np.ascontiguousarray(x, np.float32)
        m = x.size // self.cols
        dx = _dev(x)
        y = DeviceArray(x.shape[:-1] + (self.rows,), np.float32)
        _lib.check(_lib.load().cthip_linear(y.ptr, self.handle, dx.ptr, m, _p(dbias), None, _ACT[act],
                                            _PRO["layernorm"], dg.ptr, db.ptr, eps))
        return y.numpy()

    def free(self):
        if self.handle:
            _lib.load().cthip_wmat_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


_ACT = {None: _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU, "silu": _lib.ACT_SILU,
        "sigmoid": _lib.ACT_SIGMOID, "tanh": _lib.ACT_TANH}
_PRO = {None: _lib.PRO_NONE, "layernorm": _lib.PRO_LAYERNORM, "rmsnorm": _lib.PRO_RMSNORM, "swiglu": _lib.PRO_SWIGLU}


def linear(x, w: WeightMatrix, bias=None, residual=None, act=None, prologue=None, norm_g=None, norm_b=None,
           eps: float = 1e-5) -> np.ndarray:
    """Linear with fused neighbours: act(prologue(x) @ W^T + bias) + residual (source/nn/linear.lisp:3-17)."""
    x = np.ascontiguousarray(x, np.float32)
    in_cols = 2 * w.cols if prologue == "swiglu" else w.cols
    if x.shape[-1] != in_cols:
        raise ValueError(f"linear: x has {x.shape[-1]} features, expected {in_cols}")
    m = x.size // in_cols
    dx, db, dr = _dev(x), _dev(bias), _dev(residual)
    dg, dbt = _dev(norm_g), _dev(norm_b)
    y = DeviceArray(x.shape[:-1] + (w.rows,), np.float32)
    _lib.check(_lib.load().cthip_linear(y.ptr, w.handle, dx.ptr, m, _p(db), _p(dr), _ACT[act], _PRO[prologue],
                                        _p(dg), _p(dbt), eps))
    return y.numpy()


def matmul(A, B, relu: bool = False, precision: str = "bf16x6") -> np.ndarray:
    """!matmul (+ fused !relu) (api/high-level-ops.lisp:76-99).

    precision: "fp32" = fp32 MFMA operands; "bf16x6" (default) = operands split in three bf16 terms,
    fp32-grade; "bf16x3" = two terms (2^-16 per product); "bf16" = operands rounded to bf16."""
    A, B = np.ascontiguousarray(A, np.float32), np.ascontiguousarray(B, np.float32)
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError("matmul: inner dimensions differ")
    dA, dB, dC = _dev(A), _dev(B), DeviceArray((M, N), np.float32)
    _lib.check(_lib.load().cthip_matmul(dC.ptr, dA.ptr, dB.ptr, M, N, K, _lib.ACT_RELU if relu else _lib.ACT_NONE,
                                        {"fp32": 0, "bf16": 1, "bf16x3": 2, "bf16x6": 3}[precision]))
    return dC.numpy()


def _rowop(fn_name, x, *vecs, eps=None):
    x = np.ascontiguousarray(x, np.float32)
    n = x.shape[-1] if x.ndim else 0
    rows = x.size // n if n else 0
    dx, dy = _dev(x), DeviceArray(x.shape, np.float32)
    dv = [_dev(v) for v in vecs]
    fn = getattr(_lib.load(), fn_name)
    args = [dy.ptr, dx.ptr] + [_p(v) for v in dv] + ([eps] if eps is not None else []) + [rows, n]
    _lib.check(fn(*args))
    return dy.numpy()


def softmax(x):
    return _rowop("cthip_softmax", x)


def layernorm(x, gamma=None, beta=None, eps=1e-5):
    return _rowop("cthip_layernorm", x, gamma, beta, eps=eps)


def rmsnorm(x, w=None, eps=1e-5):
    return _rowop("cthip_rmsnorm", x, w, eps=eps)


def layernorm_softmax(x, gamma=None, beta=None, eps=1e-5):
    return _rowop("cthip_layernorm_softmax", x, gamma, beta, eps=eps)


def unary(kind: str, x):
    x = np.ascontiguousarray(x, np.float32)
    dx, dy = _dev(x), DeviceArray(x.shape, np.float32)
    _lib.check(_lib.load().cthip_unary(_ACT[kind], dy.ptr, dx.ptr, x.size))
    return dy.numpy()


def relu(x):
    return unary("relu", x)


def gelu(x):
    return unary("gelu", x)


def silu(x):
    return unary("silu", x)


def sigmoid(x):
    return unary("sigmoid", x)


def tanh(x):
    return unary("tanh", x)


def embedding(W, idx):
    W = np.ascontiguousarray(W, np.float32)
    idx = np.ascontiguousarray(idx, np.float32)
    V, D = W.shape
    dW, di, out = _dev(W), _dev(idx), DeviceArray(idx.shape + (D,), np.float32)
    _lib.check(_lib.load().cthip_embedding(out.ptr, dW.ptr, di.ptr, idx.size, V, D))
    return out.numpy()


def argmax(x):
    x = np.ascontiguousarray(x, np.float32)
    n = x.shape[-1]
    rows = x.size // n
    dx, out = _dev(x), DeviceArray(x.shape[:-1] if x.ndim > 1 else (1,), np.int64)
    _lib.check(_lib.load().cthip_argmax(out.ptr, dx.ptr, rows, n))
    r = out.numpy()
    return r if x.ndim > 1 else int(r[0])


def rope(x, base=10000.0, start_pos=0):
    x = np.ascontiguousarray(x, np.float32)
    B, S, H, Dh = x.shape
    dx, out = _dev(x), DeviceArray(x.shape, np.float32)
    _lib.check(_lib.load().cthip_rope(out.ptr, dx.ptr, B, S, H, Dh, base, start_pos))
    return out.numpy()


def sdpa_cached(q, k_cache, v_cache, start_pos: int):
    """q (S,H,Dh) at positions start_pos.., caches (max_len,Hkv,Dh) -> (S,H,Dh), causal."""
    q = np.ascontiguousarray(q, np.float32)
    S, H, Dh = q.shape
    Hkv = k_cache.shape[1]
    dq, dk, dv = _dev(q), _dev(k_cache), _dev(v_cache)
    out = DeviceArray(q.shape, np.float32)
    _lib.check(_lib.load().cthip_sdpa_cached(out.ptr, dq.ptr, dk.ptr, dv.ptr, S, start_pos, H, Hkv, Dh))
    return out.numpy()


def kv_plan(lens, new_lens, tables, free_pages, max_rows: int, n_free: Optional[int] = None) -> dict:
    """Block tables and slot maps of a step of a batch (cthip_kv_plan_paged): `lens` rows held and `new_lens` new ones per
    sequence, `tables` (n, stride) page ids, `free_pages` a stack of which the last `n_free` entries are taken first."""
    lens, new_lens, tables, free_pages = (np.ascontiguousarray(a, np.int32) for a in (lens, new_lens, tables, free_pages))
    n = lens.size
    if new_lens.size != n or tables.ndim != 2 or tables.shape[0] != n:
        raise ValueError(f"kv_plan: {n} lengths, {new_lens.size} new lengths and a table of shape {tables.shape}")
    n_free = free_pages.size if n_free is None else int(n_free)
    if not 0 <= n_free <= free_pages.size:
        raise ValueError(f"kv_plan: {n_free} free pages of a stack of {free_pages.size}")
    d_lens, d_new, d_tables, d_free, d_n = (DeviceArray.from_numpy(a) for a in (lens, new_lens, tables, free_pages, np.array([n_free], np.int32)))
    slots, positions, starts, refused = (DeviceArray((m,), np.int32) for m in (max_rows, max_rows, n + 1, 1))
    _lib.check(_lib.load().cthip_kv_plan_paged(slots.ptr, positions.ptr, starts.ptr, d_tables.ptr, tables.shape[1], d_lens.ptr, d_n.ptr, refused.ptr, d_lens.ptr,
                                               d_new.ptr, n, d_free.ptr, d_n.ptr, max_rows))
    return dict(slots=slots.numpy(), positions=positions.numpy(), starts=starts.numpy(), tables=d_tables.numpy(), lens=d_lens.numpy(), n_free=int(d_n.numpy()[0]),
                refused=int(refused.numpy()[0]))


def kv_free_pages(tables, lens, n_pages: int) -> np.ndarray:
    """The pages of a pool that no sequence's rows are in (cthip_kv_free_paged), as a stack for `kv_plan`."""
    tables, lens = (np.ascontiguousarray(a, np.int32) for a in (tables, lens))
    if tables.ndim != 2 or tables.shape[0] != lens.size:
        raise ValueError(f"kv_free_pages: {lens.size} lengths and a table of shape {tables.shape}")
    d_tables, d_lens = DeviceArray.from_numpy(tables), DeviceArray.from_numpy(lens)
    d_free, d_n = DeviceArray((max(n_pages, 1),), np.int32), DeviceArray((1,), np.int32)
    _lib.check(_lib.init().cthip_kv_free_paged(d_free.ptr, d_n.ptr, d_tables.ptr, tables.shape[1], d_lens.ptr, lens.size, n_pages))
    return d_free.numpy()[:int(d_n.numpy()[0])]


class PagedCacheQ4:
    """The keys and values of a batch of sequences in 4 bits, in pages of 64 rows (one layer, or `layers` of them)."""

    def __init__(self, n_pages: int, kv_heads: int, head_dim: int, layers: int = 1):
        self.n_pages, self.kv_heads, self.head_dim, self.layers = n_pages, kv_heads, head_dim, layers
        lib = _lib.init()
        self.page_bytes = int(lib.cthip_kv_page_bytes_q4(kv_heads, head_dim))
        if self.page_bytes < 0:
            _lib.check(self.page_bytes)
        self.k, self.v = (DeviceArray((layers, n_pages, self.page_bytes), np.uint8) for _ in range(2))
        self.workspace = DeviceArray((int(lib.cthip_sdpa_paged_q4_workspace(head_dim)),), np.uint8)

    def _pools(self, layer):
        if not 0 <= layer < self.layers:
            raise ValueError(f"PagedCacheQ4: layer {layer} of {self.layers}")
        at = layer * self.n_pages * self.page_bytes
        return self.k.ptr + at, self.v.ptr + at

    def append(self, k, v, slots, layer: int = 0) -> None:
        """Rows (n, kv_heads, head_dim) into the cache rows `slots`."""
        width = self.kv_heads * self.head_dim
        k, v = (np.ascontiguousarray(a, np.float32).reshape(-1, width) for a in (k, v))
        slots = np.ascontiguousarray(slots, np.int32).ravel()
        if k.shape != v.shape or slots.size != k.shape[0]:
            raise ValueError(f"PagedCacheQ4.append: keys {k.shape}, values {v.shape}, {slots.size} slots")
        dk, dv, ds = (DeviceArray.from_numpy(a) for a in (k, v, slots))
        kp, vp = self._pools(layer)
        _lib.check(_lib.load().cthip_kv_append_paged_q4(kp, vp, dk.ptr, dv.ptr, width, width, ds.ptr, slots.size, self.n_pages, self.kv_heads, self.head_dim))

    def rows(self, slots, layer: int = 0):
        """The keys and values of cache rows, (n, kv_heads, head_dim) each; rows outside the pool are zero."""
        slots = np.ascontiguousarray(slots, np.int32).ravel()
        ds = DeviceArray.from_numpy(slots)
        k, v = (DeviceArray((slots.size, self.kv_heads, self.head_dim), np.float32) for _ in range(2))
        kp, vp = self._pools(layer)
        _lib.check(_lib.load().cthip_kv_rows_paged_q4(k.ptr, v.ptr, kp, vp, ds.ptr, slots.size, self.n_pages, self.kv_heads, self.head_dim))
        return k.numpy(), v.numpy()

    def attend(self, q, tables, lens, starts, layer: int = 0) -> np.ndarray:
        """q (rows, heads, head_dim): rows starts[i] .. starts[i + 1] are the last ones of sequence i, which holds lens[i] keys."""
        q = np.ascontiguousarray(q, np.float32)
        n_rows, heads, dh = q.shape
        if dh != self.head_dim:
            raise ValueError(f"PagedCacheQ4.attend: heads of {dh}, the cache's have {self.head_dim}")
        tables, lens, starts = (np.ascontiguousarray(a, np.int32) for a in (tables, lens, starts))
        if tables.ndim != 2 or tables.shape[0] != lens.size or starts.size != lens.size + 1:
            raise ValueError(f"PagedCacheQ4.attend: a table of shape {tables.shape}, {lens.size} lengths, {starts.size} starts")
        dq, dt, dl, ds = (DeviceArray.from_numpy(a) for a in (q, tables, lens, starts))
        out = DeviceArray(q.shape, np.float32)
        kp, vp = self._pools(layer)
        _lib.check(_lib.load().cthip_sdpa_paged_q4(out.ptr, dq.ptr, heads * dh, kp, vp, self.n_pages, dt.ptr, tables.shape[1], dl.ptr, ds.ptr, lens.size, n_rows, heads,
                                                   self.kv_heads, dh, self.workspace.ptr))
        return out.numpy()

    def reorder(self, tables, lens, parents, history=None, tokens=None, step: int = 0):
        """A beam search's reordering (cthip_beam_reorder_paged_q4) in all layers: `parents` (requests, beams), `lens` per
        request, `tables` (requests * beams, stride).  Returns the new tables, and the new history where one is given."""
        tables, lens, parents = (np.ascontiguousarray(a, np.int32) for a in (tables, lens, parents))
        if parents.ndim != 2 or lens.size != parents.shape[0] or tables.ndim != 2 or tables.shape[0] != parents.size:
            raise ValueError(f"PagedCacheQ4.reorder: parents {parents.shape}, {lens.size} lengths, a table of shape {tables.shape}")
        dt, dl, dp = (DeviceArray.from_numpy(a) for a in (tables, lens, parents))
        out = DeviceArray(tables.shape, np.int32)
        dh = do = dtok = dstep = None
        cols = 0
        if history is not None:
            history, tokens = np.ascontiguousarray(history, np.int32), np.ascontiguousarray(tokens, np.int32)
            if history.ndim != 2 or history.shape[0] != parents.size or tokens.size != parents.size:
                raise ValueError(f"PagedCacheQ4.reorder: a history of shape {history.shape} and {tokens.size} tokens for {parents.size} beams")
            cols = history.shape[1]
            dh, dtok, dstep, do = DeviceArray.from_numpy(history), DeviceArray.from_numpy(tokens), DeviceArray.from_numpy(np.array([step], np.int32)), DeviceArray(history.shape, np.int32)
        _lib.check(_lib.load().cthip_beam_reorder_paged_q4(out.ptr, _p(do), self.k.ptr, self.v.ptr, self.layers, self.n_pages, dt.ptr, tables.shape[1], dl.ptr, dp.ptr, parents.shape[0],
                                                           parents.shape[1], self.kv_heads, self.head_dim, _p(dh), cols, _p(dtok), _p(dstep)))
        return out.numpy() if history is None else (out.numpy(), do.numpy())


def beam_select(logits, scores, finished=None, eos: int = -1) -> dict:
    """The best continuations of each request's beams (cthip_beam_select): logits (requests, beams, vocab), scores (requests, beams)."""
    logits, scores = np.ascontiguousarray(logits, np.float32), np.ascontiguousarray(scores, np.float32)
    if logits.ndim != 3 or logits.shape[:2] != scores.shape:
        raise ValueError(f"beam_select: logits {logits.shape}, scores {scores.shape}")
    if finished is not None and np.shape(finished) != scores.shape:
        raise ValueError(f"beam_select: scores {scores.shape}, finished {np.shape(finished)}")
    n, k, vocab = logits.shape
    size = int(_lib.init().cthip_beam_select_workspace(n, k))
    if size < 0:
        _lib.check(size)
    dl, dsc, ws = DeviceArray.from_numpy(logits), DeviceArray.from_numpy(scores), DeviceArray((size,), np.uint8)
    df = _dev(finished, np.int32)
    tokens, parents, done = (DeviceArray((n, k), np.int32) for _ in range(3))
    best = DeviceArray((n, k), np.float32)
    _lib.check(_lib.load().cthip_beam_select(tokens.ptr, parents.ptr, best.ptr, done.ptr, dl.ptr, vocab, dsc.ptr, _p(df), n, k, vocab, eos, ws.ptr))
    return dict(tokens=tokens.numpy(), parents=parents.numpy(), scores=best.numpy(), finished=done.numpy())
