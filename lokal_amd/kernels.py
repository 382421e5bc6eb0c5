"""Kernel-level entry points of the HIP backend on device buffers.

These wrap the "kernels" part of include/lokal_hip.h: device memory
(DeviceArray), weights uploaded in their GGUF type (Weight), and one call per
hot-path kernel.  Calls are asynchronous on the given stream (None = null
stream); DeviceArray.numpy() synchronises.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import LKHIP_F16, LKHIP_F32, KvPagesDesc, PageTableDesc, check, lib

F16, F32 = LKHIP_F16, LKHIP_F32  # KV cache types
NO_PAGE = 0xFFFFFFFF


class DeviceArray:
    """A device allocation with a numpy dtype and shape."""

    def __init__(self, shape, dtype=np.float32):
        self.shape = tuple(int(s) for s in (shape if isinstance(shape, (tuple, list)) else (shape,)))
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape, dtype=np.int64)) * self.dtype.itemsize
        p = C.c_void_p()
        check(lib().lkhip_malloc(C.byref(p), max(self.nbytes, 4)))
        self.ptr = p

    @classmethod
    def from_numpy(cls, a: np.ndarray) -> "DeviceArray":
        a = np.ascontiguousarray(a)
        d = cls(a.shape, a.dtype)
        if d.nbytes:
            check(lib().lkhip_memcpy_htod(d.ptr, a.ctypes.data, d.nbytes))
        return d

    def numpy(self) -> np.ndarray:
        out = np.empty(self.shape, dtype=self.dtype)
        check(lib().lkhip_synchronize())
        if self.nbytes:
            check(lib().lkhip_memcpy_dtoh(out.ctypes.data, self.ptr, self.nbytes))
        return out

    def upload(self, a: np.ndarray) -> None:
        a = np.ascontiguousarray(a, dtype=self.dtype)
        assert a.nbytes == self.nbytes
        check(lib().lkhip_memcpy_htod(self.ptr, a.ctypes.data, self.nbytes))

    def zero(self) -> None:
        check(lib().lkhip_memset(self.ptr, 0, self.nbytes))

    def free(self) -> None:
        if self.ptr:
            check(lib().lkhip_free(self.ptr))
            self.ptr = None

    def __del__(self):
        try:
            if self.ptr:
                lib().lkhip_free(self.ptr)
        except Exception:
            pass


class Weight:
    """A weight matrix in its GGUF type (F16, Q8_0, Q4_0, Q5_0, Q4_K, Q5_K, Q6_K), resident on device."""

    def __init__(self, ggml_type: int, rows: int, cols: int, data: np.ndarray):
        data = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        h = C.c_void_p()
        check(lib().lkhip_weight_create(ggml_type, rows, cols, data.ctypes.data, data.size, C.byref(h)))
        self._h = h
        self.ggml_type, self.rows, self.cols = ggml_type, rows, cols

    @property
    def nbytes(self) -> float:
        return float(lib().lkhip_weight_bytes(self._h))

    def close(self):
        if self._h:
            lib().lkhip_weight_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _p(d):
    return None if d is None else d.ptr


def dequant_rows(w: Weight, row0: int, n_rows: int, out: DeviceArray, stream=None) -> None:
    check(lib().lkhip_dequant_rows(w._h, row0, n_rows, out.ptr, stream))


def matvec(w: Weight, x: DeviceArray, y: DeviceArray, bias: DeviceArray | None = None, accumulate=False,
           stream=None) -> None:
    check(lib().lkhip_matvec(w._h, x.ptr, _p(bias), y.ptr, int(accumulate), stream))


def matmul(w: Weight, x: DeviceArray, n_rows: int, y: DeviceArray, bias: DeviceArray | None = None,
           accumulate=False, ldx: int | None = None, ldy: int | None = None, stream=None) -> None:
    """y[r, :rows] (+)= W x[r, :cols] (+ bias) for n_rows rows (multi-row GEMM)."""
    check(lib().lkhip_matmul(w._h, x.ptr, n_rows, ldx or w.cols, _p(bias), y.ptr, ldy or w.rows, int(accumulate),
                             stream))


def q8_0_matvec(w, x, y, bias=None, accumulate=False, stream=None) -> None:
    check(lib().lkhip_q8_0_matvec(w._h, x.ptr, _p(bias), y.ptr, int(accumulate), stream))


def q4_k_matvec(w, x, y, bias=None, accumulate=False, stream=None) -> None:
    check(lib().lkhip_q4_k_matvec(w._h, x.ptr, _p(bias), y.ptr, int(accumulate), stream))


def rmsnorm(x: DeviceArray, w: DeviceArray, n_rows: int, n: int, eps: float, y: DeviceArray, stream=None) -> None:
    check(lib().lkhip_rmsnorm(x.ptr, w.ptr, n_rows, n, eps, y.ptr, stream))


def rope_pairs(x: DeviceArray, n_rows: int, n: int, head_dim: int, pos: DeviceArray, theta: float,
               stream=None) -> None:
    check(lib().lkhip_rope_pairs(x.ptr, n_rows, n, head_dim, pos.ptr, theta, stream))


def swiglu(g: DeviceArray, u: DeviceArray, n: int, out: DeviceArray, stream=None) -> None:
    check(lib().lkhip_swiglu(g.ptr, u.ptr, n, out.ptr, stream))


def embed_gather(table: Weight, ids: DeviceArray, n_ids: int, out: DeviceArray, stream=None) -> None:
    check(lib().lkhip_embed_gather(table._h, ids.ptr, n_ids, out.ptr, stream))


def attn_decode(q: DeviceArray, k: DeviceArray, v: DeviceArray, ctx_len: DeviceArray, n_seq: int, n_heads: int,
                n_kv_heads: int, head_dim: int, max_seq: int, out: DeviceArray, stream=None) -> None:
    check(lib().lkhip_attn_decode(q.ptr, k.ptr, v.ptr, ctx_len.ptr, n_seq, n_heads, n_kv_heads, head_dim, max_seq,
                                  out.ptr, stream))


def attn_decode_noalloc(q: DeviceArray, k: DeviceArray, v: DeviceArray, ctx_len: DeviceArray, n_seq: int,
                        n_heads: int, n_kv_heads: int, head_dim: int, max_seq: int, out: DeviceArray,
                        stream=None) -> None:
    check(lib().lkhip_attn_decode_noalloc(q.ptr, k.ptr, v.ptr, ctx_len.ptr, n_seq, n_heads, n_kv_heads, head_dim,
                                          max_seq, out.ptr, stream))


def argmax(x: DeviceArray, n_rows: int, n: int, out: DeviceArray, stream=None) -> None:
    check(lib().lkhip_argmax(x.ptr, n_rows, n, out.ptr, stream))


# ------------------------------------------------------------ paged KV cache

class KvPages:
    """K and V pools of pages (lkhip_kv_pages); strides in elements, dense [layer][page][kv head][row][dim] if left out."""

    def __init__(self, k: DeviceArray, v: DeviceArray, kv_type: int, n_layers: int, n_pages: int, n_kv_heads: int,
                 page_size: int, head_dim: int, page_stride: int | None = None, head_stride: int | None = None,
                 layer_stride: int | None = None):
        head = page_size * head_dim if head_stride is None else head_stride
        page = n_kv_heads * page_size * head_dim if page_stride is None else page_stride
        layer = n_pages * n_kv_heads * page_size * head_dim if layer_stride is None else layer_stride
        self.k, self.v = k, v
        self.desc = KvPagesDesc(k.ptr, v.ptr, kv_type, head_dim, n_kv_heads, page_size, n_layers, 0, n_pages, page,
                                head, layer)
        self._ref = C.byref(self.desc)


class PageTable:
    """Page ids [n_seq][max_pages], lengths and reference counts (lkhip_page_table); the last two may be None where
    pages_fork / pages_grow / pages_trim are not used."""

    def __init__(self, table: DeviceArray, length: DeviceArray | None, refs: DeviceArray | None, n_seq: int,
                 max_pages: int):
        self.table, self.length, self.refs = table, length, refs
        self.desc = PageTableDesc(table.ptr, _p(length), _p(refs), n_seq, max_pages)
        self._ref = C.byref(self.desc)


def pages_fork(pages: KvPages, table: PageTable, src: DeviceArray, dst: DeviceArray, n: int, ok: DeviceArray,
               stream=None) -> None:
    check(lib().lkhip_pages_fork(pages._ref, table._ref, src.ptr, dst.ptr, n, ok.ptr, stream))


def pages_grow(pages: KvPages, table: PageTable, slots: DeviceArray, add: DeviceArray, n: int, ok: DeviceArray,
               copied: DeviceArray, stream=None) -> None:
    check(lib().lkhip_pages_grow(pages._ref, table._ref, slots.ptr, add.ptr, n, ok.ptr, copied.ptr, stream))


def pages_trim(pages: KvPages, table: PageTable, slots: DeviceArray, keep: DeviceArray, n: int, stream=None) -> None:
    check(lib().lkhip_pages_trim(pages._ref, table._ref, slots.ptr, keep.ptr, n, stream))


def pages_write(pages: KvPages, table: PageTable, layer: int, k: DeviceArray, v: DeviceArray, slots: DeviceArray,
                pos: DeviceArray, n_rows: int, ld: int | None = None, stream=None) -> None:
    d = pages.desc
    check(lib().lkhip_pages_write(pages._ref, table._ref, layer, k.ptr, v.ptr, ld or d.n_kv_heads * d.head_dim,
                                  slots.ptr, pos.ptr, n_rows, stream))


def pages_compact(pages: KvPages, table: PageTable, slots: DeviceArray, start: DeviceArray, path: DeviceArray,
                  n_path: DeviceArray, n: int, ld_path: int, stream=None) -> None:
    check(lib().lkhip_pages_compact(pages._ref, table._ref, slots.ptr, start.ptr, path.ptr, ld_path, n_path.ptr, n,
                                    stream))


def tree_attn_workspace(pages: KvPages, table: PageTable, n: int, max_draft: int, n_heads: int) -> int:
    b = C.c_size_t()
    check(lib().lkhip_tree_attn_workspace(pages._ref, table._ref, n, max_draft, n_heads, C.byref(b)))
    return b.value


def tree_attn(pages: KvPages, table: PageTable, layer: int, q: DeviceArray, ctx_len: DeviceArray,
              n_draft: DeviceArray | None, mask: DeviceArray | None, n: int, max_draft: int, n_heads: int,
              ws: DeviceArray | None, ws_bytes: int, out: DeviceArray, slots: DeviceArray | None = None,
              stream=None) -> None:
    """Drafted tokens over their contexts: out[i, t] for t < n_draft[i], seeing what mask's bits allow of the draft."""
    check(lib().lkhip_tree_attn(pages._ref, table._ref, layer, q.ptr, _p(slots), ctx_len.ptr, _p(n_draft), _p(mask), n,
                                max_draft, n_heads, _p(ws), ws_bytes, out.ptr, stream))


def page_bounds(pages: KvPages, table: PageTable, layer: int, start: DeviceArray, end: DeviceArray, n: int,
                bounds: DeviceArray, slots: DeviceArray | None = None, stream=None) -> None:
    check(lib().lkhip_page_bounds(pages._ref, table._ref, layer, _p(slots), start.ptr, end.ptr, n, bounds.ptr, stream))


def sparse_attn_workspace(pages: KvPages, table: PageTable, n: int, n_heads: int, n_take: int) -> int:
    b = C.c_size_t()
    check(lib().lkhip_sparse_attn_workspace(pages._ref, table._ref, n, n_heads, n_take, C.byref(b)))
    return b.value


def sparse_attn(pages: KvPages, table: PageTable, layer: int, q: DeviceArray, ctx_len: DeviceArray,
                bounds: DeviceArray, n: int, n_heads: int, n_take: int, n_first: int, n_last: int, taken: DeviceArray,
                ws: DeviceArray, ws_bytes: int, out: DeviceArray, slots: DeviceArray | None = None,
                stream=None) -> None:
    """One token per sequence over n_take pages of its context; taken gets their numbers."""
    check(lib().lkhip_sparse_attn(pages._ref, table._ref, layer, q.ptr, _p(slots), ctx_len.ptr, bounds.ptr, n, n_heads,
                                  n_take, n_first, n_last, taken.ptr, _p(ws), ws_bytes, out.ptr, stream))


def memset(d: DeviceArray, value: int) -> None:
    check(lib().lkhip_memset(d.ptr, value, d.nbytes))


def memcpy_dtod(dst: DeviceArray, src: DeviceArray) -> None:
    check(lib().lkhip_memcpy_dtod(dst.ptr, src.ptr, min(dst.nbytes, src.nbytes)))


def synchronize() -> None:
    check(lib().lkhip_synchronize())


def device_count() -> int:
    return int(lib().lkhip_device_count())


class Stream:
    def __init__(self):
        p = C.c_void_p()
        check(lib().lkhip_stream_create(C.byref(p)))
        self.ptr = p

    def synchronize(self):
        check(lib().lkhip_stream_synchronize(self.ptr))

    def close(self):
        if self.ptr:
            check(lib().lkhip_stream_destroy(self.ptr))
            self.ptr = None


class Event:
    def __init__(self):
        p = C.c_void_p()
        check(lib().lkhip_event_create(C.byref(p)))
        self.ptr = p

    def record(self, stream=None):
        check(lib().lkhip_event_record(self.ptr, None if stream is None else stream.ptr))

    def elapsed_ms(self, end: "Event") -> float:
        ms = C.c_float()
        check(lib().lkhip_event_elapsed_ms(self.ptr, end.ptr, C.byref(ms)))
        return float(ms.value)
