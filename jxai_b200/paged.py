"""The paged 8-bit KV cache (include/jx_attn.h, jx_pkv).

Rows of K and V are held as 8-bit codes with one power-of-two scale for each
block of 16 rows and kv head, in pages of 32 rows that sequences take from a
pool, share after a fork and give back.  ``attn_step``, ``attn_prefill``,
``StepPlan`` and ``KVCacheSlot`` take a ``PagedKVCache`` where they take a
``KVCache``.
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from ._lib import JX_BF16, JX_E4M3, JX_F32, JX_I8, JxError, PkvDesc, check, load
from .attention import _i32_array, _stream_ptr

PAGED_DTYPES = {"int8": JX_I8, "i8": JX_I8, "e4m3": JX_E4M3, "fp8": JX_E4M3,
                JX_I8: JX_I8, JX_E4M3: JX_E4M3}


class PagedKVCache:
    """A pool of pages and the sequences that hold them.

    ``n_pages`` defaults to as many as all sequences need at ``capacity`` rows;
    with fewer, a call that finds none free (or no memory for a prompt's
    workspaces) raises ``JxError`` (code -3) and changes nothing.  A sequence holds the rows ``[0, seq_pos)``: a step or prompt
    writes from a position up to ``seq_pos`` on, and the sequence then ends at the
    row after the last one written.
    """

    PAGE = 32    # rows of a page
    BLOCK = 16   # rows that share a scale
    entry_prefix = "jx_pkv_attn_"

    def __init__(self, n_seqs: int, n_layers: int, capacity: int, n_kv_heads: int, head_dim: int,
                 n_pages: int | None = None, dtype="int8", device: int = 0):
        if dtype not in PAGED_DTYPES:
            raise JxError(-1, f"dtype {dtype!r}: a paged cache holds int8 or e4m3")
        self.lib = load()
        self.dtype = PAGED_DTYPES[dtype]
        self.n_seqs, self.n_layers, self.capacity = n_seqs, n_layers, capacity
        self.n_kv_heads, self.head_dim, self.device = n_kv_heads, head_dim, device
        if n_pages is None:
            n_pages = n_seqs * (-(-capacity // self.PAGE))
        self.n_pages = n_pages
        d = PkvDesc(n_seqs, n_layers, capacity, n_kv_heads, head_dim, n_pages, self.dtype, device)
        h = C.c_void_p()
        check(self.lib.jx_pkv_create(C.byref(d), C.byref(h)))
        self.handle = h

    # lifetime ---------------------------------------------------------------
    def close(self) -> None:
        if getattr(self, "handle", None):
            self.lib.jx_pkv_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def nbytes(self) -> int:
        """Bytes of the page pool.  The handle holds more: cosines and sines of every position
        (capacity * head_dim * 4 bytes per RoPE setting) and, from the first tensor-core prompt on,
        its fp16 rows (up to 1 GiB, or one sequence and layer where that is more)."""
        record = 2 * self.PAGE * self.head_dim + 16
        return self.n_pages * self.n_layers * self.n_kv_heads * record

    # rows and pages -----------------------------------------------------------
    def _count(self, call, *args) -> int:
        v = C.c_uint32()
        check(call(self.handle, *args, C.byref(v)))
        return v.value

    def seq_pos(self, seq: int) -> int:
        return self._count(self.lib.jx_pkv_get_seq_pos, seq)

    def set_seq_pos(self, seq: int, pos: int) -> None:
        check(self.lib.jx_pkv_set_seq_pos(self.handle, seq, pos))

    @property
    def free_pages(self) -> int:
        return self._count(self.lib.jx_pkv_free_pages)

    def held_pages(self, seq: int) -> int:
        """Pages the sequence holds, those it shares with forks included."""
        return self._count(self.lib.jx_pkv_held_pages, seq)

    def clear(self, seq: int, stream=None) -> None:
        check(self.lib.jx_pkv_clear(self.handle, seq))

    def rollback(self, seq: int, new_seq_pos: int) -> None:
        check(self.lib.jx_pkv_rollback(self.handle, seq, new_seq_pos))

    def fork(self, src: int, dst: int, n_rows: int | None = None, stream=None) -> None:
        """dst becomes the first n_rows rows of src (default: all), on the same pages."""
        n = self.seq_pos(src) if n_rows is None else n_rows
        check(self.lib.jx_pkv_fork(self.handle, src, dst, n, _stream_ptr(stream, self.device)))

    def copy(self, src: int, dst: int, stream=None) -> None:
        """dst becomes a copy of src on pages of its own."""
        check(self.lib.jx_pkv_copy(self.handle, src, dst, _stream_ptr(stream, self.device)))

    def keep(self, seq: int, rows: Sequence[int], stream=None) -> None:
        """Cuts the sequence down to the given rows (ascending), in every layer.  Their keys stay as
        they were rotated; the next row stands at position len(rows)."""
        arr = _i32_array(rows)
        check(self.lib.jx_pkv_keep(self.handle, seq, arr, len(arr), _stream_ptr(stream, self.device)))

    def compact(self, seq: int, keep_recent: int = 128, stream=None) -> None:
        check(self.lib.jx_pkv_compact(self.handle, seq, keep_recent, _stream_ptr(stream, self.device)))

    # contents ---------------------------------------------------------------
    def _tensor(self, t, name: str, shape, dtypes, stream):
        import torch
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise JxError(-1, f"{name} must be a CUDA tensor")
        if tuple(t.shape) != tuple(shape) or t.dtype not in dtypes:
            raise JxError(-1, f"{name} must be {tuple(shape)} of {dtypes[0]}, got {tuple(t.shape)} "
                              f"of {t.dtype}")
        if stream is not None and not t.is_contiguous():
            # the copy would be made on torch's current stream
            raise JxError(-1, f"{name} must be contiguous where a stream is given")
        return t.contiguous()

    def load(self, seq: int, row0: int, k_codes, k_scales, v_codes, v_scales, stream=None) -> None:
        """Rows [row0, row0 + n) from codes [n_layers, n, n_kv_heads, head_dim] (int8 or e4m3, or
        their bytes as uint8) and scales [n_layers, ceil(n / 16), n_kv_heads] (float32); row0 a
        multiple of 16.  Scales are taken down to powers of two."""
        import torch
        n = k_codes.shape[1] if getattr(k_codes, "ndim", 0) == 4 else -1
        kinds = (torch.int8 if self.dtype == JX_I8 else torch.float8_e4m3fn, torch.uint8)
        codes = (self.n_layers, n, self.n_kv_heads, self.head_dim)
        scales = (self.n_layers, -(-n // self.BLOCK), self.n_kv_heads)
        keep = [self._tensor(k_codes, "k_codes", codes, kinds, stream),
                self._tensor(k_scales, "k_scales", scales, (torch.float32,), stream),
                self._tensor(v_codes, "v_codes", codes, kinds, stream),
                self._tensor(v_scales, "v_scales", scales, (torch.float32,), stream)]
        check(self.lib.jx_pkv_load_rows(self.handle, seq, row0, n, *(t.data_ptr() for t in keep),
                                        _stream_ptr(stream, self.device)))

    def read(self, seqs: Sequence[int], row0: Sequence[int], n_rows: int, dtype=None, out=None,
             stream=None):
        """Values of rows [row0[i], row0[i] + n_rows) of each listed sequence: a tensor [len(seqs),
        n_layers, 2, n_rows, n_kv_heads, head_dim] (K, then V) of bfloat16 (default) or float32;
        both hold every value exactly.  With `stream`, `out` has to be given."""
        import torch
        ids, first = _i32_array(seqs), _i32_array(row0)
        if len(ids) != len(first):
            raise JxError(-1, "read: one first row per sequence")
        shape = (len(ids), self.n_layers, 2, n_rows, self.n_kv_heads, self.head_dim)
        if dtype not in (None, torch.bfloat16, torch.float32):
            raise JxError(-1, "rows are read as bfloat16 or float32")
        if out is None:
            if stream is not None:
                raise JxError(-1, "read: give out where a stream is given")
            out = torch.empty(shape, dtype=dtype or torch.bfloat16,
                              device=torch.device("cuda", self.device))
        elif (not out.is_cuda or tuple(out.shape) != shape or not out.is_contiguous()
                or out.dtype not in ((torch.bfloat16, torch.float32) if dtype is None else (dtype,))):
            raise JxError(-1, f"out must be a contiguous CUDA tensor {shape} of bfloat16 or float32")
        kind = JX_F32 if out.dtype == torch.float32 else JX_BF16
        check(self.lib.jx_pkv_read_rows(self.handle, ids, first, len(ids), n_rows, kind,
                                        out.data_ptr(), _stream_ptr(stream, self.device)))
        return out

    # plumbing -----------------------------------------------------------------
    def set_option(self, key: str, value: int) -> None:
        check(self.lib.jx_pkv_set_option(self.handle, key.encode(), value))

    def check_device_error(self, stream=None) -> int:
        code = C.c_int()
        rc = self.lib.jx_pkv_check_device_error(self.handle, C.byref(code), _stream_ptr(stream, self.device))
        if rc not in (0, -6):
            check(rc)
        return code.value

    def last_launch_count(self) -> int:
        n = C.c_int()
        check(self.lib.jx_pkv_last_launch_count(self.handle, C.byref(n)))
        return n.value
