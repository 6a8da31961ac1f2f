"""A paged KV cache over torch tensors: the operators ``fl_kv_append_device``,
``fl_kv_gather_device`` and ``fl_attn_paged_device`` of the C ABI.

    cache = PagedKvCache.empty(n_pages, 16, n_kv_heads, head_dim, torch.int8)   # or torch.float16, torch.float8_e4m3fn
    batch = PagedBatch(page_table, seq_len, row_start, max_rows=5)
    cache.append(batch, k, v)                      # K, V of the step's new rows
    out = cache.attention(batch, q, scale=1 / math.sqrt(head_dim), window=4096, softcap=0.0)
    k, v = cache.gather(batch, n_rows, torch.float16)

The formats, the layout of the pages, the meaning of a batch and what a row
attends to are stated in ``include/foundry_cuda.h``.  The reference's
``KvCache`` (src/DotNetFoundryLLM.Core KvCache.cs:59-173) is one F32 array per
sequence; pages, 8-bit formats and several new rows a step have no counterpart
there.

All calls are enqueued on the current stream of the tensors' device, allocate
only their outputs and a workspace (from torch's allocator, so captured graphs
hold their own), and, but for ``synchronize``, do not synchronize.  Argument errors raise
``ArgumentError`` / ``NotSupportedError`` before anything is enqueued.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _native as N
from .runtime import ArgumentError, NotSupportedError, check

KV_DTYPES = {torch.float16: N.FL_KV_F16, torch.int8: N.FL_KV_Q8, torch.float8_e4m3fn: N.FL_KV_F8}
ROW_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}  # GGML type ids


def _cuda_tensor(name: str, t: torch.Tensor, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ArgumentError(f"{name} must be a CUDA tensor")
    if t.get_device() != device.index:
        raise ArgumentError(f"{name} is on {t.device}, the others on {device}")


def _int32(name: str, t: torch.Tensor, shape: tuple, device: torch.device) -> None:
    _cuda_tensor(name, t, device)
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ArgumentError(f"{name} must be a contiguous int32 tensor of shape {shape}, not {t.dtype} {tuple(t.shape)}")


def _row_type(name: str, dtype: torch.dtype) -> int:
    rt = ROW_TYPES.get(dtype)
    if rt is None:
        raise NotSupportedError(f"{name}: {dtype} (float32, float16 and bfloat16 are built)")
    return rt


def _enqueue(device: torch.device, what: str, fn, *args) -> None:
    """fn(*args, stream) on the device's current stream, with that device current for the call."""
    i = device.index
    stream = torch._C._cuda_getCurrentRawStream(i)
    if torch._C._cuda_getDevice() == i:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(i):
            rc = fn(*args, stream)
    if rc:
        check(rc, what)


def _raw(name: str, *types):
    """The library's entry `name` with descriptors passed as packed bytes, which are quicker to make than ctypes structures."""
    fn = N.cuda()[name]
    fn.restype, fn.argtypes = C.c_int, types
    return fn


# fl_paged_attn_desc, as _native.FlPagedAttnDesc
_ATTN = struct.Struct("=5i2fiQqQqQQQ")
assert _ATTN.size == C.sizeof(N.FlPagedAttnDesc)


class PagedBatch:
    """The new rows of a step (``fl_paged_batch``): page_table [n_seqs, cols],
    seq_len [n_seqs] (new rows included) and row_start [n_seqs + 1], int32
    CUDA tensors that are read on the device at each call.  ``max_rows``: the
    most rows a sequence has, if known on the host; it affects speed only."""

    def __init__(self, page_table: torch.Tensor, seq_len: torch.Tensor, row_start: torch.Tensor, max_rows: int = 0):
        if not isinstance(page_table, torch.Tensor) or not page_table.is_cuda:
            raise ArgumentError("page_table must be a CUDA tensor")
        if page_table.dim() != 2:
            raise ArgumentError(f"page_table must be [n_seqs, pages], not {tuple(page_table.shape)}")
        self.device = page_table.device
        n = page_table.shape[0]
        _int32("page_table", page_table, tuple(page_table.shape), self.device)
        _int32("seq_len", seq_len, (n,), self.device)
        _int32("row_start", row_start, (n + 1,), self.device)
        if not 0 <= max_rows < 2 ** 31:
            raise ArgumentError(f"max_rows {max_rows} is not in [0, 2^31)")
        self.page_table, self.seq_len, self.row_start = page_table, seq_len, row_start
        self.desc = N.FlPagedBatch(C.sizeof(N.FlPagedBatch), n, page_table.shape[1], max_rows, page_table.data_ptr(),
                                   seq_len.data_ptr(), row_start.data_ptr())
        self._ref = C.byref(self.desc)
        self._at = C.addressof(self.desc)
        self._sizes = (n, page_table.shape[1], max_rows)


class PagedKvCache:
    """Pages of K and V: k, v [n_pages, n_kv_heads, page_size, head_dim] of
    torch.float16, torch.int8 or torch.float8_e4m3fn; for the 8-bit types
    k_scale, v_scale [n_pages, n_kv_heads, page_size] float32.  The tensors
    stay the caller's."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None):
        if not isinstance(k, torch.Tensor) or not k.is_cuda:
            raise ArgumentError("k must be a CUDA tensor")
        self.device = k.device
        _cuda_tensor("v", v, self.device)
        if k.dtype not in KV_DTYPES:
            raise NotSupportedError(f"cache of {k.dtype} (float16, int8 and float8_e4m3fn are built)")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or not k.is_contiguous() or not v.is_contiguous():
            raise ArgumentError("k and v must be contiguous [n_pages, n_kv_heads, page_size, head_dim] tensors of one type")
        n_pages, n_kv, page, hd = k.shape
        if k.dtype == torch.float16:
            if k_scale is not None or v_scale is not None:
                raise ArgumentError("a float16 cache has no scales")
        else:
            for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
                if t is None:
                    raise ArgumentError(f"a cache of {k.dtype} needs {name}")
                _cuda_tensor(name, t, self.device)
                if t.dtype != torch.float32 or t.shape != k.shape[:3] or not t.is_contiguous():
                    raise ArgumentError(f"{name} must be a contiguous float32 tensor of shape {tuple(k.shape[:3])}")
        if hd not in (64, 128, 256):
            raise NotSupportedError(f"head_dim {hd} (64, 128 and 256 are built)")
        if page < 16 or page > 1024 or page & (page - 1):
            raise ArgumentError(f"page_size {page} is not a power of two in [16, 1024]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_kv_heads, self.page_size, self.head_dim = n_kv, page, hd
        self.desc = N.FlPagedKv(C.sizeof(N.FlPagedKv), KV_DTYPES[k.dtype], n_pages, page, n_kv, hd, k.data_ptr(),
                                v.data_ptr(), k_scale.data_ptr() if k_scale is not None else None,
                                v_scale.data_ptr() if v_scale is not None else None)
        self._ref = C.byref(self.desc)
        self._at = C.addressof(self.desc)
        self.lib = N.cuda()
        self._append = _raw("fl_kv_append_device", *[C.c_void_p] * 2, C.c_int32, C.c_int32, C.c_void_p, C.c_int64, C.c_void_p,
                            C.c_int64, C.c_void_p)
        self._gather = _raw("fl_kv_gather_device", *[C.c_void_p] * 2, C.c_int32, C.c_int32, C.c_void_p, C.c_int64, C.c_void_p,
                            C.c_int64, C.c_void_p)
        self._attend = _raw("fl_attn_paged_device", C.c_void_p, C.c_void_p, C.c_char_p, C.c_void_p)
        self._space: dict[tuple, int] = {}  # workspace bytes by sizes

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype,
              device: torch.device | str = "cuda") -> "PagedKvCache":
        """A cache of its own, zeroed."""
        if dtype not in KV_DTYPES:
            raise NotSupportedError(f"cache of {dtype} (float16, int8 and float8_e4m3fn are built)")
        shape = (n_pages, n_kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype == torch.float16:
            return cls(k, v)
        return cls(k, v, *(torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))

    def _rows(self, name: str, t: torch.Tensor, heads: int) -> int:
        """Checks a packed row tensor [rows, heads, head_dim]; its row stride in elements."""
        _cuda_tensor(name, t, self.device)
        shape = t.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim:
            raise ArgumentError(f"{name} must be [rows, {heads}, {self.head_dim}], not {tuple(t.shape)}")
        s = t.stride()
        if s[2] != 1 or (s[1] != self.head_dim and heads > 1):
            raise ArgumentError(f"{name}: heads and elements of a row must be dense (strides {s})")
        return s[0]

    def _batch(self, batch: PagedBatch) -> None:
        if batch.device is not self.device and batch.device != self.device:
            raise ArgumentError(f"the batch is on {batch.device}, the cache on {self.device}")

    def append(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor) -> None:
        """``fl_kv_append_device``: writes the batch's new rows (k, v: [rows,
        n_kv_heads, head_dim], of one type; rows may be strided)."""
        self._batch(batch)
        ks, vs = self._rows("k", k, self.n_kv_heads), self._rows("v", v, self.n_kv_heads)
        if v.dtype != k.dtype or v.shape[0] != k.shape[0]:
            raise ArgumentError("k and v must have the same type and number of rows")
        _enqueue(self.device, "fl_kv_append_device", self._append, self._at, batch._at, _row_type("k", k.dtype), k.shape[0],
                 k.data_ptr(), ks, v.data_ptr(), vs)

    def gather(self, batch: PagedBatch, n_rows: int, dtype: torch.dtype = torch.float32,
               out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """``fl_kv_gather_device``: the values of the batch's rows as two
        [n_rows, n_kv_heads, head_dim] tensors of ``dtype`` (or into ``out``).
        Rows behind the last sequence are left as they were (new tensors:
        zero only where a sequence's row is unmapped, else undefined)."""
        self._batch(batch)
        if out is None:
            if n_rows < 0:
                raise ArgumentError("n_rows must be >= 0")
            _row_type("dtype", dtype)
            shape = (n_rows, self.n_kv_heads, self.head_dim)
            out = (torch.empty(shape, dtype=dtype, device=self.device), torch.empty(shape, dtype=dtype, device=self.device))
        k, v = out
        ks, vs = self._rows("k", k, self.n_kv_heads), self._rows("v", v, self.n_kv_heads)
        if v.dtype != k.dtype or k.shape[0] != n_rows or v.shape[0] != n_rows:
            raise ArgumentError(f"out must be two tensors of one type with {n_rows} rows")
        _enqueue(self.device, "fl_kv_gather_device", self._gather, self._at, batch._at, _row_type("out", k.dtype), n_rows,
                 k.data_ptr(), ks, v.data_ptr(), vs)
        return out

    def attention(self, batch: PagedBatch, q: torch.Tensor, scale: float, window: int = 0, softcap: float = 0.0,
                  out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
        """``fl_attn_paged_device``: the new rows' attention over the cache (q:
        [rows, n_heads, head_dim]; their own K and V already appended).  With
        ``lse`` ([rows, n_heads] float32, contiguous) the logarithms of the
        softmax sums are written too.  Rows behind the last sequence are left
        as they were (undefined in a new tensor)."""
        self._batch(batch)
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ArgumentError("q must be a [rows, n_heads, head_dim] tensor")
        n_rows, n_heads = q.shape[0], q.shape[1]
        qs = self._rows("q", q, n_heads)
        rt = _row_type("q", q.dtype)
        if out is None:
            out = torch.empty(n_rows, n_heads, self.head_dim, dtype=q.dtype, device=self.device)
            os = n_heads * self.head_dim
        else:
            os = self._rows("out", out, n_heads)
            if out.shape[0] != n_rows or out.dtype != q.dtype:
                raise ArgumentError("out must have q's shape and type")
        if lse is not None:
            _cuda_tensor("lse", lse, self.device)
            if lse.dtype != torch.float32 or tuple(lse.shape) != (n_rows, n_heads) or not lse.is_contiguous():
                raise ArgumentError(f"lse must be a contiguous float32 tensor of shape {(n_rows, n_heads)}")
        key = (n_rows, n_heads, batch._sizes)
        need = self._space.get(key)
        if need is None:
            got = C.c_uint64()
            check(self.lib.fl_attn_paged_workspace(self._ref, batch._ref, n_rows, n_heads, C.byref(got)), "fl_attn_paged_workspace")
            if len(self._space) >= 4096:
                self._space.clear()
            need = self._space[key] = got.value
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        try:
            d = _ATTN.pack(_ATTN.size, rt, n_rows, n_heads, window, scale, softcap, 0, q.data_ptr(), qs, out.data_ptr(), os,
                           lse.data_ptr() if lse is not None else 0, ws.data_ptr(), need)
        except (struct.error, OverflowError) as e:
            raise ArgumentError(f"window {window}, scale {scale} or softcap {softcap} is no number of 32 bits: {e}") from None
        _enqueue(self.device, "fl_attn_paged_device", self._attend, self._at, batch._at, d)
        return out

    def synchronize(self) -> None:
        """``fl_attn_paged_status``: waits for the current stream of the cache's device and raises
        ``DeviceTimeoutError`` if a bounded wait of an attention call on that device ran out since
        the last query; the rows that it concerns are NaN."""
        expired = C.c_uint32()
        with torch.cuda.device(self.device):
            check(self.lib.fl_attn_paged_status(C.byref(expired), torch.cuda.current_stream().cuda_stream), "fl_attn_paged_status")
