"""The paged key/value store: pages shared by many sequences, written, read
back and attended over (the ``kivi_pages_*`` entries of include/kivi_gpu.h; no
counterpart in the reference, whose caches are one contiguous batch each).

Everything is on the device and stream-ordered.  Arguments are CUDA tensors, or
device pointers (ints) with the sizes and types that a tensor would carry::

    config = PagesConfig(bits=8, num_pages=4096, page_size=32, num_kv_heads=8, head_dim=128)
    data, params = config.sizes()                     # bytes and floats of each side
    pages = KvPages(config, keys, values, key_params, value_params)
    batch = PagesBatch(block_table, cu_tokens, kv_lens, total_tokens, max_tokens)
    pages.write_dev(batch, new_keys, new_values)      # [total_tokens, num_kv_heads, head_dim]
    pages.attention_dev(batch, query, num_q_heads, scale, out)
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
_TENSOR_TYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
_types = {}  # the same by dtype object, filled as they are met


class _PagesConfig(C.Structure):
    _fields_ = [("bits", C.c_uint32), ("dtype", C.c_int32)] + [(n, C.c_uint64) for n in (
        "num_pages", "page_size", "num_kv_heads", "head_dim")]


class _PagesBatch(C.Structure):
    _fields_ = [("block_table", C.c_void_p), ("table_stride", C.c_uint64),
                ("table_width", C.c_uint64), ("cu_tokens", C.c_void_p), ("kv_lens", C.c_void_p),
                ("batch", C.c_uint64), ("total_tokens", C.c_uint64), ("max_tokens", C.c_uint64)]


def signatures(P, sz, i32, f32, e):
    """ctypes signatures of the kivi_pages_* entries."""
    cfg, bat, u64p = C.POINTER(_PagesConfig), C.POINTER(_PagesBatch), C.POINTER(C.c_uint64)
    return {
        "kivi_pages_sizes": ([cfg, u64p, u64p, e], i32),
        "kivi_pages_new": ([cfg, P, P, P, P, i32, C.POINTER(P), e], i32),
        "kivi_pages_free": ([P], None),
        "kivi_pages_write_dev": ([P, bat, i32, P, P, sz, sz, P, e], i32),
        "kivi_pages_read_dev": ([P, bat, i32, P, P, sz, sz, P, e], i32),
        "kivi_pages_attention_dev": ([P, bat, i32, P, sz, sz, sz, f32, sz, sz, P, sz, sz, P, P, e],
                                     i32),
        "kivi_pages_workspace_size": ([i32, u64p, e], i32),
        "kivi_pages_set_workspace": ([P, P, sz, e], i32),
        "kivi_pages_status": ([P, e], i32),
    }


from . import KiviError, _check, _Err, _ptr, _stream, lib  # noqa: E402

_INVALID = 101


def _bad(message):
    return KiviError(_INVALID, message=message)


def _code(dtype):
    if dtype in DTYPES:
        return DTYPES[dtype]
    raise _bad(f"unknown element type {dtype!r}: use one of {sorted(DTYPES)}")


def _place(device):
    return "the CPU" if device < 0 else f"device {device}"


def _rows(x, dtype, strides, heads, dim, total, what, device):
    """(pointer, type code, token stride, head stride) of dense rows
    [total, heads, dim]: a tensor's own, or a pointer's as given (contiguous
    where no strides are)."""
    if x is None or isinstance(x, int):
        if dtype is None:
            raise _bad(f"{what}: a pointer needs dtype=")
        token, head = strides if strides is not None else (heads * dim, dim)
        return x, _code(dtype), token, head
    if x.get_device() != device:
        raise _bad(f"{what}: on {_place(x.get_device())}, the pages are on {_place(device)}")
    if x.shape != (total, heads, dim):
        raise _bad(f"{what}: expected shape {(total, heads, dim)}, got {tuple(x.shape)}")
    code = _types.get(x.dtype)
    if code is None:
        code = _TENSOR_TYPES.get(str(x.dtype))
        if code is None:
            raise _bad(f"{what}: unsupported element type {x.dtype}")
        _types[x.dtype] = code
    token, head, inner = x.stride()
    if inner != 1 and total:
        raise _bad(f"{what}: the elements of a row must be contiguous, their stride is {inner}")
    # the stride of a dimension of one says nothing
    return x.data_ptr(), code, token if total > 1 else heads * dim, head if heads > 1 and total else dim


def pages_workspace_size(device=0):
    """Bytes of an attention workspace on `device` (KvPages.set_workspace)."""
    size, err = C.c_uint64(), _Err()
    _check(lib().kivi_pages_workspace_size(int(device), C.byref(size), C.byref(err)), err)
    return int(size.value)


@dataclass(frozen=True)
class PagesConfig:
    """Geometry of a paged store: ``bits`` 16 (elements of ``dtype``, "bf16" or
    "f16") or 8 / 4 (codes with one (scale, zero) per token and head)."""

    bits: int = 16
    dtype: str = "bf16"
    num_pages: int = 1
    page_size: int = 64
    num_kv_heads: int = 1
    head_dim: int = 128

    def _c(self):
        code = _code(self.dtype) if self.bits == 16 else 0
        return _PagesConfig(self.bits, code, self.num_pages, self.page_size, self.num_kv_heads,
                            self.head_dim)

    def sizes(self):
        """(bytes of one side's data, floats of one side's params)."""
        data, params, err = C.c_uint64(), C.c_uint64(), _Err()
        c = self._c()
        _check(lib().kivi_pages_sizes(C.byref(c), C.byref(data), C.byref(params), C.byref(err)), err)
        return int(data.value), int(params.value)


class PagesBatch:
    """One step's sequences, shared by every layer's calls: ``block_table``
    [batch, width] int32, ``cu_tokens`` [batch + 1] int32 offsets of the newest
    tokens' rows, ``kv_lens`` [batch] int32 tokens including them, all on the
    device; ``total_tokens`` = cu_tokens[batch], ``max_tokens`` >= the most newest
    tokens of one sequence.  Keeps references to its tensors.  With pointers,
    pass batch=, table_width= (and table_stride=)."""

    def __init__(self, block_table, cu_tokens, kv_lens, total_tokens, max_tokens, batch=None,
                 table_width=None, table_stride=None):
        self.tensors = (block_table, cu_tokens, kv_lens)
        for name, x in zip(("block_table", "cu_tokens", "kv_lens"), self.tensors):
            if not isinstance(x, int) and str(x.dtype) != "torch.int32":
                raise _bad(f"{name} must be int32, not {x.dtype}")
        if not isinstance(kv_lens, int):
            batch = kv_lens.shape[0] if batch is None else batch
            if kv_lens.dim() != 1 or kv_lens.shape[0] < batch or not kv_lens.is_contiguous():
                raise _bad("kv_lens must be contiguous [batch]")
        if not isinstance(cu_tokens, int) and batch is not None and (
                cu_tokens.dim() != 1 or cu_tokens.shape[0] < batch + 1
                or not cu_tokens.is_contiguous()):
            raise _bad("cu_tokens must be contiguous [batch + 1]")
        if not isinstance(block_table, int):
            if block_table.dim() != 2 or (block_table.shape[1] > 1 and block_table.stride(1) != 1) or (
                    batch is not None and block_table.shape[0] < batch):
                raise _bad("block_table must be [batch, width] with contiguous rows")
            table_width = block_table.shape[1] if table_width is None else table_width
            if table_width > block_table.shape[1]:
                raise _bad("table_width is more than a row of block_table holds")
            table_stride = block_table.stride(0) if table_stride is None else table_stride
        if batch is None or table_width is None:
            raise _bad("pointers need batch= and table_width=")
        if min(batch, table_width, total_tokens, max_tokens) < 0:
            raise _bad("negative size")
        devices = {x.get_device() for x in self.tensors if not isinstance(x, int)}
        if len(devices) > 1:
            raise _bad("block_table, cu_tokens and kv_lens lie on different devices")
        self.device = devices.pop() if devices else None  # None: pointers, the caller's to vouch for
        self.total_tokens = int(total_tokens)
        self._c = _PagesBatch(_ptr(block_table),
                              table_width if table_stride is None else table_stride, table_width,
                              _ptr(cu_tokens), _ptr(kv_lens), batch, total_tokens, max_tokens)
        self._ref = C.byref(self._c)


class KvPages:
    """A paged store over the caller's memory: ``d_keys`` / ``d_values`` hold
    ``config.sizes()[0]`` bytes each, the params (codes only) ``[1]`` floats."""

    def __init__(self, config, d_keys, d_values, d_key_params=None, d_value_params=None, device=None):
        self._h = None
        c, err, h = config._c(), _Err(), C.c_void_p()
        self._tensors = (d_keys, d_values, d_key_params, d_value_params)
        data, params = config.sizes()
        for x, size, unit in zip(self._tensors, (data, data, params, params), (1, 1, 4, 4)):
            if x is None or isinstance(x, int):
                continue
            if not x.is_cuda or not x.is_contiguous():
                raise _bad("page memory must be contiguous device memory")
            if x.numel() * x.element_size() < size * unit:
                raise _bad(f"page memory of {x.numel() * x.element_size()} bytes, need {size * unit}")
            if device is None:
                device = x.device.index
            if x.device.index != device:
                raise _bad(f"page memory on {_place(x.device.index)}, not on {_place(device)}")
        self.device = 0 if device is None else int(device)
        _check(lib().kivi_pages_new(C.byref(c), _ptr(d_keys), _ptr(d_values), _ptr(d_key_params),
                                    _ptr(d_value_params), self.device, C.byref(h), C.byref(err)), err)
        self._h = h.value
        self.config = config
        self._heads, self._dim = config.num_kv_heads, config.head_dim
        self._write, self._read = lib().kivi_pages_write_dev, lib().kivi_pages_read_dev
        self._attention = lib().kivi_pages_attention_dev

    def close(self):
        if getattr(self, "_h", None):
            lib().kivi_pages_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _batch_here(self, batch):
        if batch.device is not None and batch.device != self.device:
            raise _bad(f"the batch is on {_place(batch.device)}, the pages are on {_place(self.device)}")

    def _sides(self, batch, d_keys, d_values, dtype, strides):
        self._batch_here(batch)
        total, device = batch.total_tokens, self.device
        k, code, token, head = _rows(d_keys, dtype, strides, self._heads, self._dim, total, "keys", device)
        v, *other = _rows(d_values, dtype, strides, self._heads, self._dim, total, "values", device)
        if other != [code, token, head]:
            raise _bad("keys and values must have the same type and strides")
        return k, v, code, token, head

    def write_dev(self, batch, d_keys, d_values, dtype=None, strides=None, stream=None):
        """Writes the batch's newest tokens, [total_tokens, num_kv_heads,
        head_dim] in f32, bf16 or f16, into their pages."""
        k, v, code, token, head = self._sides(batch, d_keys, d_values, dtype, strides)
        err = _Err()
        rc = self._write(self._h, batch._ref, code, k, v, token, head, _stream(stream), C.byref(err))
        if rc:
            _check(rc, err)

    def read_dev(self, batch, d_keys, d_values, dtype=None, strides=None, stream=None):
        """Reads the batch's newest tokens back (whole sequences where cu_tokens
        counts them whole)."""
        k, v, code, token, head = self._sides(batch, d_keys, d_values, dtype, strides)
        err = _Err()
        rc = self._read(self._h, batch._ref, code, k, v, token, head, _stream(stream), C.byref(err))
        if rc:
            _check(rc, err)

    def attention_dev(self, batch, d_query, num_q_heads, scale, d_out, window=0, sinks=0, d_lse=None,
                      dtype=None, query_strides=None, out_strides=None, stream=None):
        """Causal attention of the batch's newest tokens over their pages:
        query and out [total_tokens, num_q_heads, head_dim].  With ``window`` a
        token sees its ``window`` last tokens (itself among them) and the first
        ``sinks``.  ``d_lse``: fp32 [total_tokens, num_q_heads] or None."""
        self._batch_here(batch)
        dim, total, device = self._dim, batch.total_tokens, self.device
        q, code, qt, qh = _rows(d_query, dtype, query_strides, num_q_heads, dim, total, "query", device)
        o, ocode, ot, oh = _rows(d_out, dtype, out_strides, num_q_heads, dim, total, "out", device)
        if ocode != code:
            raise _bad("query and out must have the same type")
        if window < 0 or sinks < 0:
            raise _bad("window and sinks must not be negative")
        if d_lse is not None and not isinstance(d_lse, int) and (
                str(d_lse.dtype) != "torch.float32" or not d_lse.is_contiguous()
                or tuple(d_lse.shape) != (total, num_q_heads) or d_lse.get_device() != device):
            raise _bad(f"lse must be contiguous fp32 [total_tokens, num_q_heads] on {_place(device)}")
        err = _Err()
        rc = self._attention(self._h, batch._ref, code, q, num_q_heads, qt, qh, scale, window, sinks, o,
                             ot, oh, _ptr(d_lse), _stream(stream), C.byref(err))
        if rc:
            _check(rc, err)

    def set_workspace(self, d_workspace, nbytes=None):
        """Later attention calls keep their partial states in `d_workspace`, a contiguous
        CUDA tensor (or a pointer with `nbytes`) of pages_workspace_size() bytes, instead of
        the device's scratch; None: the scratch again.  Before a capture whose graph may run
        beside other attention calls.  Handles may share one; calls that use it, replays
        among them, must follow one another."""
        if d_workspace is not None and not isinstance(d_workspace, int):
            if d_workspace.get_device() != self.device or not d_workspace.is_contiguous():
                raise _bad(f"a workspace must be contiguous memory of device {self.device}")
            nbytes = d_workspace.numel() * d_workspace.element_size()
        err = _Err()
        _check(lib().kivi_pages_set_workspace(self._h, _ptr(d_workspace), nbytes or 0, C.byref(err)), err)
        self._workspace = d_workspace

    def status(self):
        """Waits for the device; raises KiviError if a call since the last
        report met a page number or length outside its array, or gave up a wait."""
        err = _Err()
        _check(lib().kivi_pages_status(self._h, C.byref(err)), err)
