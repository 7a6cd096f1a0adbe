"""Low-bit operands: 4-bit microscaled matrices for the linears, and a paged 8- or 4-bit
key/value cache with the single-query attention that reads it.

32 consecutive elements of a row share one power-of-two scale; elements are 4-bit e2m1 or
8-bit e4m3 floating point (``include/vdit.h``, "microscaled operands").  The wrappers are
reached through ``fast_kernels`` beside the bf16 operators they stand in for: ``linear_mxfp4``
for ``linear``, ``attention_1q_cached`` for ``attention_1q``.  The reference has no counterpart:
it computes in bf16.
"""
from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Optional, Tuple, Union

import torch

from ._lib import KvCacheStruct, check, lib

BF16 = torch.bfloat16
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}     # VDIT_BF16, VDIT_F16, VDIT_F32
BLOCK = 32                                                           # elements that share a scale

# The calls here are a few microseconds of GPU work at their smallest, so the host path is kept
# short: raw stream handles and device indices, no device context unless another device is current.
_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice


def _need_cuda(index: int) -> None:
    if index < 0:
        raise RuntimeError("vdit kernels need CUDA tensors (no CPU path)")


def _same_device(what: str, index: int, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.get_device() != index:
            raise ValueError(f"{what}: tensors on different devices ({t.device} and cuda:{index})" if index >= 0 else
                             f"{what}: tensors on different devices ({t.device} and cpu)")


def _rows_view(what: str, name: str, t: torch.Tensor, dtypes) -> int:
    """Checks a 2D view with unit column stride; returns its row stride (a single row's may be
    anything, so it gets its own width, rounded up to the alignment rows need)."""
    if t.dim() != 2 or t.dtype not in dtypes or t.stride(1) != 1:
        raise ValueError(f"{what}: {name} must be a 2D view with unit column stride of type "
                         f"{' or '.join(str(d) for d in dtypes)}, got {tuple(t.shape)} {t.dtype}")
    rows, cols = t.shape
    if rows <= 1:
        return (cols + 7) & ~7
    ld = t.stride(0)
    if ld < cols:
        raise ValueError(f"{what}: the rows of {name} overlap")
    return ld


# ----------------------------------------------------------------------------- 4-bit matrices

def _scale_bytes(rows: int, cols: int) -> int:
    """vdit_mxfp4_scale_bytes: 512 bytes for every 128 rows x 128 columns begun."""
    return ((rows + 127) // 128) * ((cols + 127) // 128) * 512


class Mxfp4Tensor:
    """A quantised matrix [rows, cols]: ``codes`` uint8 [rows, cols / 2] (two elements a byte) and
    ``scales`` uint8 in the block-scaled MMA's order (opaque to callers).  ``quantize_mxfp4`` puts
    both into one buffer and makes the two views when they are asked for."""
    __slots__ = ("rows", "cols", "_data", "_codes", "_scales", "_pc", "_ps", "_index")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int):
        for t in (codes, scales):
            if t.dtype != torch.uint8 or not t.is_contiguous():
                raise ValueError("Mxfp4Tensor: codes and scales must be contiguous uint8")
        if (rows < 0 or cols < BLOCK or cols % BLOCK or codes.numel() != rows * cols // 2 or
                scales.numel() != _scale_bytes(rows, cols)):
            raise ValueError(f"Mxfp4Tensor: {codes.numel()} codes and {scales.numel()} scale bytes are not those "
                             f"of [{rows}, {cols}]")
        self._index = codes.get_device()
        _same_device("Mxfp4Tensor", self._index, scales)
        self.rows, self.cols, self._data, self._codes, self._scales = rows, cols, None, codes, scales
        self._pc, self._ps = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _new(cls, like: torch.Tensor, rows: int, cols: int) -> "Mxfp4Tensor":
        q = cls.__new__(cls)
        at = rows * cols // 2                               # a multiple of 16
        q._data = data = like.new_empty(at + _scale_bytes(rows, cols), dtype=torch.uint8)
        q.rows, q.cols, q._codes, q._scales, q._index = rows, cols, None, None, data.get_device()
        q._pc = pc = data.data_ptr()
        q._ps = pc + at
        return q

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            self._codes = self._data[:self.rows * self.cols // 2].view(self.rows, self.cols // 2)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._data[self.rows * self.cols // 2:]
        return self._scales

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.rows, self.cols)


def quantize_mxfp4(x: torch.Tensor) -> Mxfp4Tensor:
    """``x`` [M, K] (bf16, fp16 or fp32, row stride free, K a multiple of 32) in 4-bit microscaled
    form.  A block of 32 with a NaN or an infinity reads back as NaN."""
    ld = _rows_view("quantize_mxfp4", "x", x, _TYPES)
    m, k = x.shape
    if k == 0 or k % BLOCK:
        raise ValueError(f"quantize_mxfp4: {k} columns, not a multiple of {BLOCK}")
    index = x.get_device()
    _need_cuda(index)
    if index != _current():
        with torch.cuda.device(index):
            return quantize_mxfp4(x)
    q = Mxfp4Tensor._new(x, m, k)
    if m:
        check(lib().vdit_mxfp4_quantize(x.data_ptr(), _TYPES[x.dtype], ld, m, k, q._pc, q._ps, _stream(index)),
              "mxfp4_quantize")
    return q


def _check_mx(what: str, name: str, q: Mxfp4Tensor) -> None:
    if not isinstance(q, Mxfp4Tensor):
        raise ValueError(f"{what}: {name} must be an Mxfp4Tensor, got {type(q).__name__}")


def dequantize_mxfp4(q: Mxfp4Tensor, dtype: torch.dtype = BF16) -> torch.Tensor:
    """The values ``q`` stands for, [M, K] in ``dtype`` (exact in bf16 and fp32; fp16 rounds what
    lies outside its range)."""
    _check_mx("dequantize_mxfp4", "q", q)
    if dtype not in _TYPES:
        raise ValueError(f"dequantize_mxfp4: dtype must be bf16, fp16 or fp32, got {dtype}")
    m, k, index = q.rows, q.cols, q._index
    _need_cuda(index)
    if index != _current():
        with torch.cuda.device(index):
            return dequantize_mxfp4(q, dtype)
    out = (q._codes if q._data is None else q._data).new_empty((m, k), dtype=dtype)
    if m:
        check(lib().vdit_mxfp4_dequantize(q._pc, q._ps, m, k, out.data_ptr(), _TYPES[dtype], k, _stream(index)),
              "mxfp4_dequantize")
    return out


@lru_cache(maxsize=4096)
def _dense_workspace(m: int, k: int) -> int:
    return int(lib().vdit_linear_mxfp4_dense_workspace_bytes(m, k))


def linear_mxfp4(a: Union[torch.Tensor, Mxfp4Tensor], w: Mxfp4Tensor, bias: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``linear`` on 4-bit operands: ``F.linear(a, w, bias)`` of the quantised values, fp32
    accumulation, bf16 out.  ``a`` is an ``Mxfp4Tensor`` [M, K] or dense rows as
    ``quantize_mxfp4`` takes them (quantised in the call); ``w`` is the quantised weight [N, K]
    (N a multiple of 8)."""
    _check_mx("linear_mxfp4", "w", w)
    dense = torch.is_tensor(a)
    if dense:
        lda = _rows_view("linear_mxfp4", "a", a, _TYPES)
    else:
        _check_mx("linear_mxfp4", "a", a)
    m, k = a.shape
    n = w.rows
    if k != w.cols:
        raise ValueError(f"linear_mxfp4: a has {k} columns and w {w.cols}")
    if bias is not None and (bias.dtype != BF16 or bias.numel() != n or not bias.is_contiguous()):
        raise ValueError(f"linear_mxfp4: bias must be a contiguous bf16 vector of {n}")
    if out is None:
        ldo = n
    else:
        if out.dtype != BF16 or out.dim() != 2 or out.shape[0] < m or out.shape[1] < n:
            raise ValueError(f"linear_mxfp4: out must be a bf16 2D view of at least [{m}, {n}]")
        ldo = _rows_view("linear_mxfp4", "out", out, (BF16,))
    index = w._index
    if (a.get_device() if dense else a._index) != index or (bias is not None and bias.get_device() != index) or \
            (out is not None and out.get_device() != index):
        raise ValueError("linear_mxfp4: tensors on different devices")
    _need_cuda(index)
    if index != _current():
        with torch.cuda.device(index):
            return linear_mxfp4(a, w, bias, out)
    if out is None:
        out = (a if dense else w._codes if w._data is None else w._data).new_empty((m, n), dtype=BF16)
    if m:
        pb = None if bias is None else bias.data_ptr()
        if dense:
            nb = _dense_workspace(m, k)
            ws = out.new_empty(nb, dtype=torch.uint8) if nb else None
            check(lib().vdit_linear_mxfp4_dense(a.data_ptr(), _TYPES[a.dtype], lda, w._pc, w._ps, pb, out.data_ptr(),
                                                ldo, m, n, k, None if ws is None else ws.data_ptr(), nb,
                                                _stream(index)), "linear_mxfp4")
        else:
            check(lib().vdit_linear_mxfp4(a._pc, a._ps, w._pc, w._ps, pb, out.data_ptr(), ldo, m, n, k,
                                          _stream(index)), "linear_mxfp4")
    return out


# ----------------------------------------------------------------------------- key/value cache

class MxKvCache:
    """A paged cache of keys and values held in 8 (e4m3) or 4 (e2m1) bits with a scale per 32
    channels.  Slot ``page * page_size + offset`` holds one row of ``kv_heads * head_dim``
    channels.  ``page_size`` is a power of two from 16 to 1024, ``head_dim`` 32, 64, 96 or 128.  Its
    buffers ``k``, ``v``, ``k_scales`` and ``v_scales`` stay where they are."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 8, device="cuda"):
        if bits not in (4, 8):
            raise ValueError(f"MxKvCache: bits must be 4 or 8, got {bits}")
        if head_dim not in (32, 64, 96, 128):
            raise ValueError(f"MxKvCache: head_dim must be 32, 64, 96 or 128, got {head_dim}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"MxKvCache: page_size must be a power of two from 16 to 1024, got {page_size}")
        if pages < 1 or kv_heads < 1:
            raise ValueError(f"MxKvCache: needs pages and heads, got {pages} and {kv_heads}")
        self.pages, self.page_size, self.kv_heads, self.head_dim, self.bits = pages, page_size, kv_heads, head_dim, bits
        self.slots, self.width = pages * page_size, kv_heads * head_dim
        shape = (pages, kv_heads, page_size)
        # zeros: a slot that was never written reads as zeros
        self._k, self._v = (torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device) for _ in range(2))
        self._ks, self._vs = (torch.zeros(*shape, head_dim // BLOCK, dtype=torch.uint8, device=device) for _ in range(2))
        self.device = self._k.device
        self._index = self._k.get_device()
        self._struct = KvCacheStruct(*(t.data_ptr() for t in (self._k, self._v, self._ks, self._vs)), pages, page_size,
                                     kv_heads, head_dim, bits)
        self._ref = ctypes.addressof(self._struct)

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scales = property(lambda self: self._ks)
    v_scales = property(lambda self: self._vs)


def _check_slots(what: str, cache: MxKvCache, slots: torch.Tensor) -> int:
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be a contiguous int64 vector, got {tuple(slots.shape)} {slots.dtype}")
    return slots.shape[0]


def kv_cache_write(cache: MxKvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise the rows ``k`` and ``v`` (bf16 [T, kv_heads * head_dim], row strides free) into
    ``slots`` (int64 [T]).  Negative slots are skipped; the others must differ from one another.
    A slot past the cache is left out and recorded in the device error word."""
    n = _check_slots("kv_cache_write", cache, slots)
    ldk = _rows_view("kv_cache_write", "k", k, (BF16,))
    ldv = _rows_view("kv_cache_write", "v", v, (BF16,))
    shape = (n, cache.width)
    if k.shape != shape or v.shape != shape:
        raise ValueError(f"kv_cache_write: k and v must be [{n}, {cache.width}], got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    index = cache._index
    _same_device("kv_cache_write", index, k, v, slots)
    _need_cuda(index)
    if n == 0:
        return
    if index != _current():
        with torch.cuda.device(index):
            return kv_cache_write(cache, k, v, slots)
    check(lib().vdit_kv_cache_write(k.data_ptr(), ldk, v.data_ptr(), ldv, slots.data_ptr(), n, cache._ref,
                                    _stream(index)), "kv_cache_write")


def kv_cache_read(cache: MxKvCache, slots: torch.Tensor, dtype: torch.dtype = BF16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that ``slots`` (int64 [T]) hold, [T, kv_heads * head_dim] each in ``dtype``
    (bf16 or fp32, both exact): the rows ``attention`` and ``flash_cross_attn`` take.  Negative
    slots give zeros; a slot past the cache too, recorded in the device error word."""
    n = _check_slots("kv_cache_read", cache, slots)
    if dtype is not BF16 and dtype is not torch.float32:
        raise ValueError(f"kv_cache_read: dtype must be bf16 or fp32, got {dtype}")
    index, d = cache._index, cache.width
    _same_device("kv_cache_read", index, slots)
    _need_cuda(index)
    if index != _current():
        with torch.cuda.device(index):
            return kv_cache_read(cache, slots, dtype)
    k = slots.new_empty((n, d), dtype=dtype)
    v = torch.empty_like(k)
    if n:
        check(lib().vdit_kv_cache_read(cache._ref, slots.data_ptr(), n, k.data_ptr(), d, v.data_ptr(), d,
                                       _TYPES[dtype], _stream(index)), "kv_cache_read")
    return k, v


@lru_cache(maxsize=4096)
def _attend_workspace(b: int, heads: int, kv_heads: int, head_dim: int, pages: int, page_size: int) -> int:
    return int(lib().vdit_attention_1q_cached_workspace_bytes(b, heads, kv_heads, head_dim, pages, page_size))


def attention_1q_cached(q: torch.Tensor, cache: MxKvCache, page_table: torch.Tensor, lengths: torch.Tensor,
                        scale: Optional[float] = None) -> torch.Tensor:
    """``attention_1q`` for a batch of sequences whose keys and values are in ``cache``: one query per
    sequence and head, ``q`` bf16 [B, heads * head_dim] (heads a multiple of the cache's; query head
    h reads key head h // (heads / kv_heads)), ``page_table`` int32 [B, P] (row stride free; 0, as of
    an expanded row, shares it), ``lengths`` int32 [B].  Key i of sequence b is in page
    ``page_table[b, i // page_size]``; entries past a length are not read, and a sequence without
    keys gives zeros.  Pages outside the cache are left out and lengths outside the table are clipped
    to it, both recorded in the device error word.  Returns bf16 [B, heads * head_dim]."""
    what = "attention_1q_cached"
    ldq = _rows_view(what, "q", q, (BF16,))
    b, d = q.shape
    if d == 0 or d % cache.width:
        raise ValueError(f"{what}: q has {d} channels, not a multiple of the cache's {cache.width}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b or \
            page_table.shape[1] < 1 or page_table.stride(1) != 1:
        raise ValueError(f"{what}: page_table must be int32 [{b}, pages >= 1] with unit column stride, "
                         f"got {tuple(page_table.shape)} {page_table.dtype}")
    if lengths.dtype != torch.int32 or lengths.dim() != 1 or lengths.shape[0] != b or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths must be a contiguous int32 [{b}], got {tuple(lengths.shape)} {lengths.dtype}")
    index = cache._index
    _same_device(what, index, q, page_table, lengths)
    _need_cuda(index)
    if index != _current():
        with torch.cuda.device(index):
            return attention_1q_cached(q, cache, page_table, lengths, scale)
    out = q.new_empty((b, d))
    if b:
        hd, pages = cache.head_dim, page_table.shape[1]
        heads = d // hd
        nb = _attend_workspace(b, heads, cache.kv_heads, hd, pages, cache.page_size)
        ws = q.new_empty(nb, dtype=torch.uint8) if nb else None
        check(lib().vdit_attention_1q_cached(q.data_ptr(), ldq, cache._ref, page_table.data_ptr(),
                                             page_table.stride(0) if b > 1 else pages, pages, lengths.data_ptr(), b,
                                             heads, 1.0 / math.sqrt(hd) if scale is None else float(scale),
                                             out.data_ptr(), d, None if ws is None else ws.data_ptr(), nb,
                                             _stream(index)), what)
    return out
