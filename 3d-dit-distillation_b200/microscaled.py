"""Low-bit operands: 4-bit microscaled matrices for the linears, and a paged 8- or 4-bit
key/value cache with the single-query attention that reads it.

32 consecutive elements of a row share one power-of-two scale; elements are 4-bit e2m1 or
8-bit e4m3 floating point (``include/vdit.h``, "microscaled operands").  The wrappers are
reached through ``fast_kernels`` beside the bf16 operators they stand in for: ``linear_mxfp4``
for ``linear``, ``attention_1q_cached`` for ``attention_1q``.  The reference has no counterpart:
it computes in bf16.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from ._lib import check, lib, ptr, stream_of

BF16 = torch.bfloat16
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}     # VDIT_BF16, VDIT_F16, VDIT_F32
BLOCK = 32                                                           # elements that share a scale


def _same_device(what: str, first: torch.Tensor, *rest: Optional[torch.Tensor]) -> None:
    for t in rest:
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def _rows_view(what: str, name: str, t: torch.Tensor, dtypes) -> None:
    """A 2D view with unit column stride whose rows start on 16-byte boundaries."""
    if t.dim() != 2 or t.dtype not in dtypes or t.stride(1) != 1:
        raise ValueError(f"{what}: {name} must be a 2D view with unit column stride of type "
                         f"{' or '.join(str(d) for d in dtypes)}, got {tuple(t.shape)} {t.dtype}")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: the rows of {name} overlap")


def _ld(t: torch.Tensor) -> int:
    """Row stride of a 2D view (a single row's stride may be anything)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], -(-t.shape[1] // 8) * 8)


# ----------------------------------------------------------------------------- 4-bit matrices

@dataclass(frozen=True)
class Mxfp4Tensor:
    """A quantised matrix [rows, cols]: ``codes`` uint8 [rows, cols / 2] (two elements a byte) and
    ``scales`` uint8 in the block-scaled MMA's order (opaque to callers)."""
    codes: torch.Tensor
    scales: torch.Tensor
    rows: int
    cols: int

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.rows, self.cols)

    @property
    def device(self) -> torch.device:
        return self.codes.device


def quantize_mxfp4(x: torch.Tensor) -> Mxfp4Tensor:
    """``x`` [M, K] (bf16, fp16 or fp32, row stride free, K a multiple of 32) in 4-bit microscaled
    form.  A block of 32 with a NaN or an infinity reads back as NaN."""
    _rows_view("quantize_mxfp4", "x", x, tuple(_TYPES))
    m, k = x.shape
    if k == 0 or k % BLOCK:
        raise ValueError(f"quantize_mxfp4: {k} columns, not a multiple of {BLOCK}")
    p = ptr(x)
    with torch.cuda.device(x.device):
        codes = torch.empty(m, k // 2, dtype=torch.uint8, device=x.device)
        scales = torch.empty(int(lib().vdit_mxfp4_scale_bytes(m, k)), dtype=torch.uint8, device=x.device)
        if m:
            check(lib().vdit_mxfp4_quantize(p, _TYPES[x.dtype], _ld(x), m, k, ptr(codes), ptr(scales),
                                            stream_of(x)), "mxfp4_quantize")
    return Mxfp4Tensor(codes, scales, m, k)


def _check_mx(what: str, name: str, q: Mxfp4Tensor) -> None:
    if not isinstance(q, Mxfp4Tensor):
        raise ValueError(f"{what}: {name} must be an Mxfp4Tensor, got {type(q).__name__}")
    for t in (q.codes, q.scales):
        if t.dtype != torch.uint8 or not t.is_contiguous():
            raise ValueError(f"{what}: {name} needs contiguous uint8 codes and scales")
    if (q.cols % BLOCK or q.codes.numel() != q.rows * q.cols // 2 or
            q.scales.numel() != int(lib().vdit_mxfp4_scale_bytes(q.rows, q.cols))):
        raise ValueError(f"{what}: {name} holds {q.codes.numel()} codes and {q.scales.numel()} scale bytes, "
                         f"not those of [{q.rows}, {q.cols}]")
    _same_device(what, q.codes, q.scales)


def dequantize_mxfp4(q: Mxfp4Tensor, dtype: torch.dtype = BF16) -> torch.Tensor:
    """The values ``q`` stands for, [M, K] in ``dtype`` (exact in bf16 and fp32; fp16 rounds what
    lies outside its range)."""
    _check_mx("dequantize_mxfp4", "q", q)
    if dtype not in _TYPES:
        raise ValueError(f"dequantize_mxfp4: dtype must be bf16, fp16 or fp32, got {dtype}")
    p = ptr(q.codes)
    with torch.cuda.device(q.device):
        out = torch.empty(q.rows, q.cols, dtype=dtype, device=q.device)
        if q.rows:
            check(lib().vdit_mxfp4_dequantize(p, ptr(q.scales), q.rows, q.cols, ptr(out), _TYPES[dtype], q.cols,
                                              stream_of(out)), "mxfp4_dequantize")
    return out


def linear_mxfp4(a: Union[torch.Tensor, Mxfp4Tensor], w: Mxfp4Tensor, bias: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``linear`` on 4-bit operands: ``F.linear(a, w, bias)`` of the quantised values, fp32
    accumulation, bf16 out.  ``a`` is an ``Mxfp4Tensor`` [M, K] or dense rows as
    ``quantize_mxfp4`` takes them (quantised in the call); ``w`` is the quantised weight [N, K]
    (N a multiple of 8)."""
    _check_mx("linear_mxfp4", "w", w)
    dense = torch.is_tensor(a)
    if dense:
        _rows_view("linear_mxfp4", "a", a, tuple(_TYPES))
    else:
        _check_mx("linear_mxfp4", "a", a)
    m, k = a.shape
    n = w.rows
    if k != w.cols:
        raise ValueError(f"linear_mxfp4: a has {k} columns and w {w.cols}")
    if bias is not None and (bias.dtype != BF16 or bias.numel() != n or not bias.is_contiguous()):
        raise ValueError(f"linear_mxfp4: bias must be a contiguous bf16 vector of {n}")
    if out is not None and (out.dtype != BF16 or out.dim() != 2 or out.shape[0] < m or out.shape[1] < n or
                            out.stride(1) != 1 or (out.shape[0] > 1 and out.stride(0) < n)):
        raise ValueError(f"linear_mxfp4: out must be a bf16 2D view of at least [{m}, {n}]")
    _same_device("linear_mxfp4", w.codes, a if dense else a.codes, bias, out)
    p = ptr(w.codes)
    with torch.cuda.device(w.device):
        if dense:
            a = quantize_mxfp4(a)
        if out is None:
            out = torch.empty(m, n, dtype=BF16, device=w.device)
        if m:
            check(lib().vdit_linear_mxfp4(ptr(a.codes), ptr(a.scales), p, ptr(w.scales), ptr(bias), ptr(out),
                                          _ld(out), m, n, k, stream_of(out)), "linear_mxfp4")
    return out


# ----------------------------------------------------------------------------- key/value cache

class MxKvCache:
    """A paged cache of keys and values held in 8 (e4m3) or 4 (e2m1) bits with a scale per 32
    channels.  Slot ``page * page_size + offset`` holds one row of ``kv_heads * head_dim``
    channels.  ``page_size`` is a power of two up to 1024, ``head_dim`` 32, 64, 96 or 128."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 8, device="cuda"):
        if bits not in (4, 8):
            raise ValueError(f"MxKvCache: bits must be 4 or 8, got {bits}")
        if head_dim not in (32, 64, 96, 128):
            raise ValueError(f"MxKvCache: head_dim must be 32, 64, 96 or 128, got {head_dim}")
        if page_size < 1 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"MxKvCache: page_size must be a power of two up to 1024, got {page_size}")
        if pages < 1 or kv_heads < 1:
            raise ValueError(f"MxKvCache: needs pages and heads, got {pages} and {kv_heads}")
        self.pages, self.page_size, self.kv_heads, self.head_dim, self.bits = pages, page_size, kv_heads, head_dim, bits
        shape = (pages, kv_heads, page_size)
        # zeros: a slot that was never written reads as zeros
        self.k, self.v = (torch.zeros(*shape, head_dim * bits // 8, dtype=torch.uint8, device=device) for _ in range(2))
        self.k_scales, self.v_scales = (torch.zeros(*shape, head_dim // BLOCK, dtype=torch.uint8, device=device)
                                        for _ in range(2))

    @property
    def slots(self) -> int:
        return self.pages * self.page_size

    @property
    def width(self) -> int:
        return self.kv_heads * self.head_dim

    @property
    def device(self) -> torch.device:
        return self.k.device

    def _pointers(self):
        return ptr(self.k), ptr(self.v), ptr(self.k_scales), ptr(self.v_scales)

    def _geometry(self):
        return self.pages, self.page_size, self.kv_heads, self.head_dim, self.bits


def _check_slots(what: str, cache: MxKvCache, slots: torch.Tensor) -> None:
    if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError(f"{what}: slots must be a contiguous int64 vector, got {tuple(slots.shape)} {slots.dtype}")
    _same_device(what, cache.k, slots)


def kv_cache_write(cache: MxKvCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise the rows ``k`` and ``v`` (bf16 [T, kv_heads * head_dim], row strides free) into
    ``slots`` (int64 [T]).  Negative slots are skipped; the others must differ from one another.
    A slot past the cache is left out and recorded in the device error word."""
    _check_slots("kv_cache_write", cache, slots)
    for t, name in ((k, "k"), (v, "v")):
        _rows_view("kv_cache_write", name, t, (BF16,))
        if t.shape != (slots.numel(), cache.width):
            raise ValueError(f"kv_cache_write: {name} must be [{slots.numel()}, {cache.width}], got {tuple(t.shape)}")
    _same_device("kv_cache_write", cache.k, k, v)
    if slots.numel() == 0:
        return
    pk = ptr(k)
    with torch.cuda.device(cache.device):
        check(lib().vdit_kv_cache_write(pk, _ld(k), ptr(v), _ld(v), ptr(slots), slots.numel(), *cache._pointers(),
                                        *cache._geometry(), stream_of(k)), "kv_cache_write")


def kv_cache_read(cache: MxKvCache, slots: torch.Tensor, dtype: torch.dtype = BF16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that ``slots`` (int64 [T]) hold, [T, kv_heads * head_dim] each in ``dtype``
    (bf16 or fp32, both exact): the rows ``attention`` and ``flash_cross_attn`` take.  Negative
    slots give zeros; a slot past the cache too, recorded in the device error word."""
    _check_slots("kv_cache_read", cache, slots)
    if dtype not in (BF16, torch.float32):
        raise ValueError(f"kv_cache_read: dtype must be bf16 or fp32, got {dtype}")
    ps = ptr(slots)
    with torch.cuda.device(cache.device):
        k = torch.empty(slots.numel(), cache.width, dtype=dtype, device=cache.device)
        v = torch.empty_like(k)
        if slots.numel():
            check(lib().vdit_kv_cache_read(*cache._pointers(), *cache._geometry(), ps, slots.numel(), ptr(k),
                                           cache.width, ptr(v), cache.width, _TYPES[dtype], stream_of(k)),
                  "kv_cache_read")
    return k, v


def attention_1q_cached(q: torch.Tensor, cache: MxKvCache, page_table: torch.Tensor, lengths: torch.Tensor,
                        scale: Optional[float] = None) -> torch.Tensor:
    """``attention_1q`` for a batch of sequences whose keys and values are in ``cache``: one query per
    sequence and head, ``q`` bf16 [B, heads * head_dim] (heads a multiple of the cache's; query head
    h reads key head h // (heads / kv_heads)), ``page_table`` int32 [B, P] (row stride free; 0, as of an expanded row, shares it),
    ``lengths`` int32 [B].  Key i of sequence b is in page ``page_table[b, i // page_size]``; entries
    past a length are not read, and a sequence of length 0 gives zeros.  Pages outside the cache
    are left out and lengths outside the table are clipped to it, both recorded in the device
    error word.  Returns bf16 [B, heads * head_dim]."""
    what = "attention_1q_cached"
    _rows_view(what, "q", q, (BF16,))
    b, d = q.shape
    if d == 0 or d % cache.width:
        raise ValueError(f"{what}: q has {d} channels, not a multiple of the cache's {cache.width}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b or \
            page_table.shape[1] < 1 or page_table.stride(1) != 1:
        raise ValueError(f"{what}: page_table must be int32 [{b}, pages >= 1] with unit column stride, "
                         f"got {tuple(page_table.shape)} {page_table.dtype}")
    if lengths.dtype != torch.int32 or lengths.shape != (b,) or not lengths.is_contiguous():
        raise ValueError(f"{what}: lengths must be a contiguous int32 [{b}], got {tuple(lengths.shape)} {lengths.dtype}")
    _same_device(what, cache.k, q, page_table, lengths)
    heads, pages = d // cache.head_dim, page_table.shape[1]
    scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
    pq = ptr(q)
    with torch.cuda.device(cache.device):
        out = torch.empty(b, d, dtype=BF16, device=cache.device)
        if b:
            nb = int(lib().vdit_attention_1q_cached_workspace_bytes(b, heads, cache.kv_heads, cache.head_dim, pages,
                                                                    cache.page_size))
            ws = torch.empty(nb, dtype=torch.uint8, device=cache.device)
            kc, vc, ks, vs = cache._pointers()
            check(lib().vdit_attention_1q_cached(pq, _ld(q), kc, vc, ks, vs, *cache._geometry(), ptr(page_table),
                                                 page_table.stride(0) if b > 1 else pages, pages, ptr(lengths), b, heads, scale,
                                                 ptr(out), d, ptr(ws), nb, stream_of(q)), what)
    return out
