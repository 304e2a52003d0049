"""Paged K/V cache: many streams, and the beams of one stream, share one pool
of pages per layer.

* ``paged_write`` -- new keys and values into pages (a prompt's, or one token a
  row), the paged form of ``RingCache::record_prefill`` / ``write_decode_step``
  (native_engine/rswa.rs:389, :451-500);
* ``paged_attention`` -- one new token per row over its pages, with the R-SWA
  rule of ``rswa::decode_attention`` (rswa.rs:855-944) where ``window`` is
  given; it can add every position's probability to ``weights``;
* ``paged_evict`` -- a row shrinks to its most attended entries by them.

A pool is ``[pages, kv_heads, page_size, head_dim]`` (f32, f16 or bf16), one for
K and one for V with the same strides; a row's position ``p`` lies in page
``table[row, p // page_size]``, slot ``p % page_size``.  The calls take CUDA
tensors on one device, enqueue work on torch's current stream of that device
and can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct

import torch

from ._lib import F32, F16, BF16, FOCR_OK, PagedCache, check, lib

_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
# a PagedCache's bytes: packing them costs a third of filling the ctypes structure
_PACK = struct.Struct("6N5Ii")
assert _PACK.size == C.sizeof(PagedCache)


def _dtype(ctx: str, name: str, t) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{ctx}: {name} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def _need(ctx: str, name: str, t, dtype, shape, device) -> None:
    """A contiguous tensor of that type and shape on that device."""
    if t.dtype != dtype:
        raise TypeError(f"{ctx}: {name} must be {dtype}, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{ctx}: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{ctx}: {name} is on {t.device}, not {device}")
    if not t.is_contiguous():
        raise ValueError(f"{ctx}: {name} must be contiguous")


def _cache(ctx: str, k_pages, v_pages, table, dims: int = 4):
    """The checked cache as the C ABI's struct; its device, kv heads, head_dim and table's shape."""
    device = k_pages.device
    if device.type != "cuda":
        raise ValueError(f"{ctx}: the pages must be CUDA tensors, not on {device}")
    code = _dtype(ctx, "k_pages", k_pages)
    shape, stride = k_pages.shape, k_pages.stride()
    if len(shape) != dims:
        raise ValueError(f"{ctx}: k_pages must have {dims} dimensions, not {len(shape)}")
    if v_pages.shape != shape or v_pages.stride() != stride or v_pages.dtype != k_pages.dtype \
            or v_pages.device != device:
        raise ValueError(f"{ctx}: v_pages must match k_pages in shape, strides, type and device")
    pages, heads, page, dim = shape[-4:]
    if stride[-1] != 1 or stride[-2] != dim:
        raise ValueError(f"{ctx}: the entries of a head's page must be contiguous")
    if table.dtype != torch.int32:
        raise TypeError(f"{ctx}: table must be torch.int32, not {table.dtype}")
    if table.dim() != 2 or table.stride(1) != 1 or table.device != device:
        raise ValueError(f"{ctx}: table must be [rows, pages] on {device} with contiguous rows")
    rows, width = table.shape
    try:
        packed = _PACK.pack(k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), stride[-4], stride[-3],
                            max(table.stride(0), width), pages, heads, page, dim, width, code)
    except struct.error as e:
        raise ValueError(f"{ctx}: a dimension exceeds 32 bits") from e
    return packed, device, heads, dim, rows, width


def _call(fn, device, *args) -> None:
    """One call of the C ABI on the device's current stream, its last argument."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != FOCR_OK:
        check(rc)


@functools.lru_cache(maxsize=256)
def _workspace(fn: str, *sizes) -> int:
    """Bytes of a call's workspace, which go by its sizes alone."""
    need = C.c_size_t()
    check(getattr(lib, fn)(*sizes, C.byref(need)))
    return need.value


def _weights(ctx: str, w, rows: int, heads: int, device):
    if w.dtype != torch.float32:
        raise TypeError(f"{ctx}: weights must be torch.float32, not {w.dtype}")
    if w.dim() != 3 or w.shape[0] != rows or w.shape[1] != heads or w.device != device:
        raise ValueError(f"{ctx}: weights must be [{rows}, {heads}, width] on {device}, "
                         f"not {tuple(w.shape)} on {w.device}")
    if w.stride(2) != 1:
        raise ValueError(f"{ctx}: the last dimension of weights must be contiguous")


def paged_write(k, v, k_pages, v_pages, table, pos, row=None) -> None:
    """Write ``k``, ``v`` ``[tokens, kv_heads, head_dim]`` into pages: token ``t``
    to position ``pos[t]`` of table row ``row[t]`` (``row`` None: row ``t``).
    Tokens with ``row[t] < 0`` are padding; rows, positions and pages out of
    range are skipped.  ``pos`` and ``row`` are int32 on the device."""
    ctx = "paged_write"
    cache, device, heads, dim, rows, _ = _cache(ctx, k_pages, v_pages, table)
    src = _dtype(ctx, "k", k)
    tokens = k.shape[0]
    shape, ks, vs = (tokens, heads, dim), k.stride(), v.stride()
    if k.shape != shape or v.shape != shape or v.dtype != k.dtype or k.device != device or v.device != device:
        raise ValueError(f"{ctx}: k and v must be [tokens, {heads}, {dim}] of one type on {device}, not "
                         f"{tuple(k.shape)} of {k.dtype} on {k.device} and {tuple(v.shape)} of {v.dtype} on {v.device}")
    if ks[2] != 1 or vs[2] != 1 or (heads > 1 and (ks[1] != dim or vs[1] != dim)):
        raise ValueError(f"{ctx}: a token of k and of v must be contiguous")
    _need(ctx, "pos", pos, torch.int32, (tokens,), device)
    if row is not None:
        _need(ctx, "row", row, torch.int32, (tokens,), device)
    _call(lib.focr_paged_write, device, cache, rows, k.data_ptr(), v.data_ptr(), src, tokens, ks[0], vs[0],
          None if row is None else row.data_ptr(), pos.data_ptr())


def paged_attention(q, k_pages, v_pages, table, lens, *, scale: float | None = None, ref_lens=None,
                    window: int = 0, weights=None, out=None):
    """``q`` ``[rows, q_heads, head_dim]`` over each row's first ``lens[row]``
    positions; returns ``[rows, q_heads, head_dim]`` of q's type.  Query head
    ``h`` reads kv head ``h // (q_heads // kv_heads)``; ``scale`` defaults to
    ``1 / sqrt(head_dim)``.  With ``window`` a row sees its first
    ``ref_lens[row]`` and its last ``window`` positions.  ``weights``
    ``[rows, kv_heads, width]`` f32 is added to: every seen position's
    probability, summed over the query heads of its kv head.

    A row that sees nothing gives zeros.  A length past the table (or the
    weights), or a page id outside the pool, gives NaN for that row."""
    ctx = "paged_attention"
    cache, device, kv_heads, dim, rows, _ = _cache(ctx, k_pages, v_pages, table)
    code = _dtype(ctx, "q", q)
    shape, stride = q.shape, q.stride()
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim or q.device != device:
        raise ValueError(f"{ctx}: q must be [{rows}, q_heads, {dim}] on {device}, "
                         f"not {tuple(shape)} on {q.device}")
    heads = shape[1]
    if stride[2] != 1 or (heads > 1 and stride[1] != dim):
        raise ValueError(f"{ctx}: a row of q must be contiguous")
    if window < 0:
        raise ValueError(f"{ctx}: window must not be negative")
    _need(ctx, "lens", lens, torch.int32, (rows,), device)
    if ref_lens is not None:
        _need(ctx, "ref_lens", ref_lens, torch.int32, (rows,), device)
    width = w_row = w_head = 0
    if weights is not None:
        _weights(ctx, weights, rows, kv_heads, device)
        width, w_row, w_head = weights.shape[2], weights.stride(0), weights.stride(1)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype, device=device)
    else:
        _need(ctx, "out", out, q.dtype, shape, device)
    need = _workspace("focr_paged_attention_workspace", rows, heads, dim, width)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _call(lib.focr_paged_attention, device, cache, q.data_ptr(), code, rows, heads, stride[0], lens.data_ptr(),
          None if ref_lens is None else ref_lens.data_ptr(), window,
          1.0 / math.sqrt(dim) if scale is None else scale, out.data_ptr(), heads * dim,
          None if weights is None else weights.data_ptr(), width, w_row, w_head, ws.data_ptr(), need)
    return out


def paged_evict(k_pages, v_pages, table, lens, weights, new_table, budget: int, *, sink: int = 0,
                recent: int = 0):
    """Shrink every row of more than ``budget`` entries to ``budget``: its first
    ``sink``, its last ``recent`` and, between them, the entries of the largest
    ``weights`` (``[rows, kv_heads, width]`` f32; equal ones: the lower
    position), each kv head for itself.  The kept entries go, in order, to the
    pages of ``new_table`` ``[rows, pages]``, none of which may be a page that a
    row of this call reads; the old pages are not written.

    Returns ``(kept, lens, weights)``: the old positions ``[rows, kv_heads,
    budget]`` (-1 behind the last), the new lengths, and the kept entries'
    weights in a tensor of ``weights``' shape, 0 behind them."""
    ctx = "paged_evict"
    cache, device, heads, _, rows, _ = _cache(ctx, k_pages, v_pages, table)
    _need(ctx, "lens", lens, torch.int32, (rows,), device)
    _weights(ctx, weights, rows, heads, device)
    if new_table.dtype != torch.int32:
        raise TypeError(f"{ctx}: new_table must be torch.int32, not {new_table.dtype}")
    if new_table.dim() != 2 or new_table.shape[0] != rows or new_table.stride(1) != 1 \
            or new_table.device != device:
        raise ValueError(f"{ctx}: new_table must be [{rows}, pages] on {device} with contiguous rows")
    if budget < 1 or sink < 0 or recent < 0:
        raise ValueError(f"{ctx}: budget must be positive, sink and recent not negative")
    width = weights.shape[2]
    kept = torch.empty((rows, heads, budget), dtype=torch.int32, device=device)
    new_lens = torch.empty((rows,), dtype=torch.int32, device=device)
    new_weights = torch.empty((rows, heads, width), dtype=torch.float32, device=device)
    _call(lib.focr_paged_evict, device, cache, rows, lens.data_ptr(), weights.data_ptr(), width, weights.stride(0),
          weights.stride(1), new_table.data_ptr(), max(new_table.stride(0), new_table.shape[1]),
          new_table.shape[1], budget, sink, recent, kept.data_ptr(), new_lens.data_ptr(), new_weights.data_ptr())
    return kept, new_lens, new_weights
