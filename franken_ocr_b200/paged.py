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
and can be captured into a CUDA graph.  They are for decoding: no gradient passes
through them, and no output requires one.

The checks are written for speed: a decode step makes these calls for every
layer, and the smallest run 2 us on the device.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct

import torch

from ._lib import (BF16, F16, F32, FOCR_OK, PagedAttentionArgs, PagedCache, PagedEvictArgs, PagedWriteArgs, check,
                   lib)

_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_F32, _I32, _U8 = torch.float32, torch.int32, torch.uint8


def _packer(kind, form: str):
    """The bytes of a ctypes structure: packing them costs a tenth of filling it, or
    of passing its fields one by one."""
    s = struct.Struct(form + "0N")
    assert s.size == C.sizeof(kind), kind
    return s.pack


_pack_cache = _packer(PagedCache, "6N5Ii")
_pack_write = _packer(PagedWriteArgs, "8Ni")
_pack_attention = _packer(PagedAttentionArgs, "15Nif")
_pack_evict = _packer(PagedEvictArgs, "15N")
# torch's own short cuts where it has them, its public calls where not: the current
# device, its stream, and an allocation on it without the dispatcher (half the time; the
# calls work on addresses, so no dispatch mode could follow them either way)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
try:
    from torch._C._dynamo.guards import _empty_strided_cuda as _quick_empty
except ImportError:
    _quick_empty = None


def _empty(shape, stride, dtype):
    try:
        return _quick_empty(shape, stride, dtype)
    except TypeError:  # there is none, or it takes something else
        return torch.empty_strided(shape, stride, dtype=dtype, device="cuda")


def _dtype(ctx: str, name: str, t) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{ctx}: {name} must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def _need(ctx: str, name: str, t, dtype, shape, index: int) -> None:
    """A contiguous tensor of that type and shape on that device."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous():
        return
    if t.dtype is not dtype:
        raise TypeError(f"{ctx}: {name} must be {dtype}, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{ctx}: {name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.get_device() != index:
        raise ValueError(f"{ctx}: {name} is on {t.device}, not cuda:{index}")
    raise ValueError(f"{ctx}: {name} must be contiguous")


def _table(ctx: str, name: str, t, index: int):
    """(rows, columns, row stride) of an int32 page table."""
    if t.dtype is not _I32:
        raise TypeError(f"{ctx}: {name} must be torch.int32, not {t.dtype}")
    if t.dim() != 2 or t.get_device() != index:
        raise ValueError(f"{ctx}: {name} must be [rows, pages] on cuda:{index}")
    rows, width = t.shape
    step, unit = t.stride()
    if unit != 1 and width > 1:
        raise ValueError(f"{ctx}: the rows of {name} must be contiguous")
    return rows, width, step if rows > 1 else width


def _cache(ctx: str, k_pages, v_pages, table, dims: int = 4):
    """The checked cache as the C ABI's struct; its device's index, kv heads,
    head_dim and table's shape."""
    index = k_pages.get_device()
    if index < 0:
        raise ValueError(f"{ctx}: the pages must be CUDA tensors, not on {k_pages.device}")
    code = _dtype(ctx, "k_pages", k_pages)
    shape, stride = k_pages.shape, k_pages.stride()
    if len(shape) != dims:
        raise ValueError(f"{ctx}: k_pages must have {dims} dimensions, not {len(shape)}")
    if v_pages.shape != shape or v_pages.stride() != stride or v_pages.dtype is not k_pages.dtype \
            or v_pages.get_device() != index:
        raise ValueError(f"{ctx}: v_pages must match k_pages in shape, strides, type and device")
    pages, heads, page, dim = shape[-4:]
    if stride[-1] != 1 or (stride[-2] != dim and page > 1):
        raise ValueError(f"{ctx}: the entries of a head's page must be contiguous")
    rows, width, step = _table(ctx, "table", table, index)
    try:
        packed = _pack_cache(k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), stride[-4], stride[-3],
                            step, pages, heads, page, dim, width, code)
    except struct.error as e:
        raise ValueError(f"{ctx}: a dimension exceeds 32 bits") from e
    return packed, index, heads, dim, rows, width


def _misfit(ctx: str, e: Exception) -> ValueError:
    """For a caller's number that its C type does not hold."""
    return ValueError(f"{ctx}: an argument is out of range ({e})")


def _elsewhere(fn, index: int, *args, **kw):
    """The same call with its tensors' device as the current one."""
    with torch.cuda.device(index):
        return fn(*args, **kw)


@functools.lru_cache(maxsize=256)
def _workspace(fn: str, index: int, *sizes) -> int:
    """Bytes of a call's workspace on device `index`, the current one, by whose number of
    SMs they go beside the sizes."""
    need = C.c_size_t()
    check(getattr(lib, fn)(*sizes, C.byref(need)))
    return need.value


def _weights(ctx: str, w, rows: int, heads: int, index: int):
    """(width, row stride, head stride) of accumulated weights."""
    if w.dtype is not _F32:
        raise TypeError(f"{ctx}: weights must be torch.float32, not {w.dtype}")
    shape = w.shape
    if len(shape) != 3 or shape[0] != rows or shape[1] != heads or w.get_device() != index:
        raise ValueError(f"{ctx}: weights must be [{rows}, {heads}, width] on cuda:{index}, "
                         f"not {tuple(shape)} on {w.device}")
    row, head, unit = w.stride()
    if unit != 1 and shape[2] > 1:
        raise ValueError(f"{ctx}: the last dimension of weights must be contiguous")
    return shape[2], row, head


def paged_write(k, v, k_pages, v_pages, table, pos, row=None) -> None:
    """Write ``k``, ``v`` ``[tokens, kv_heads, head_dim]`` into pages: token ``t``
    to position ``pos[t]`` of table row ``row[t]`` (``row`` None: row ``t``).
    Tokens with ``row[t] < 0`` are padding; rows, positions and pages out of
    range are skipped.  No two tokens of a call may name the same place.
    ``pos`` and ``row`` are int32 on the device."""
    ctx = "paged_write"
    cache, index, heads, dim, rows, _ = _cache(ctx, k_pages, v_pages, table)
    if index != _device():
        return _elsewhere(paged_write, index, k, v, k_pages, v_pages, table, pos, row)
    src = _dtype(ctx, "k", k)
    shape = k.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape or v.dtype is not k.dtype \
            or k.get_device() != index or v.get_device() != index:
        raise ValueError(f"{ctx}: k and v must be [tokens, {heads}, {dim}] of one type on cuda:{index}, not "
                         f"{tuple(shape)} of {k.dtype} on {k.device} and {tuple(v.shape)} of {v.dtype} on {v.device}")
    tokens, ks, vs = shape[0], k.stride(), v.stride()
    if ks[2] != 1 or vs[2] != 1 or (heads > 1 and (ks[1] != dim or vs[1] != dim)):
        raise ValueError(f"{ctx}: a token of k and of v must be contiguous")
    _need(ctx, "pos", pos, _I32, (tokens,), index)
    if row is not None:
        _need(ctx, "row", row, _I32, (tokens,), index)
    rc = lib.focr_paged_write(cache, _pack_write(
        k.data_ptr(), v.data_ptr(), 0 if row is None else row.data_ptr(), pos.data_ptr(), rows, tokens, ks[0], vs[0],
        src), _stream(index))
    if rc != FOCR_OK:
        check(rc)


def paged_attention(q, k_pages, v_pages, table, lens, *, scale: float | None = None, ref_lens=None,
                    window: int = 0, weights=None, out=None):
    """``q`` ``[rows, q_heads, head_dim]`` over each row's first ``lens[row]``
    positions; returns ``[rows, q_heads, head_dim]`` of q's type.  Query head
    ``h`` reads kv head ``h // (q_heads // kv_heads)``; ``scale`` defaults to
    ``1 / sqrt(head_dim)``.  With ``window`` a row sees its first
    ``ref_lens[row]`` and its last ``window`` positions.  ``weights``
    ``[rows, kv_heads, width]`` f32 is added to: every seen position's
    probability, summed over the query heads of its kv head.

    With ``weights`` the call's workspace holds 4 bytes for each of up to 1024 rows,
    each query head and each position of the table or the weights, the narrower of
    them, whatever the lengths.

    A row that sees nothing gives zeros.  Scores that are all -inf, a length past
    the table (or the weights), or a page id outside the pool give NaN for that
    row."""
    ctx = "paged_attention"
    cache, index, kv_heads, dim, rows, pages = _cache(ctx, k_pages, v_pages, table)
    if index != _device():
        return _elsewhere(paged_attention, index, q, k_pages, v_pages, table, lens, scale=scale, ref_lens=ref_lens,
                          window=window, weights=weights, out=out)
    code = _dtype(ctx, "q", q)
    shape, stride = q.shape, q.stride()
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim or q.get_device() != index:
        raise ValueError(f"{ctx}: q must be [{rows}, q_heads, {dim}] on cuda:{index}, "
                         f"not {tuple(shape)} on {q.device}")
    heads = shape[1]
    if stride[2] != 1 or (heads > 1 and stride[1] != dim):
        raise ValueError(f"{ctx}: a row of q must be contiguous")
    if window < 0:
        raise ValueError(f"{ctx}: window must not be negative")
    _need(ctx, "lens", lens, _I32, (rows,), index)
    if ref_lens is not None:
        _need(ctx, "ref_lens", ref_lens, _I32, (rows,), index)
    width = w_row = w_head = 0
    if weights is not None:
        width, w_row, w_head = _weights(ctx, weights, rows, kv_heads, index)
    wide = heads * dim
    if out is None:
        out = _empty((rows, heads, dim), (wide, dim, 1), q.dtype)
    else:
        _need(ctx, "out", out, q.dtype, shape, index)
    need = _workspace("focr_paged_attention_workspace", index, rows, heads, dim, min(width, pages * k_pages.shape[2]))
    ws = _empty((need,), (1,), _U8)  # lives until the kernels are enqueued
    try:
        args = _pack_attention(
            q.data_ptr(), lens.data_ptr(), 0 if ref_lens is None else ref_lens.data_ptr(), out.data_ptr(),
            0 if weights is None else weights.data_ptr(), ws.data_ptr(), rows, heads, stride[0], wide, window, width,
            w_row, w_head, need, code, 1.0 / math.sqrt(dim) if scale is None else scale)
    except (struct.error, OverflowError) as e:
        raise _misfit(ctx, e) from e
    rc = lib.focr_paged_attention(cache, args, _stream(index))
    if rc != FOCR_OK:
        check(rc)
    return out


def paged_evict(k_pages, v_pages, table, lens, weights, new_table, budget: int, *, sink: int = 0,
                recent: int = 0):
    """Shrink every row of more than ``budget`` entries to ``budget``: its first
    ``sink``, its last ``recent`` and, between them, the entries of the largest
    ``weights`` (``[rows, kv_heads, width]`` f32; equal ones: the lower
    position), each kv head for itself.  The kept entries go, in order, to the
    pages of ``new_table`` ``[rows, pages]``, which must differ from one another
    and from every page that a row of this call reads; the old pages are not
    written.

    A length below 0, past the table or past the weights (for which attention gives
    NaN) counts as 0 and leaves an empty row; an entry on a page outside the pool
    becomes NaN.

    Returns ``(kept, lens, weights)``: the old positions ``[rows, kv_heads,
    budget]`` (-1 behind the last), the new lengths, and the kept entries'
    weights in a tensor of ``weights``' shape, 0 behind them."""
    ctx = "paged_evict"
    cache, index, heads, _, rows, _ = _cache(ctx, k_pages, v_pages, table)
    if index != _device():
        return _elsewhere(paged_evict, index, k_pages, v_pages, table, lens, weights, new_table, budget, sink=sink,
                          recent=recent)
    _need(ctx, "lens", lens, _I32, (rows,), index)
    width, w_row, w_head = _weights(ctx, weights, rows, heads, index)
    new_rows, new_pages, new_step = _table(ctx, "new_table", new_table, index)
    if new_rows != rows:
        raise ValueError(f"{ctx}: new_table has {new_rows} rows, table {rows}")
    if budget < 1 or sink < 0 or recent < 0:
        raise ValueError(f"{ctx}: budget must be positive, sink and recent not negative")
    if budget > new_pages * k_pages.shape[2]:
        raise ValueError(f"{ctx}: the new pages hold fewer entries than the budget")
    kept = _empty((rows, heads, budget), (heads * budget, budget, 1), _I32)
    new_lens = _empty((rows,), (1,), _I32)
    new_weights = _empty((rows, heads, width), (heads * width, width, 1), _F32)
    try:
        args = _pack_evict(
            lens.data_ptr(), weights.data_ptr(), new_table.data_ptr(), kept.data_ptr(), new_lens.data_ptr(),
            new_weights.data_ptr(), rows, width, w_row, w_head, new_step, new_pages, budget, sink, recent)
    except (struct.error, OverflowError) as e:
        raise _misfit(ctx, e) from e
    rc = lib.focr_paged_evict(cache, args, _stream(index))
    if rc != FOCR_OK:
        check(rc)
    return kept, new_lens, new_weights
