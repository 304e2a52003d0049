"""Beam search beside the greedy ``argmax_row`` (sampler.rs:168-186):

* ``beam_select`` -- the best continuations over beams and vocabulary, from the
  lm-head's logits;
* ``beam_reorder`` -- every beam gets its parent's paged cache.

CUDA tensors on one device, torch's current stream; both can be captured, and
no gradient passes through them.
"""
from __future__ import annotations

import struct

import torch

from ._lib import FOCR_OK, BeamReorderArgs, BeamSelectArgs, check, lib
from .paged import _F32, _I32, _U8, _cache, _device, _dtype, _elsewhere, _empty, _misfit, _need, _packer, _stream, _workspace

_pack_select = _packer(BeamSelectArgs, "13Nii")
_pack_reorder = _packer(BeamReorderArgs, "15N")


def beam_select(logits, scores, n: int | None = None, *, done=None, end_token: int = 1):
    """From ``logits`` ``[batch, beams, vocab]`` (f32, f16 or bf16) and the beams'
    cumulated log probabilities ``scores`` ``[batch, beams]`` f32: the ``n`` (by
    default ``beams``) best continuations of every entry as ``(scores, parent,
    token)``, each ``[batch, n]``, best first.  ``beams`` and ``n`` are at most 64.

    A candidate's score is ``scores[b, i] + log_softmax(logits[b, i])[t]``, held
    in 64 bits for the ranking, of which a beam's log-sum is good to 2^-27 (the
    same for the same logits); equal ones go to the lower beam, then the larger
    logit, then the lower token.  A beam with ``done[b, i]`` offers ``end_token``
    alone with its score unchanged; -inf and NaN logits and beams with a score
    that is not finite offer nothing.  Missing candidates: -inf, -1, -1."""
    ctx = "beam_select"
    shape, stride = logits.shape, logits.stride()
    if len(shape) != 3:
        raise ValueError(f"{ctx}: logits must be [batch, beams, vocab], not {tuple(shape)}")
    index = logits.get_device()
    if index < 0:
        raise ValueError(f"{ctx}: logits must be a CUDA tensor, not on {logits.device}")
    if index != _device():
        return _elsewhere(beam_select, index, logits, scores, n, done=done, end_token=end_token)
    code = _dtype(ctx, "logits", logits)
    batch, beams, vocab = shape
    if (stride[2] != 1 and vocab > 1) or (batch > 1 and beams > 1 and stride[0] != beams * stride[1]):
        raise ValueError(f"{ctx}: the rows of logits must be contiguous and evenly spaced")
    _need(ctx, "scores", scores, _F32, (batch, beams), index)
    if done is not None:
        if done.dtype is torch.bool:
            done = done.view(_U8)
        _need(ctx, "done", done, _U8, (batch, beams), index)
    if n is None:
        n = beams
    if n < 1:
        raise ValueError(f"{ctx}: n must be positive")
    need = _workspace("focr_beam_select_workspace", index, batch, beams, vocab, n)
    shape = (batch, n)
    out, parent, token = _empty(shape, (n, 1), _F32), _empty(shape, (n, 1), _I32), _empty(shape, (n, 1), _I32)
    ws = _empty((need,), (1,), _U8)  # lives until the kernels are enqueued
    row = stride[1] if beams > 1 else stride[0] if batch > 1 else vocab
    try:
        args = _pack_select(
            logits.data_ptr(), scores.data_ptr(), 0 if done is None else done.data_ptr(), out.data_ptr(),
            parent.data_ptr(), token.data_ptr(), ws.data_ptr(), batch, beams, vocab, row, n, need, code, end_token)
    except (struct.error, OverflowError) as e:
        raise _misfit(ctx, e) from e
    rc = lib.focr_beam_select(args, _stream(index))
    if rc != FOCR_OK:
        check(rc)
    return out, parent, token


def beam_reorder(k_pages, v_pages, table, lens, parent, fresh, *, weights=None):
    """Row ``i`` of entry ``b = i // beams`` becomes row ``b * beams + parent[b,
    i % beams]`` of ``table`` ``[batch * beams, max_pages]``: full pages are
    shared, the partly filled one is copied to page ``fresh[i]`` (which takes its
    place also where it is still empty), in every layer of ``k_pages`` /
    ``v_pages`` ``[layers, pages, kv_heads, page_size, head_dim]`` (or one layer,
    without the first dimension).  ``weights`` ``[layers, rows, kv_heads, width]``
    f32 (without the first dimension for one layer) follow.

    Returns ``(table, lens, weights or None)``, new tensors.  A parent outside
    ``[0, beams)`` leaves an empty row, as does a length past the table; a partly
    filled page outside the pool stays missing (-1).  The fresh pages must differ from one
    another and from every page the table uses."""
    ctx = "beam_reorder"
    layered = k_pages.dim() == 5
    cache, index, heads, _, rows, width = _cache(ctx, k_pages, v_pages, table, 5 if layered else 4)
    if index != _device():
        return _elsewhere(beam_reorder, index, k_pages, v_pages, table, lens, parent, fresh, weights=weights)
    layers = k_pages.shape[0] if layered else 1
    if parent.dim() != 2:
        raise ValueError(f"{ctx}: parent must be [batch, beams], not {tuple(parent.shape)}")
    batch, beams = parent.shape
    if batch * beams != rows:
        raise ValueError(f"{ctx}: table has {rows} rows for {batch} x {beams} beams")
    _need(ctx, "parent", parent, _I32, (batch, beams), index)
    _need(ctx, "lens", lens, _I32, (rows,), index)
    _need(ctx, "fresh", fresh, _I32, (rows,), index)
    w_out, span, w_layer, w_row, w_head = None, 0, 0, 0, 0
    if weights is not None:
        lead = (layers, rows, heads) if layered else (rows, heads)
        shape, stride = weights.shape, weights.stride()
        if weights.dtype is not _F32:
            raise TypeError(f"{ctx}: weights must be torch.float32, not {weights.dtype}")
        if shape[:-1] != lead or weights.get_device() != index:
            raise ValueError(f"{ctx}: weights must be {list(lead)} + [width] on cuda:{index}, "
                             f"not {tuple(shape)} on {weights.device}")
        span, w_row, w_head = shape[-1], stride[-3], stride[-2]
        if stride[-1] != 1 and span > 1:
            raise ValueError(f"{ctx}: the last dimension of weights must be contiguous")
        w_layer = stride[0] if layered else 0
        wide = rows * heads * span
        w_out = _empty(tuple(shape), (wide, heads * span, span, 1)[0 if layered else 1:], _F32)
    new_table = _empty((rows, width), (width, 1), _I32)
    new_lens = _empty((rows,), (1,), _I32)
    rc = lib.focr_beam_reorder(cache, _pack_reorder(
        lens.data_ptr(), parent.data_ptr(), fresh.data_ptr(), new_table.data_ptr(), new_lens.data_ptr(),
        0 if weights is None else weights.data_ptr(), 0 if w_out is None else w_out.data_ptr(), layers,
        k_pages.stride(0) if layered else 0, batch, beams, span, w_layer, w_row, w_head), _stream(index))
    if rc != FOCR_OK:
        check(rc)
    return new_table, new_lens, w_out
