"""Refusals of the paged-cache and beam calls, without a GPU: every check runs
before any device work."""
import ctypes as C

import pytest

from franken_ocr_b200._lib import (BF16, F16, F32, BeamReorderArgs, BeamSelectArgs, FocrError, PagedAttentionArgs,
                                   PagedCache, PagedEvictArgs, PagedWriteArgs, check, lib)

PTR = 1 << 20  # never read: the calls refuse first


def cache(**kw):
    d = dict(k=PTR, v=PTR, table=PTR, page_stride=2 * 16 * 64, head_stride=16 * 64, table_stride=4, n_pages=10,
             kv_heads=2, page_size=16, head_dim=64, max_pages=4, dtype=F32)
    d.update(kw)
    return PagedCache(*[d[n] for n, _ in PagedCache._fields_])


def write(c, rows=4, k=PTR, v=PTR, src=F32, tokens=4, ks=128, vs=128, row=None, pos=PTR):
    check(lib.focr_paged_write(C.byref(c) if c else None, C.byref(PagedWriteArgs(k, v, row, pos, rows, tokens, ks, vs,
                                                                                 src)), None))


def attend(c, q=PTR, qt=F32, rows=4, heads=4, qs=256, lens=PTR, refs=None, window=0, scale=0.125, out=2 * PTR, os=256,
           w=None, ww=0, wr=0, wh=0, ws=PTR, wsb=1 << 40):
    check(lib.focr_paged_attention(C.byref(c), C.byref(PagedAttentionArgs(
        q, lens, refs, out, w, ws, rows, heads, qs, os, window, ww, wr, wh, wsb, qt, scale)), None))


def evict(c, rows=2, lens=PTR, w=PTR, width=64, wr=128, wh=64, into=2 * PTR, is_=4, ip=4, budget=32, sink=4, recent=8,
          kept=PTR, lo=3 * PTR, wo=2 * PTR):
    check(lib.focr_paged_evict(C.byref(c), C.byref(PagedEvictArgs(lens, w, into, kept, lo, wo, rows, width, wr, wh, is_,
                                                                  ip, budget, sink, recent)), None))


def select(x=PTR, dt=F32, batch=2, beams=4, vocab=100, stride=100, scores=PTR, n=4, out=PTR, ws=PTR, wsb=1 << 30):
    check(lib.focr_beam_select(C.byref(BeamSelectArgs(x, scores, None, out, out, out, ws, batch, beams, vocab, stride, n,
                                                      wsb, dt, 1)), None))


def reorder(c, layers=2, ls=10 * 2 * 16 * 64, batch=2, beams=2, lens=PTR, parent=PTR, fresh=PTR, to=2 * PTR, lo=3 * PTR,
            w=None, width=0, wl=0, wr=0, wh=0, wo=None):
    check(lib.focr_beam_reorder(C.byref(c), C.byref(BeamReorderArgs(lens, parent, fresh, to, lo, w, wo, layers, ls, batch,
                                                                    beams, width, wl, wr, wh)), None))


@pytest.mark.parametrize("bad,code,text", [
    (dict(dtype=3), -2, "unknown cache type 3"), (dict(n_pages=0), -1, "empty dimension"),
    (dict(page_size=0), -1, "empty dimension"), (dict(head_dim=0), -1, "empty dimension"),
    (dict(max_pages=0), -1, "empty dimension"), (dict(kv_heads=0), -1, "empty dimension"),
    (dict(head_dim=260, head_stride=16 * 260, page_stride=32 * 260), -7, "head_dim 260"),
    (dict(head_dim=62), -7, "head_dim 62"), (dict(head_dim=68, dtype=BF16), -7, "head_dim 68"),
    (dict(max_pages=1 << 27, table_stride=1 << 27), -7, "max_pages * page_size"),
    (dict(max_pages=(1 << 27) - 4095, table_stride=1 << 27), -7, "max_pages * page_size"),
    (dict(page_stride=2049), -7, "multiples of 16"), (dict(head_stride=1023 * 4, dtype=F16), -7, "multiples of 16"),
    (dict(head_stride=512), -1, "shorter than"), (dict(page_stride=512), -1, "shorter than"),
    (dict(page_stride=1 << 62), -1, "stride overflow"), (dict(table_stride=3), -1, "table_stride 3 < max_pages 4"),
    (dict(k=None), -2, "null pointer"), (dict(v=None), -2, "null pointer"), (dict(table=None), -2, "null pointer"),
    (dict(k=PTR + 8), -2, "16-byte aligned"), (dict(v=PTR + 4), -2, "16-byte aligned"),
    (dict(n_pages=1 << 31), -7, "int32"),
])
def test_every_call_checks_its_cache(bad, code, text):
    if "head_stride" in bad and bad.get("dtype") == F16:
        bad = dict(bad, head_stride=1025)
    for call, name in ((write, "paged_write"), (attend, "paged_attention"), (evict, "paged_evict"),
                       (reorder, "beam_reorder")):
        with pytest.raises(FocrError) as e:
            call(cache(**bad))
        assert e.value.code == code and text in str(e.value) and str(e.value).startswith(name)


def test_null_cache_and_arguments():
    with pytest.raises(FocrError, match="paged_write: null cache"):
        write(None)
    c = cache()
    for name in ("paged_write", "paged_attention", "paged_evict", "beam_reorder"):
        with pytest.raises(FocrError, match=name + ": null arguments"):
            check(getattr(lib, "focr_" + name)(C.byref(c), None, None))
    with pytest.raises(FocrError, match="beam_select: null arguments"):
        check(lib.focr_beam_select(None, None))


@pytest.mark.parametrize("bad,code,text", [
    (dict(src=7), -2, "unknown source type 7"), (dict(k=None), -2, "null"), (dict(pos=None), -2, "null"),
    (dict(tokens=5), -1, "5 tokens without rows for a table of 4"), (dict(ks=127), -1, "token stride"),
    (dict(vs=1 << 62), -1, "overflow"),
])
def test_write_refusals(bad, code, text):
    with pytest.raises(FocrError) as e:
        write(cache(), **bad)
    assert e.value.code == code and text in str(e.value)


@pytest.mark.parametrize("bad,code,text", [
    (dict(qt=-1), -2, "unknown query type"), (dict(heads=3), -1, "3 query heads over 2 kv heads"),
    (dict(heads=0), -1, "0 query heads"), (dict(scale=0.0), -2, "scale"), (dict(scale=-1.0), -2, "scale"),
    (dict(scale=float("nan")), -2, "scale"), (dict(scale=3e38), -2, "scale"), (dict(out=PTR), -2, "out must not be q"), (dict(scale=float("inf")), -2, "scale"), (dict(q=None), -2, "null"),
    (dict(lens=None), -2, "null"), (dict(out=None), -2, "null"), (dict(ws=None), -2, "null"),
    (dict(qs=255), -1, "row stride"), (dict(os=255), -1, "row stride"), (dict(wsb=100), -2, "workspace needs"),
    (dict(ws=PTR + 8), -2, "workspace needs"), (dict(w=PTR, ww=0, wr=10, wh=10), -1, "weights_width"),
    (dict(w=PTR, ww=10, wr=10, wh=9), -1, "weights stride"), (dict(w=PTR, ww=10, wr=9, wh=10), -1, "weights stride"),
])
def test_attention_refusals(bad, code, text):
    with pytest.raises(FocrError) as e:
        attend(cache(), **bad)
    assert e.value.code == code and text in str(e.value)


@pytest.mark.parametrize("bad,code,text", [
    (dict(budget=0, sink=0, recent=0), -1, "over budget 0"), (dict(sink=30, recent=3), -1, "sink 30 + recent 3"),
    (dict(sink=33), -1, "sink 33"), (dict(lens=None), -2, "null"), (dict(wo=None), -2, "null"),
    (dict(budget=65), -1, "fewer entries than the budget"), (dict(is_=3), -1, "fewer entries"),
    (dict(wh=63), -1, "weights stride"), (dict(wr=63), -1, "weights stride"), (dict(width=0), -1, "weights stride"),
    (dict(wo=PTR), -2, "must not be weights"), (dict(into=PTR), -2, "must not be the old ones"),
    (dict(lo=PTR), -2, "must not be lens"), (dict(rows=70000), -7, "out of range"),
])
def test_evict_refusals(bad, code, text):
    with pytest.raises(FocrError) as e:
        evict(cache(), **bad)
    assert e.value.code == code and text in str(e.value)


@pytest.mark.parametrize("bad,code,text", [
    (dict(dt=9), -2, "unknown logits type 9"), (dict(beams=0), -1, "must not be 0"), (dict(vocab=0), -1, "must not be 0"),
    (dict(n=0), -1, "must not be 0"), (dict(n=65), -7, "at most 64"), (dict(beams=65), -7, "at most 64"),
    (dict(batch=20000), -7, "65535 rows"), (dict(vocab=2**31, stride=2**31), -7, "vocab"), (dict(stride=99), -1, "row_stride 99"),
    (dict(x=None), -2, "null"), (dict(ws=None), -2, "null"), (dict(wsb=8), -2, "workspace needs"),
    (dict(stride=1 << 62), -1, "overflow"),
])
def test_select_refusals(bad, code, text):
    with pytest.raises(FocrError) as e:
        select(**bad)
    assert e.value.code == code and text in str(e.value)


@pytest.mark.parametrize("bad,code,text", [
    (dict(beams=0), -1, "must not be 0"), (dict(layers=0), -1, "must not be 0"), (dict(lens=None), -2, "null"),
    (dict(fresh=None), -2, "null"), (dict(to=PTR), -2, "must not be the inputs"), (dict(lo=PTR), -2, "must not be the inputs"),
    (dict(ls=100), -1, "layer stride"), (dict(ls=10 * 2 * 16 * 64 + 1), -1, "layer stride"),
    (dict(batch=70000), -7, "out of range"), (dict(w=PTR, width=8, wl=99, wr=16, wh=8), -2, "weights_out"),
    (dict(w=PTR, wo=PTR, width=8, wl=99, wr=16, wh=8), -2, "weights_out"),
    (dict(w=PTR, wo=2 * PTR, width=8, wl=99, wr=16, wh=7), -1, "weights stride"),
])
def test_reorder_refusals(bad, code, text):
    with pytest.raises(FocrError) as e:
        reorder(cache(), **bad)
    assert e.value.code == code and text in str(e.value)


def test_nothing_to_do_is_no_error():
    c = cache(table=None)
    write(c, rows=0, tokens=0)
    attend(c, rows=0)
    evict(c, rows=0)
    select(batch=0)
    reorder(c, batch=0)


def test_workspaces_grow_with_their_calls():
    def size(f, *a):
        n = C.c_size_t()
        check(getattr(lib, f)(*a, C.byref(n)))
        return n.value

    assert size("focr_beam_select_workspace", 1, 4, 129280, 4) > size("focr_beam_select_workspace", 1, 1, 1, 1) > 0
    with pytest.raises(FocrError):
        size("focr_beam_select_workspace", 1, 4, 100, 65)
    with pytest.raises(FocrError):
        size("focr_paged_attention_workspace", 1 << 40, 1 << 20, 128, 1 << 20)


@pytest.mark.parametrize("beams,n", [(4, 65), (33, 66), (65, 4)])
def test_select_workspace_names_the_limit(beams, n):
    """It is what the Python call asks first."""
    with pytest.raises(FocrError, match=f"at most 64, not {beams} and {n}") as e:
        check(lib.focr_beam_select_workspace(1, beams, 1000, n, C.byref(C.c_size_t())))
    assert e.value.code == -7


def test_attention_workspace_holds_the_rows_of_one_launch():
    """Rows past 1024 go in launches of their own, one behind the other."""
    def size(rows):
        n = C.c_size_t()
        check(lib.focr_paged_attention_workspace(rows, 8, 128, 4096, C.byref(n)))
        return n.value

    assert size(1023) < size(1024) == size(1025) == size(100000)


def test_workspace_sizes_are_kept_for_each_device(monkeypatch):
    """They go by the device's SMs: one device's size is not another's."""
    from types import SimpleNamespace

    from franken_ocr_b200 import paged

    current = 0

    def query(rows, out):
        out._obj.value = rows * (148 if current == 0 else 20)
        return 0

    monkeypatch.setattr(paged, "lib", SimpleNamespace(focr_query=query))
    paged._workspace.cache_clear()
    try:
        assert paged._workspace("focr_query", 0, 3) == 3 * 148
        current = 1
        assert paged._workspace("focr_query", 1, 3) == 3 * 20
        assert paged._workspace("focr_query", 0, 3) == 3 * 148
    finally:
        paged._workspace.cache_clear()


def test_public_torch_calls_stand_in_for_missing_short_cuts(monkeypatch):
    """Without torch's internal calls, or with others of that name, the public ones serve."""
    import subprocess
    import sys
    from pathlib import Path

    import torch

    from franken_ocr_b200 import paged

    code = ("import sys, types, torch\n"
            "del torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream\n"
            "sys.modules['torch._C._dynamo.guards'] = types.ModuleType('guards')\n"
            "from franken_ocr_b200 import beam, paged\n"
            "assert paged._device is torch.cuda.current_device and paged._quick_empty is None\n"
            "torch.cuda.current_stream = lambda i: types.SimpleNamespace(cuda_stream=70 + i)\n"
            "assert paged._stream(3) == 73\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=Path(paged.__file__).parents[1])
    seen = []
    monkeypatch.setattr(torch, "empty_strided", lambda *a, **k: seen.append((a, k)))
    for quick in (None, lambda shape: None):
        monkeypatch.setattr(paged, "_quick_empty", quick)
        paged._empty((2, 3), (3, 1), torch.float32)
    assert seen == [(((2, 3), (3, 1)), dict(dtype=torch.float32, device="cuda"))] * 2


def test_python_checks_types_shapes_and_devices():
    import torch

    from franken_ocr_b200 import beam, paged

    k = torch.zeros((4, 2, 16, 64))
    t = torch.zeros((1, 2), dtype=torch.int32)
    n = torch.zeros((1,), dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        paged.paged_attention(torch.zeros((1, 2, 64)), k, k, t, n)
    with pytest.raises(ValueError, match="CUDA tensors"):
        paged.paged_write(torch.zeros((1, 2, 64)), torch.zeros((1, 2, 64)), k, k, t, n)
    with pytest.raises(ValueError, match="CUDA tensors"):
        paged.paged_evict(k, k, t, n, torch.zeros((1, 2, 32)), t, 4)
    with pytest.raises(ValueError, match="CUDA tensors"):
        beam.beam_reorder(k, k, t, n, n.view(1, 1), n)
    with pytest.raises(ValueError, match="CUDA tensor"):
        beam.beam_select(torch.zeros((1, 1, 5)), torch.zeros((1, 1)))
