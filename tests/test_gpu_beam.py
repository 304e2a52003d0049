"""Beam selection and reordering on the GPU against their definitions in 64 bits."""
import math

import pytest
import torch

from tests.paged_cases import DTYPES, Cache, select
from tests.test_gpu_paged import same_bits, stale_memory  # noqa: F401

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("stale_memory")]


def check_select(logits, scores, n, done=None, end=1, dev=None):
    from franken_ocr_b200 import beam

    x = logits.cuda() if dev is None else dev
    got = beam.beam_select(x, scores.cuda(), n, done=None if done is None else done.cuda(), end_token=end)
    score, parent, token = (t.cpu() for t in got)
    for b, want in enumerate(select(logits, scores, n, done, end)):
        for k in range(n):
            if k >= len(want):
                assert (float(score[b, k]), int(parent[b, k]), int(token[b, k])) == (-math.inf, -1, -1)
                continue
            s, i, t = want[k]
            assert (int(parent[b, k]), int(token[b, k])) == (i, t), (b, k)
            # one rounding to f32; the 64-bit sum's own error lies far below it
            assert abs(float(score[b, k]) - s) <= 2.0 ** -24 * abs(s) * 1.001 + 1e-12 or math.isinf(float(score[b, k]))
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch,beams,vocab,n", [(1, 1, 1, 1), (1, 1, 129280, 1), (2, 4, 1000, 4), (3, 5, 8193, 10),
                                                 (1, 16, 32, 32), (2, 3, 5, 20), (1, 64, 700, 64), (5, 2, 50001, 3)])
def test_select_matches_the_definition(cuda, dtype, batch, beams, vocab, n):
    g = torch.Generator().manual_seed(vocab + n)
    x = (torch.randn((batch, beams, vocab), generator=g) * 3).to(DTYPES[dtype])
    check_select(x, torch.randn((batch, beams), generator=g) * 2 - 10, n)


def test_select_equals_argmax_for_one_beam(cuda):
    from franken_ocr_b200 import beam

    x = torch.randn((6, 1, 4000), generator=torch.Generator().manual_seed(1)).half().cuda()
    _, parent, token = beam.beam_select(x, torch.zeros((6, 1), device="cuda"))
    assert token[:, 0].tolist() == x.float().cpu().argmax(-1)[:, 0].tolist() and bool((parent == 0).all())


def test_select_ties_masks_and_values_that_are_no_numbers(cuda):
    g = torch.Generator().manual_seed(3)
    low = float(torch.finfo(torch.float32).min)
    x = torch.randn((8, 4, 9000), generator=g)
    x[0] = 0.0                                      # everything equal
    x[1] = x[1].round()                             # many ties
    x[2, :, :] = -math.inf                          # rows with nothing left
    x[2, 1, 8999] = 1.0
    x[3, 0] = low                                   # masked by the type's lowest value
    x[3, 1, 1:] = low
    x[4, :2] = math.nan
    x[4, 2, ::3] = math.nan
    x[5, 0, 17] = x[5, 0, 8500] = math.inf
    x[6] = x[6, :1].expand(4, -1)                   # equal beams
    x[7, 3, :] = 80.0 * (x[7, 3] > 3)               # a steep row
    scores = torch.randn((8, 4), generator=g) - 5
    scores[1] = scores[1, 0]
    scores[6] = -1.5
    scores[7, 1:3] = torch.tensor([-math.inf, math.nan])
    scores[3, 2] = -1e9                             # a beam as good as dead
    for n in (4, 8, 64):
        check_select(x, scores, n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_select_many_ties_beside_values_that_are_no_numbers(cuda, dtype):
    """More equal logits in a strip than are listed, with NaN, -inf or +inf among them."""
    x = torch.zeros((4, 2, 20000))
    x[0, :, 5] = math.nan
    x[1, :, ::3] = math.nan
    x[2, 0, 7::2] = -math.inf
    x[2, 1, 16000:] = math.nan
    x[3, 0, 2000:9000] = math.inf
    x[3, 0, 3] = math.nan
    scores = torch.tensor([-1.0, -1.25]).expand(4, 2).contiguous()
    for n in (1, 6):
        check_select(x.to(DTYPES[dtype]), scores, n)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_select_lowest_value_of_small_types(cuda, dtype):
    t = DTYPES[dtype]
    x = torch.full((2, 3, 500), torch.finfo(t).min, dtype=t)
    x[0, 1, 77] = 2.0
    x[1, 2, 5] = torch.finfo(t).max
    check_select(x, torch.zeros((2, 3)) - 1, 6)


def test_select_close_scores_of_different_beams(cuda):
    """Scores that differ by less than f32 resolves are still ranked rightly."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn((1, 2, 30000), generator=g) * 2
    p = torch.log_softmax(x.double(), -1).amax(-1)[0]
    scores = torch.tensor([[-40.0, 0.0]])
    for step in (-1, 1):
        scores[0, 1] = torch.nextafter((scores[0, 0].double() + p[0] - p[1]).float(), torch.tensor(step * 1e9))
        check_select(x, scores, 4)


@pytest.mark.parametrize("at", [1.0, -900.0, 1023.5, 5000.0, -70000.0, 1e12, -3e38])
def test_select_logits_far_from_zero(cuda, at):
    """Log probabilities do not depend on where the logits lie."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn((2, 3, 5000), generator=g) * 3 + at
    check_select(x, torch.randn((2, 3), generator=g), 6)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["first", "last", "rising", "falling", "alone", "tied"])
def test_select_beams_far_ahead_of_the_others(cuda, dtype, kind):
    """The best lists hold nearly all that is chosen: more candidates reach the other
    lists' best than are ranked at a time."""
    beams, n = 64, 64
    g = torch.Generator().manual_seed(21)
    x = torch.randn((2, beams, 20000), generator=g).to(DTYPES[dtype])
    cum = torch.full((2, beams), -40.0)
    if kind == "first":
        cum[:, 0] = -1.0
    elif kind == "last":
        cum[:, 60:] = torch.tensor([-3.0, -1.0, -2.0, -2.5])
    elif kind == "rising":
        cum = -70 + torch.arange(beams).float().expand(2, beams) * 0.25
    elif kind == "falling":
        cum = -torch.arange(beams).float().expand(2, beams) * 0.25
    elif kind == "alone":
        cum[:] = -math.inf
        cum[0, 5] = cum[1, 63] = 0.0
    else:
        x[:] = x[:, :1]
        x[:, :, 10:] = 0.0
    check_select(x, cum.contiguous(), n)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 7, 5000, 20001])
def test_select_ties_of_beams_whose_sums_are_whole_numbers(cuda, dtype, vocab):
    """Beams that leave one token, or equal ones, wherever those logits lie: their scores
    are equal, and equal ones go to the lower beam."""
    beams = 16
    g = torch.Generator().manual_seed(vocab)
    at = (torch.randn((beams, 1), generator=g) * 20).to(DTYPES[dtype])
    x = torch.full((4, beams, vocab), -math.inf, dtype=DTYPES[dtype])
    x[0] = at                                           # all equal
    x[1, :, vocab // 2] = at[:, 0]                      # one token
    x[2, :, ::3] = at                                   # a third of them
    x[3] = torch.finfo(DTYPES[dtype]).min               # masked by the lowest value
    x[3, :, vocab // 2] = at[:, 0]
    for n in (1, 5, 40):
        check_select(x, torch.full((4, beams), -3.0), n)


def flat_beam(value, vocab):
    """A logit 0 every thousand, all others `value`: their exponentials are all rounded
    alike, and lie below the largest wherever a strip begins."""
    x = torch.full((vocab,), value)
    x[300::1000] = 0.0
    return x


def near_the_score(score, want):
    """One rounding to f32, and what a term of the sum may be off by: of its 2^(s + k / 16),
    |s| <= 1/32, s has two roundings of half a step, 2^-30, each ln 2 of that in the term;
    2^s - 1 < 2^-5 has one of 2^-25 in its factor of s and one of 2^-30; four terms are
    added up with three of 2^-25 of 2^-5.5: 2^-27.5 together."""
    if math.isinf(want):
        return float(score) == want
    half = math.ldexp(1.0, math.frexp(want)[1] - 25) if want else 0.0
    return abs(float(score) - want) <= half + 2.0 ** -27.5


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [-0.03125, -0.99, -1.01, -1.3, -2.0, -2.71875, -3.0, -5.0, -9.5, -20.0])
def test_select_sums_of_repeated_logits(cuda, dtype, value):
    """A flat tail, as padding or masks by one value leave it, far from zero too."""
    from franken_ocr_b200 import beam

    for vocab, at in ((129280, 0.0), (40000, 0.0), (129280, 640.0), (5000, -1536.0)):
        x = (flat_beam(value, vocab) + at).to(DTYPES[dtype])[None, None]
        score, _, token = (t.cpu() for t in beam.beam_select(x.cuda(), torch.zeros((1, 1), device="cuda"), 3))
        want = select(x, torch.zeros((1, 1)), 3)[0]
        assert token[0].tolist() == [t for _, _, t in want]
        for k in range(3):
            assert near_the_score(score[0, k], want[k][0]), (vocab, at, float(score[0, k]) - want[k][0])


def test_select_scores_are_infinite_only_where_due(cuda):
    """Masks by the lowest value, +inf logits and beams as good as dead: finite scores
    stay finite, and what lies past f32 is -inf."""
    from franken_ocr_b200 import beam

    g = torch.Generator().manual_seed(12)
    x = torch.randn((5, 3, 9000), generator=g)
    low = float(torch.finfo(torch.float32).min)
    x[0, 1, 4:] = low
    x[1, 0, 17] = x[1, 2, 8500] = math.inf
    x[2, 1] = -math.inf
    x[2, 2, 1:] = -math.inf
    x[3, :, 2:] = -math.inf
    scores = torch.randn((5, 3), generator=g) - 5
    scores[0, 0] = low
    scores[4, 1] = -1e38
    for n in (3, 40):
        got, parent, token = (t.cpu() for t in beam.beam_select(x.cuda(), scores.cuda(), n))
        for b, want in enumerate(select(x, scores, n)):
            for k, (s, i, t) in enumerate(want):
                assert (int(parent[b, k]), int(token[b, k])) == (i, t)
                assert near_the_score(got[b, k], float(torch.tensor(s, dtype=torch.float64).float()) if abs(s) > 1e30 else s)
            assert got[b, len(want):].tolist() == [-math.inf] * (n - len(want))


@pytest.mark.parametrize("value", [-1.01, -1.3, -2.0, -2.71875, -3.0, -5.0, -9.5])
def test_select_ranks_a_flat_beam_and_an_exact_one(cuda, value):
    """Two beams whose scores differ by 1e-8 to 5e-8, either way: a flat tail of f32 terms
    against a beam of equal logits, whose sum is a whole number."""
    from franken_ocr_b200 import beam

    vocab = 129280
    x = torch.full((2, 2, vocab), -math.inf)
    x[0, 0] = flat_beam(value, vocab)
    x[0, 1, :max(1, round(float(x[0, 0].double().exp().sum())))] = 0.0
    x[1] = x[0].flip(0)
    norm = torch.logsumexp(x.double(), -1)
    for gap in (-5e-8, -2e-8, -1e-8, 1e-8, 2e-8, 5e-8):
        # the second beam's best score is `gap` above the first one's
        scores = torch.zeros((2, 2))
        scores[:, 1] = (norm[:, 1] - norm[:, 0] + gap).float()
        best = scores.double() - norm
        # scores below 0.05 in f32: the gap is met to 2^-29
        assert bool(((best[:, 1] - best[:, 0] - gap).abs() < 2.0 ** -29).all()), best
        got, parent, _ = beam.beam_select(x.cuda(), scores.cuda(), 1)
        assert parent[:, 0].tolist() == [int(gap > 0)] * 2, gap
        for b in range(2):
            assert near_the_score(got[b, 0], float(best[b].max()))


def test_select_probabilities_add_up(cuda):
    """Flat, steep and mixed rows: exp of the scores of a whole small vocabulary is 1."""
    from franken_ocr_b200 import beam

    g = torch.Generator().manual_seed(9)
    for scale in (0.0, 1e-3, 1.0, 30.0):
        x = (torch.randn((1, 1, 64), generator=g) * scale).cuda()
        score, _, _ = beam.beam_select(x, torch.zeros((1, 1), device="cuda"), 64)
        assert abs(float(score.double().exp().sum()) - 1) <= 64 * 2.0 ** -23   # each rounded to f32


@pytest.mark.parametrize("kind", ["bool", "uint8"])
def test_select_ended_beams(cuda, kind):
    g = torch.Generator().manual_seed(5)
    x = torch.randn((4, 3, 600), generator=g)
    done = torch.tensor([[0, 1, 0], [1, 1, 1], [0, 0, 0], [1, 0, 1]]).to(getattr(torch, kind))
    x[3, 0] = math.nan                               # an ended beam's logits do not matter
    scores = torch.randn((4, 3), generator=g) - 3
    scores[0, 1] = 0.0
    for n in (1, 3, 7):
        check_select(x, scores, n, done, end=37)


def test_select_strided_and_unaligned_rows(cuda):
    g = torch.Generator().manual_seed(6)
    for dtype in DTYPES.values():
        wide = torch.randn((2, 3, 5011), generator=g).to(dtype)
        dev = wide.cuda()
        check_select(wide[:, :, 5:5008], torch.zeros((2, 3)), 5, dev=dev[:, :, 5:5008])
        one = torch.randn((4, 1, 333), generator=g).to(dtype)
        check_select(one, torch.zeros((4, 1)), 2)
        # one beam an entry, entries apart
        apart = torch.randn((4, 3, 333), generator=g).to(dtype)
        check_select(apart[:, 1:2], torch.zeros((4, 1)), 2, dev=apart.cuda()[:, 1:2])


def test_broadcast_inputs_are_refused(cuda):
    """An expanded tensor has no rows of its own to read."""
    from franken_ocr_b200 import beam, paged
    from franken_ocr_b200._lib import FocrError

    x = torch.randn((1, 1, 50), device="cuda")
    with pytest.raises(FocrError, match="row_stride 0"):
        beam.beam_select(x.expand(1, 4, 50), torch.zeros((1, 4), device="cuda"))
    with pytest.raises(FocrError, match="row_stride 0"):
        beam.beam_select(x.expand(4, 1, 50), torch.zeros((4, 1), device="cuda"))
    kp = torch.zeros((4, 1, 16, 64), device="cuda")
    table = torch.zeros((1, 2), dtype=torch.int32, device="cuda").expand(3, 2)
    lens = torch.ones((3,), dtype=torch.int32, device="cuda")
    with pytest.raises(FocrError, match="table_stride 0"):
        paged.paged_attention(torch.zeros((3, 1, 64), device="cuda"), kp, kp, table, lens)
    with pytest.raises(FocrError, match="shorter"):
        paged.paged_attention(torch.zeros((3, 2, 64), device="cuda"), kp.expand(4, 2, 16, 64), kp.expand(4, 2, 16, 64),
                              table.contiguous(), lens)
    with pytest.raises(FocrError, match="weights stride"):
        paged.paged_attention(torch.zeros((3, 1, 64), device="cuda"), kp, kp, table.contiguous(), lens,
                              weights=torch.zeros((1, 1, 32), device="cuda").expand(3, 1, 32))


def test_select_in_a_graph_and_twice_the_same(cuda):
    from franken_ocr_b200 import beam

    g = torch.Generator().manual_seed(7)
    x = torch.randn((3, 4, 20000), generator=g).cuda()
    s = torch.randn((3, 4), generator=g).cuda()
    want = beam.beam_select(x, s, 8)
    graph = torch.cuda.CUDAGraph()
    held = x.clone()
    with torch.cuda.graph(graph):
        got = beam.beam_select(held, s, 8)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(same_bits(a, b) for a, b in zip(got, want))
    held.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(got, beam.beam_select(held, s, 8)))


# ---- reordering -----------------------------------------------------------------

def reorder_case(layers, batch, beams, lens, heads, page, dim, dtype, seed, width=None):
    rows = batch * beams
    c = Cache([lens[i // beams] for i in range(rows)], heads, page, dim, dtype, seed=seed, spare=rows,
              capacity=max(lens) + 2 * page)
    g = torch.Generator().manual_seed(seed + 1)
    k = torch.stack([c.k] + [torch.randn(c.k.shape, generator=g).to(dtype) for _ in range(layers - 1)])
    v = torch.stack([c.v] + [torch.randn(c.k.shape, generator=g).to(dtype) for _ in range(layers - 1)])
    parent = torch.randint(0, beams, (batch, beams), generator=g, dtype=torch.int32)
    w = None if width is None else torch.rand((layers, rows, heads, width), generator=g)
    return c, k, v, parent, w


def check_reorder(c, k, v, parent, w, flat=False):
    from franken_ocr_b200 import beam

    batch, beams = parent.shape
    fresh = torch.tensor(c.spare, dtype=torch.int32)
    kd, vd = k.cuda(), v.cuda()
    wd = None if w is None else w.cuda()
    args = (kd[0], vd[0]) if flat else (kd, vd)
    table, lens, wo = beam.beam_reorder(*args, c.table.cuda(), c.lens.cuda(), parent.cuda(), fresh.cuda(),
                                        weights=None if wd is None else wd[0] if flat else wd)
    want = torch.full_like(c.table, -1)
    k, v = k.clone(), v.clone()
    ww = None if w is None else torch.zeros_like(w)
    new = []
    for i in range(batch * beams):
        p = int(parent[i // beams, i % beams])
        src = i // beams * beams + p
        n = int(c.lens[src]) if 0 <= p < beams else 0
        full, rest = divmod(n, c.page)
        new.append(n)
        if n:
            want[i, :full] = c.table[src, :full]
        want[i, full] = fresh[i]
        if rest:
            at = int(c.table[src, full])
            k[:, int(fresh[i]), :, :rest] = k[:, at, :, :rest]
            v[:, int(fresh[i]), :, :rest] = v[:, at, :, :rest]
        if w is not None and n:
            ww[:, i, :, :n] = w[:, src, :, :n]
    assert torch.equal(table.cpu(), want) and lens.tolist() == new
    assert same_bits(kd, k) and same_bits(vd, v)
    if w is not None:
        assert same_bits(wo, ww[0] if flat else ww)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layers,batch,beams,lens,heads,page,dim,width", [
    (12, 1, 4, [37], 10, 16, 128, None), (1, 3, 2, [16, 0, 31], 2, 16, 64, 40), (2, 2, 5, [1, 50], 3, 7, 80, 55),
    (3, 1, 1, [9], 1, 1, 64, 9), (2, 2, 8, [63, 64], 1, 64, 256, None)])
def test_reorder_matches_the_definition(cuda, dtype, layers, batch, beams, lens, heads, page, dim, width):
    check_reorder(*reorder_case(layers, batch, beams, lens, heads, page, dim, DTYPES[dtype], seed=dim, width=width))


def test_reorder_one_layer_without_its_dimension_and_parents_out_of_range(cuda):
    case = reorder_case(1, 3, 4, [20, 33, 5], 2, 16, 64, torch.float32, seed=3, width=64)
    check_reorder(*case, flat=True)
    case[3][0] = torch.tensor([-1, 4, 100, 2])
    check_reorder(*case)


def test_reorder_beyond_32_bits_and_in_a_replayed_graph(cuda):
    from franken_ocr_b200 import beam

    layers, pages, page, dim = 3, 50000, 64, 256
    kp = torch.empty((layers, pages, 1, page, dim), dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    table = torch.tensor([[0, pages - 1, -1], [1, pages - 2, -1]], dtype=torch.int32, device="cuda")
    fresh = torch.tensor([pages - 3, pages - 4], dtype=torch.int32, device="cuda")
    lens = torch.tensor([90, 90], dtype=torch.int32, device="cuda")
    parent = torch.tensor([[1, 1]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in (pages - 1, pages - 2):
        kp[:, p] = torch.randn((layers, 1, page, dim), generator=g, device="cuda")
        vp[:, p] = torch.randn((layers, 1, page, dim), generator=g, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, _, _ = beam.beam_reorder(kp, vp, table, lens, parent, fresh)
    for want in ([1, 1], [1, 0]):
        parent.copy_(torch.tensor([want]))
        graph.replay()
        torch.cuda.synchronize()
        assert new.tolist() == [[table[w, 0].item(), f, -1] for w, f in zip(want, (pages - 3, pages - 4))]
        for i, w in enumerate(want):
            for pool in (kp, vp):
                assert same_bits(pool[:, pages - 3 - i, :, :26], pool[:, pages - 1 - w, :, :26])


def test_reorder_skips_pages_outside_the_pool(cuda):
    from franken_ocr_b200 import beam

    c, k, v, parent, _ = reorder_case(2, 1, 3, [20], 2, 16, 64, torch.float32, seed=4)
    kd, vd = k.cuda(), v.cuda()
    fresh = torch.tensor([c.k.shape[0], -1, c.spare[0]], dtype=torch.int32, device="cuda")
    table = c.table.cuda()
    table[int(parent[0, 2]), 1] = -9
    beam.beam_reorder(kd, vd, table, c.lens.cuda(), parent.cuda(), fresh)
    assert same_bits(kd, k) and same_bits(vd, v)


def test_reorder_keeps_a_lost_tail_lost(cuda):
    """A row whose tail page is not in the pool gives NaN before and after: the fresh page's
    old contents are not its own."""
    from franken_ocr_b200 import beam, paged

    c, k, v, _, _ = reorder_case(1, 2, 2, [20, 32], 2, 16, 64, torch.float32, seed=6)
    kd, vd = k[0].cuda().nan_to_num(1.0), v[0].cuda().nan_to_num(1.0)
    table, fresh = c.table.cuda(), torch.tensor(c.spare, dtype=torch.int32, device="cuda")
    table[1, 1] = c.k.shape[0]
    parent = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device="cuda")
    new, lens, _ = beam.beam_reorder(kd, vd, table, c.lens.cuda(), parent, fresh)
    assert new[:, 0].tolist() == table[[1, 0, 3, 3], 0].tolist()
    assert new[:2, 1].tolist() == [-1, c.spare[1]]                  # 20 entries: the tail is the second page
    assert new[2:, 1:3].tolist() == [[int(table[3, 1]), c.spare[2]], [int(table[3, 1]), c.spare[3]]]
    out = paged.paged_attention(torch.ones((4, 2, 64), device="cuda"), kd, vd, new, lens)
    assert bool(out[0].isnan().all()) and bool(out[1:].isfinite().all())


def test_calls_while_another_device_is_current(cuda, monkeypatch):
    """Tensors elsewhere than on the current device: the same call, with theirs as the
    current one, every argument handed on."""
    from franken_ocr_b200 import beam, paged

    real = paged._device
    c, k, v, parent, w = reorder_case(2, 2, 2, [20, 33], 2, 16, 64, torch.float32, seed=7, width=64)
    table, lens, fresh = c.table.cuda(), c.lens.cuda(), torch.tensor(c.spare, dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(1)
    q, x = torch.randn((4, 4, 64), generator=g).cuda(), torch.randn((2, 2, 500), generator=g).cuda()
    done = torch.tensor([[True, False], [False, False]]).cuda()

    def calls():
        """Everything that the five calls return or change."""
        kd, vd, wd = k.cuda(), v.cuda(), w.cuda()
        add = torch.zeros((4, 2, 70), device="cuda")
        out = torch.empty_like(q)
        paged.paged_attention(q, kd[0], vd[0], table, lens, scale=0.3, ref_lens=lens // 4, window=7, weights=add, out=out)
        new, n, ww = beam.beam_reorder(kd, vd, table, lens, parent.cuda(), fresh, weights=wd)
        row = torch.tensor([3, -1, 0], dtype=torch.int32).cuda()
        paged.paged_write(q[:3, :2].contiguous(), q[:3, 2:].contiguous(), kd[1], vd[1], new, n[[3, 0, 0]].contiguous(), row=row)
        evicted = paged.paged_evict(kd[1], vd[1], table, lens, wd[1], fresh[:, None].contiguous(), 16, sink=2, recent=5)
        chosen = beam.beam_select(x, torch.zeros((2, 2), device="cuda"), 5, done=done, end_token=9)
        return [out, add, new, n, ww, kd, vd, *evicted, *chosen]

    want = calls()
    asked = []

    def device():
        asked.append(None)
        return real() + len(asked) % 2      # every first question of a call: another one

    for module in (paged, beam):
        monkeypatch.setattr(module, "_device", device)
    got = calls()
    torch.cuda.synchronize()
    assert len(asked) == 10
    assert all(same_bits(a, b) for a, b in zip(got, want))


def test_calls_at_once_on_two_streams(cuda):
    """Selections, reorderings and evictions side by side do not see one another's
    workspaces."""
    from franken_ocr_b200 import beam, paged

    g = torch.Generator().manual_seed(8)
    work = []
    for i in range(2):
        c, k, v, parent, w = reorder_case(3, 2, 4, [200, 77], 2, 16, 64, torch.float16, seed=20 + i, width=220)
        spare = torch.tensor(c.spare, dtype=torch.int32).cuda()
        x, s = (torch.randn((3, 4, 30000), generator=g) * 2).cuda(), torch.randn((3, 4), generator=g).cuda()
        work.append((c.table.cuda(), c.lens.cuda(), spare, k.cuda(), v.cuda(), parent.cuda(), w.cuda(), x, s))

    def calls(table, lens, spare, k, v, parent, w, x, s):
        first = beam.beam_select(x, s, 8)
        new = beam.beam_reorder(k, v, table, lens, parent, spare, weights=w)
        kept = paged.paged_evict(k[0], v[0], table, lens, w[0], spare[:, None].contiguous(), 16, sink=1, recent=3)
        return [*first, *new, *kept]

    want = [calls(*a) for a in work]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(calls(*work[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(same_bits(a, b) for a, b in zip(one, want[i]))


# ---- together -------------------------------------------------------------------------

def test_beams_over_a_paged_cache_as_they_are_used(cuda):
    """Prompt, then steps of select, reorder, write and attend, and an eviction on
    the way: the cache and the outputs follow a dense 64-bit copy per beam."""
    from franken_ocr_b200 import beam, paged

    g = torch.Generator().manual_seed(11)
    batch, beams, heads, group, dim, page, vocab = 2, 3, 2, 2, 64, 8, 300
    rows, prompt, steps, budget = batch * beams, [21, 9], 14, 16
    width = 8
    pages = batch * width + rows * 2 * (steps + 2) + rows * 4
    pool_k = torch.full((pages, heads, page, dim), math.nan, device="cuda")
    pool_v = pool_k.clone()
    free = torch.randperm(pages, generator=g).tolist()
    # every beam of an entry starts on the same prompt pages
    table = torch.full((rows, width), -1, dtype=torch.int32)
    lens = torch.tensor([prompt[i // beams] for i in range(rows)], dtype=torch.int32)
    dense = [None] * rows
    for b in range(batch):
        own = [free.pop() for _ in range(-(-prompt[b] // page))]
        k = torch.randn((prompt[b], heads, dim), generator=g)
        v = torch.randn((prompt[b], heads, dim), generator=g)
        for i in range(b * beams, (b + 1) * beams):
            table[i, :len(own)] = torch.tensor(own, dtype=torch.int32)
            dense[i] = (k.clone(), v.clone(), torch.zeros((heads, prompt[b]), dtype=torch.float64))
        first = torch.full((prompt[b],), b * beams, dtype=torch.int32).cuda()
        paged.paged_write(k.cuda(), v.cuda(), pool_k, pool_v, table.cuda(),
                          torch.arange(prompt[b], dtype=torch.int32).cuda(), row=first)
    table, lens = table.cuda(), lens.cuda()
    w = torch.zeros((rows, heads, width * page), device="cuda")
    scores = torch.full((batch, beams), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    for step in range(steps):
        logits = torch.randn((batch, beams, vocab), generator=g) * 2
        old = scores.cpu()
        scores, parent, token = beam.beam_select(logits.cuda(), scores)
        for b, want in enumerate(select(logits, old, beams)):
            assert [(i, t) for _, i, t in want] == list(zip(parent[b].tolist(), token[b].tolist()))
        fresh = torch.tensor([free.pop() for _ in range(rows)], dtype=torch.int32).cuda()
        table, lens, w = beam.beam_reorder(pool_k, pool_v, table, lens, parent, fresh, weights=w)
        source = [i // beams * beams + p for i, p in enumerate(parent.view(-1).tolist())]
        dense = [tuple(x.clone() for x in dense[s]) for s in source]
        k, v = torch.randn((rows, heads, dim), generator=g), torch.randn((rows, heads, dim), generator=g)
        paged.paged_write(k.cuda(), v.cuda(), pool_k, pool_v, table, lens)
        lens += 1
        q = torch.randn((rows, heads * group, dim), generator=g)
        out = paged.paged_attention(q.cuda(), pool_k, pool_v, table, lens, weights=w).cpu().double()
        for i in range(rows):
            dk, dv = torch.cat([dense[i][0], k[i:i + 1]]), torch.cat([dense[i][1], v[i:i + 1]])
            dw = torch.cat([dense[i][2], torch.zeros((heads, 1), dtype=torch.float64)], 1)
            for h in range(heads):
                p = torch.softmax(q[i, h * group:(h + 1) * group].double() @ dk[:, h].double().T / 8, -1)
                # ~40 entries, scores below 2^5: a few hundred units of 2^-24 of values below 2^2
                assert torch.allclose(out[i, h * group:(h + 1) * group], p @ dv[:, h].double(), rtol=0, atol=1e-4)
                dw[h] += p.sum(0)
            dense[i] = (dk, dv, dw)
        if step == 6:
            n = lens.tolist()
            into = torch.tensor([free.pop() for _ in range(rows * (budget // page))], dtype=torch.int32)
            small = torch.full((rows, width), -1, dtype=torch.int32)
            small[:, :budget // page] = into.view(rows, -1)
            small = small.cuda()
            kept, lens, w = paged.paged_evict(pool_k, pool_v, table, lens, w, small, budget, sink=1, recent=4)
            table = small
            for i in range(rows):
                pick = kept[i].cpu().long()
                live = min(n[i], budget)
                pick = pick[:, :live]
                dk = torch.stack([dense[i][0][pick[h], h] for h in range(heads)], 1)
                dv = torch.stack([dense[i][1][pick[h], h] for h in range(heads)], 1)
                dense[i] = (dk, dv, dense[i][2].gather(1, pick))
                assert pick[:, 0].tolist() == [0] * heads and pick[:, -1].tolist() == [n[i] - 1] * heads
    assert torch.allclose(w[0, :, :int(lens[0])].cpu().double(), dense[0][2], rtol=0, atol=1e-4)
