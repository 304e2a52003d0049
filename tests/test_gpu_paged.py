"""The paged K/V cache on the GPU against plain 64-bit forms: writes into pages,
attention of one token over them, and eviction by accumulated weight."""
import math

import pytest
import torch

from tests.paged_cases import DTYPES, HALF_STEP, Cache, attention, evict_kept, visible

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("stale_memory")]


@pytest.fixture
def stale_memory(cuda):
    """Workspaces and outputs come from memory that holds NaN (and indexes far
    out of range): nothing may go by what a buffer held before."""
    held = [torch.full((n,), math.nan, device="cuda") for n in (1 << 7, 1 << 12, 1 << 17, 1 << 22, 1 << 24)]
    del held


def same_bits(a, b):
    kind = {4: torch.int32, 2: torch.int16}[a.element_size()]
    return torch.equal(a.contiguous().cpu().view(kind), b.contiguous().cpu().view(kind))


# ---- write -----------------------------------------------------------------

@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pool", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,page,dim,strided", [(10, 16, 128, False), (1, 1, 64, False), (3, 7, 80, True),
                                                    (2, 24, 256, True)])
def test_write_rounds_once_and_touches_nothing_else(cuda, src, pool, heads, page, dim, strided):
    from franken_ocr_b200 import paged

    lens = [5, 0, 3 * page + 2, 1]
    c = Cache([3 * page + 2] * 4, heads, page, dim, DTYPES[pool], seed=dim, strided=strided)
    kp, vp, table = c.cuda()
    row = torch.tensor([r for r, n in enumerate(lens) for _ in range(n)] + [-1, -1], dtype=torch.int32)
    pos = torch.tensor([p for n in lens for p in range(n)] + [0, 1], dtype=torch.int32)
    mix = torch.randperm(len(row), generator=torch.Generator().manual_seed(1))
    row, pos = row[mix], pos[mix]
    g = torch.Generator().manual_seed(2)
    k = torch.randn((len(row), heads, dim), generator=g).to(DTYPES[src])
    v = torch.randn((len(row), heads, dim), generator=g).to(DTYPES[src])
    paged.paged_write(k.cuda(), v.cuda(), kp, vp, table, pos.cuda(), row=row.cuda())
    for t in range(len(row)):
        r, p = int(row[t]), int(pos[t])
        if r >= 0:
            at = int(c.table[r, p // page])
            c.k[at, :, p % page] = k[t].to(c.dtype)
            c.v[at, :, p % page] = v[t].to(c.dtype)
    assert same_bits(kp, c.k) and same_bits(vp, c.v)


def test_write_from_a_fused_projection_and_unaligned_rows(cuda):
    """k and v as slices of one [tokens, q|k|v] buffer, on and off 16-byte boundaries."""
    from franken_ocr_b200 import paged

    heads, dim, page = 3, 64, 16
    for shift in (0, 1):
        c = Cache([20] * 5, heads, page, dim, torch.bfloat16, seed=3)
        kp, vp, table = c.cuda()
        qkv = torch.randn((5, 3 * heads * dim + shift), generator=torch.Generator().manual_seed(4))
        dev = qkv.cuda()
        part = [dev[:, shift + i * heads * dim:shift + (i + 1) * heads * dim].view(5, heads, dim) for i in (1, 2)]
        pos = torch.tensor([0, 15, 16, 19, 7], dtype=torch.int32)
        paged.paged_write(part[0], part[1], kp, vp, table, pos.cuda())
        for r in range(5):
            at, s = int(c.table[r, int(pos[r]) // page]), int(pos[r]) % page
            c.k[at, :, s] = qkv[r, shift + heads * dim:shift + 2 * heads * dim].view(heads, dim).to(c.dtype)
            c.v[at, :, s] = qkv[r, shift + 2 * heads * dim:].view(heads, dim).to(c.dtype)
        assert same_bits(kp, c.k) and same_bits(vp, c.v)


def test_write_skips_what_is_out_of_range(cuda):
    from franken_ocr_b200 import paged

    c = Cache([16, 16], 2, 8, 64, torch.float32, seed=5)
    kp, vp, table = c.cuda()
    table[1, 0], table[1, 1] = c.k.shape[0], -1
    row = torch.tensor([-5, 2, 0, 0, 1, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 0, -1, 16, 3, 9], dtype=torch.int32, device="cuda")
    x = torch.ones((6, 2, 64), device="cuda")
    paged.paged_write(x, x, kp, vp, table, pos, row=row)
    assert same_bits(kp, c.k) and same_bits(vp, c.v)
    paged.paged_write(x[:0], x[:0], kp, vp, table, pos[:0], row=row[:0])
    assert same_bits(kp, c.k)


# ---- attention ----------------------------------------------------------------

def check_attention(c, q, lens, refs=None, window=0, weights=False, scale=None, width=None, dev=None):
    from franken_ocr_b200 import paged

    kp, vp, table = dev or c.cuda()
    rows = len(lens)
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    dr = None if refs is None else torch.tensor(refs, dtype=torch.int32, device="cuda")
    w = w0 = None
    if weights:
        w0 = torch.rand((rows, c.heads, width or c.width * c.page), generator=torch.Generator().manual_seed(8))
        w = w0.cuda()
    used = 1 / math.sqrt(c.dim) if scale is None else scale
    want, probs, bound = attention(c, q, lens, used, refs, window)
    got = paged.paged_attention(q.cuda(), kp, vp, table, dl, ref_lens=dr, window=window, weights=w, scale=scale)
    assert got.dtype == q.dtype and got.shape == q.shape
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max())} bounds"
    if weights:
        group = q.shape[1] // c.heads
        rest = torch.ones_like(w0, dtype=torch.bool)
        gw = w.cpu()
        for (r, h), (at, p) in probs.items():
            rest[r, h, at] = False
            new = gw[r, h, at].double() - w0[r, h, at].double()
            # bound of a probability (as in `attention`), the group's sum, the add's rounding
            tol = group * (bound_of_p(c, q, r, h, at, used, group)) * p + 2.0 ** -24 * (w0[r, h, at] + p + 1)
            assert bool(((new - p).abs() <= tol).all())
        assert torch.equal(gw[rest], w0[rest])
    return got


def bound_of_p(c, q, r, h, at, scale, group):
    qs = q[r, h * group:(h + 1) * group].double()
    k = c.row(r, at)[h]
    s = (scale * qs @ k.T).abs()
    ds = float((scale * qs.abs() @ k.abs().T).max()) * (c.dim + 2) * 2.0 ** -24
    return 2 * ds + 2 * (len(at) + 16) * 2.0 ** -24 + 2.0 ** -21 + float(s.max()) * 2.0 ** -22


@pytest.mark.parametrize("q_type,pool", [(a, b) for a in DTYPES for b in DTYPES])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_types(cuda, q_type, pool, dim):
    lens = [1, 2, 0, 63, 64, 65, 257]
    c = Cache(lens, 2, 16, dim, DTYPES[pool], seed=dim)
    q = torch.randn((len(lens), 2, dim), generator=torch.Generator().manual_seed(1)).to(DTYPES[q_type])
    check_attention(c, q, lens)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("q_type,pool", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")])
def test_attention_head_groups_with_weights(cuda, group, q_type, pool):
    lens = [130, 1, 0, 77]
    c = Cache(lens, 3, 16, 128, DTYPES[pool], seed=group)
    q = torch.randn((4, 3 * group, 128), generator=torch.Generator().manual_seed(group)).to(DTYPES[q_type])
    check_attention(c, q, lens, weights=True)


@pytest.mark.parametrize("dim,pool", [(8, "bf16"), (16, "f32"), (72, "f16"), (80, "bf16"), (96, "f32"), (4, "f32"),
                                      (100, "f32"), (136, "bf16"), (192, "f16"), (200, "f32"), (248, "f16")])
@pytest.mark.parametrize("group", [1, 6])
def test_attention_odd_dims(cuda, dim, pool, group):
    lens = [31, 100]
    c = Cache(lens, 2, 8, dim, DTYPES[pool], seed=dim)
    for q_type in ("f32", pool):
        q = torch.randn((2, 2 * group, dim), generator=torch.Generator().manual_seed(dim)).to(DTYPES[q_type])
        check_attention(c, q, lens, weights=True)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 100, 256])
@pytest.mark.parametrize("pool,group", [("f32", 1), ("bf16", 8)])
def test_attention_pages_that_end_inside_a_tile(cuda, page, pool, group):
    lens = [1, page, page + 1, 5 * page - 1, 300]
    c = Cache(lens, 2, page, 64, DTYPES[pool], seed=page, strided=True)
    q = torch.randn((5, 2 * group, 64), generator=torch.Generator().manual_seed(page)).to(DTYPES[pool])
    check_attention(c, q, lens, weights=True)


@pytest.mark.parametrize("window", [1, 17, 128, 4000])
@pytest.mark.parametrize("pool,group", [("f32", 1), ("f16", 5)])
def test_attention_reference_and_window(cuda, window, pool, group):
    """The R-SWA rule: hidden entries hold NaN and infinities."""
    lens = [1, 40, 200, 300, 300, 300, 0, 513]
    refs = [0, 40, 64, 300, 1000, -3, 5, 100]
    c = Cache(lens, 2, 16, 64, DTYPES[pool], seed=window)
    for r, n in enumerate(lens):
        seen = set(visible(n, max(0, min(refs[r], n)), window))
        for j in range(n):
            if j not in seen:
                at = int(c.table[r, j // 16])
                c.k[at, :, j % 16] = math.inf if j % 2 else math.nan
                c.v[at, :, j % 16] = -math.inf
    q = torch.randn((len(lens), 2 * group, 64), generator=torch.Generator().manual_seed(5)).to(DTYPES[pool])
    clamped = [max(0, min(a, n)) for a, n in zip(refs, lens)]
    kp = c.cuda()
    out = check_attention(c, q, lens, refs=clamped, window=window, weights=True, dev=kp)
    from franken_ocr_b200 import paged
    raw = paged.paged_attention(q.cuda(), *kp, torch.tensor(lens, dtype=torch.int32, device="cuda"), window=window,
                                ref_lens=torch.tensor(refs, dtype=torch.int32, device="cuda"))
    assert same_bits(raw, out)


@pytest.mark.parametrize("rows,high", [(1, 20000), (3, 9000), (37, 700), (700, 9)])
@pytest.mark.parametrize("pool,group,dim", [("f32", 1, 128), ("bf16", 8, 128), ("bf16", 2, 64)])
def test_attention_split_and_joined(cuda, rows, high, pool, group, dim):
    """Rows that many blocks share, and blocks that many rows share."""
    lens = [(high * (7 * r % 11 + 1)) // 11 if r % 5 != 3 else 0 for r in range(rows)]
    lens[0] = high
    c = Cache(lens, 1, 16, dim, DTYPES[pool], seed=rows)
    q = torch.randn((rows, group, dim), generator=torch.Generator().manual_seed(rows)).to(DTYPES[pool]) * 2
    check_attention(c, q, lens, weights=rows == 3)


def test_attention_over_a_thousand_rows(cuda):
    lens = [(5 * r) % 23 for r in range(1500)]
    c = Cache(lens, 1, 8, 64, torch.bfloat16, seed=1)
    q = torch.randn((1500, 2, 64), generator=torch.Generator().manual_seed(1))
    check_attention(c, q, lens, weights=True)


@pytest.mark.parametrize("q_type,pool,group,dim", [("f32", "f32", 1, 256), ("bf16", "bf16", 6, 64)])
def test_attention_behind_a_table_of_all_the_positions_there_are(cuda, q_type, pool, group, dim):
    """A row of such a table has up to 2^26 tiles: a launch takes only as many rows as
    32 bits count tiles of, and the rows beyond follow."""
    from franken_ocr_b200 import paged

    page, rows = 1 << 12, 70
    lens = [(13 * r) % 90 for r in range(rows)]
    c = Cache(lens, 1, page, dim, DTYPES[pool], seed=3, capacity=1)
    # short pages' contents, packed into pages that are long
    pages, width = c.k.shape[0], (2**31 - 2**16) // page
    kp, vp, _ = c.cuda()
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table.cuda()
    q = torch.randn((rows, group, dim), generator=torch.Generator().manual_seed(4)).to(DTYPES[q_type])
    check_attention(c, q, lens, dev=(kp, vp, table))
    check_attention(c, q, lens, refs=[r % 20 for r in range(rows)], window=30, dev=(kp, vp, table))


def test_attention_workspace_goes_by_the_narrower_of_table_and_weights(cuda):
    """Weights far wider than the table ask for no more than the table's scores."""
    from franken_ocr_b200 import paged

    c = Cache([40] * 3, 2, 16, 64, torch.float32, seed=2)
    kp, vp, table = c.cuda()
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(1)).cuda()
    lens = torch.full((3,), 40, dtype=torch.int32, device="cuda")
    w = torch.zeros((3, 2, 1 << 20), device="cuda")
    paged.paged_attention(q, kp, vp, table, lens, weights=w)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = paged.paged_attention(q, kp, vp, table, lens, weights=w)
    plain = paged.paged_attention(q, kp, vp, table, lens)
    # the partial sums' part is there without weights too; scores of 48 positions beside it
    assert torch.cuda.max_memory_allocated() - before < 4 << 20
    assert same_bits(out, plain) and abs(float(w.sum()) - 3 * 2 * 2 * 2) < 1e-3


def test_attention_peaks_and_scales(cuda):
    """Scores far apart, a maximum at either end, another scale."""
    n = 700
    c = Cache([n, n, n], 1, 16, 128, torch.float32, seed=2)
    q = torch.randn((3, 1, 128), generator=torch.Generator().manual_seed(3))
    for r, j in enumerate((0, n - 1, n // 2)):
        c.k[int(c.table[r, j // 16]), 0, j % 16] = q[r, 0] * 1.0
    check_attention(c, q, [n] * 3, scale=0.7)
    check_attention(c, q, [n] * 3, scale=1e-6)


def test_attention_unseen_nan_and_bad_pages(cuda):
    from franken_ocr_b200 import paged

    lens = [40, 40, 40, 200, -4]
    c = Cache([40, 40, 40, 40, 40], 2, 16, 64, torch.float32, seed=6)
    kp, vp, table = c.cuda()
    table[1, 1] = kp.shape[0]
    table[2, 2] = -1
    q = torch.randn((5, 4, 64), generator=torch.Generator().manual_seed(7)).cuda()
    w = torch.ones((5, 2, 48), device="cuda")
    out = paged.paged_attention(q, kp, vp, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), weights=w)
    good = attention(c, q.cpu()[:1], [40], 1 / 8)[0]
    assert torch.allclose(out[0].cpu().double(), good[0], atol=1e-4)
    assert bool(out[1:4].isnan().all())
    assert bool((out[4] == 0).all())
    assert bool((w[1:] == 1).all())          # rows that give NaN, and empty ones, leave their weights
    assert abs(float((w[0] - 1).sum()) - 4) < 1e-4  # two kv heads, two query heads each
    q[0] = math.nan
    out = paged.paged_attention(q, kp, vp, table, torch.tensor([40, 0, 0, 0, 0], dtype=torch.int32, device="cuda"))
    assert bool(out[0].isnan().all()) and bool((out[1:] == 0).all())


# (query type, pool, query heads a kv head, head_dim): every kernel
KINDS = [("f32", "f32", 1, 64), ("f16", "f16", 2, 128), ("bf16", "bf16", 3, 128), ("f16", "f16", 5, 64), ("f16", "f16", 4, 256),
         ("bf16", "bf16", 17, 256), ("f32", "bf16", 6, 128), ("f32", "f16", 7, 64), ("f32", "f16", 5, 256)]


def around_the_shares(c):
    """The cache's tensors for each way of sharing the rows out: by its own table, by one
    for long contexts, and among many short rows."""
    kp, vp, table = c.cuda()
    wide = torch.full((table.shape[0], 1 << 15), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    times = -(-1200 // table.shape[0])
    return [(kp, vp, table, 1), (kp, vp, wide, 1), (kp, vp, table.repeat(times, 1), times)]


@pytest.mark.parametrize("q_type,pool,group,dim", KINDS)
def test_attention_where_every_score_is_minus_infinity(cuda, q_type, pool, group, dim):
    """The softmax of nothing but -inf has no value: NaN, and the weights stay; a row
    without positions gives zeros beside it."""
    from franken_ocr_b200 import paged

    lens = [50, 0, 50]
    c = Cache(lens, 1, 16, dim, DTYPES[pool], seed=dim)
    for j in range(50):
        c.k[int(c.table[0, j // 16]), 0, j % 16, 3] = -math.inf
    q = torch.randn((3, group, dim), generator=torch.Generator().manual_seed(group)).to(DTYPES[q_type])
    q[:, :, 3] = q[:, :, 3].abs() + 0.25
    for kp, vp, table, times in around_the_shares(c):
        w = torch.zeros((3 * times, 1, 64), device="cuda")
        out = paged.paged_attention(q.cuda().repeat(times, 1, 1), kp, vp, table, c.lens.cuda().repeat(times), weights=w).view(
            times, 3, group, dim)
        assert bool(out[:, 0].isnan().all()) and bool((out[:, 1] == 0).all()) and bool(out[:, 2].isfinite().all())
        assert bool((w.view(times, 3, 64)[:, :2] == 0).all())


@pytest.mark.parametrize("q_type,pool,group,dim", KINDS)
@pytest.mark.parametrize("size", [1e7, 3e8, 1e10, 1e20])
def test_attention_of_scores_past_2_24(cuda, q_type, pool, group, dim, size):
    """Scores whose products round by more than 1: the largest, a tied few, share the
    probability, and the others, far behind, have none."""
    from franken_ocr_b200 import paged

    n = 50
    c = Cache([n, n], 1, 16, dim, DTYPES[pool], seed=dim)
    g = torch.Generator().manual_seed(group)
    q = (1 + torch.rand((2, group, dim), generator=g)).to(DTYPES[q_type])
    top = (1 + torch.rand((dim,), generator=g)).to(DTYPES[pool])
    best = [3, 17, 40]
    for r in range(2):
        for j in range(n):
            # a lower key has half of every product or less
            c.k[int(c.table[r, j // 16]), 0, j % 16] = top if j in best else (top.float() * (j % 4) / 8).to(c.dtype)
    want = c.row(0, best, "v")[0].mean(0), c.row(1, best, "v")[0].mean(0)
    scale = size / float((q.double() @ top.double()).max())
    for kp, vp, table, times in around_the_shares(c):
        w = torch.zeros((2 * times, 1, 64), device="cuda")
        out = paged.paged_attention(q.cuda().repeat(times, 1, 1), kp, vp, table, c.lens.cuda().repeat(times), scale=scale,
                                    weights=w).view(times, 2, group, dim).cpu().double()
        for r in range(2):
            # three equal probabilities: a few roundings, and the output's own
            off = (out[:, r] - want[r]).abs()
            assert bool((off <= 2.0 ** -16 * 3 + want[r].abs() * HALF_STEP[q.dtype]).all())
        # a third each for every query head, to a few roundings
        got = w.view(times, 2, 64).cpu().double()
        assert bool(((got[:, :, best] - group / 3).abs() <= group * 2.0 ** -20).all())
        got[:, :, best] = 0
        assert bool((got == 0).all())


@pytest.mark.parametrize("q_type,pool,group,dim", KINDS)
def test_attention_of_infinite_keys(cuda, q_type, pool, group, dim):
    """A score of -inf has probability 0, whatever the kernel; one of +inf, or of both, has
    none: NaN. Queries with an infinity of their own likewise."""
    from franken_ocr_b200 import paged

    n = 60
    c = Cache([n, n, n], 1, 16, dim, DTYPES[pool], seed=dim)
    q = torch.randn((3, group, dim), generator=torch.Generator().manual_seed(group)).to(DTYPES[q_type])
    q[:, :, 5] = q[:, :, 5].abs() + 0.25
    q[:, :, 9] = -q[:, :, 9].abs() - 0.25
    for r in range(3):
        for j in range(n):
            at = c.k[int(c.table[r, j // 16]), 0, j % 16]
            at[5], at[9] = at[5].abs() + 0.25, at[9].abs() + 0.25
            if r == 0 and j % 3 == 1:      # -inf by either sign of the query
                at[5 if j % 2 else 9] = math.inf * (-1 if j % 2 else 1)
            if r == 1 and j == 30:
                at[5] = math.inf
    q[2, :, 9] = -math.inf                  # every score of the row
    seen = [j for j in range(n) if j % 3 != 1]
    p = torch.softmax(q[0].double() @ c.row(0, seen)[0].T / math.sqrt(dim), -1)
    v = c.row(0, seen, "v")[0]
    # (dim + 2) roundings of a score, the sums' and the exponential's, as in `attention`
    rel = 2 * (dim + 2) * 2.0 ** -24 * float((q[0].double().abs() @ c.row(0, seen)[0].abs().T).max()) / math.sqrt(dim)
    bound = (rel + 2.0 ** -13) * (p @ v.abs()) + (p @ v).abs() * HALF_STEP[q.dtype]
    for kp, vp, table, times in around_the_shares(c):
        w = torch.zeros((3 * times, 1, 64), device="cuda")
        out = paged.paged_attention(q.cuda().repeat(times, 1, 1), kp, vp, table, c.lens.cuda().repeat(times), weights=w)
        out = out.view(times, 3, group, dim).cpu()
        assert bool(((out[:, 0].double() - p @ v).abs() <= bound).all())
        assert bool(out[:, 1:].isnan().all())
        w = w.view(times, 3, 64).cpu()
        assert bool((w[:, 0, 1:n:3] == 0).all()) and bool((w[:, 1:] == 0).all())


@pytest.mark.parametrize("q_type,pool,group,dim", KINDS)
def test_attention_of_infinite_values(cuda, q_type, pool, group, dim):
    """A visible infinity in V is the output's, in its column alone and whatever the kernel;
    with its opposite, or NaN, it has none."""
    from franken_ocr_b200 import paged

    n = 70
    c = Cache([n, n], 1, 16, dim, DTYPES[pool], seed=dim)
    q = torch.randn((2, group, dim), generator=torch.Generator().manual_seed(group)).to(DTYPES[q_type])

    def put(j, d, x):
        c.v[int(c.table[0, j // 16]), 0, j % 16, d] = x

    # every position once, so every part of a probability meets one
    for j in range(n):
        put(j, j % 30, math.inf if j % 2 else -math.inf)
    want = torch.full((dim,), math.nan)
    want[30] = 0.0          # stands for any finite value
    for d in range(30):
        signs = {j % 2 for j in range(n) if j % 30 == d}
        want[d] = math.nan if len(signs) == 2 else math.inf if 1 in signs else -math.inf
    put(40, 31, math.inf)
    put(41, 31, -math.inf)
    put(69, 32, math.nan)
    want[33:] = 0.0
    plain, _, bound = attention(c, q, [n, n], 1 / math.sqrt(dim))
    for kp, vp, table, times in around_the_shares(c):
        out = paged.paged_attention(q.cuda().repeat(times, 1, 1), kp, vp, table, c.lens.cuda().repeat(times))
        out = out.view(times, 2, group, dim).cpu()
        got = torch.where(out[:, 0].isfinite(), torch.zeros(()), out[:, 0].float())
        assert torch.equal(got.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0),
                           want.nan_to_num(nan=7.0, posinf=8.0, neginf=9.0).expand(got.shape))
        assert bool(((out[:, 0, :, 33:].double() - plain[0, :, 33:]).abs() <= bound[0, :, 33:]).all())
        assert bool(((out[:, 1].double() - plain[1]).abs() <= bound[1]).all())


def test_attention_strided_queries_and_out(cuda):
    from franken_ocr_b200 import paged

    c = Cache([50, 60], 2, 16, 64, torch.bfloat16, seed=9)
    kp, vp, table = c.cuda()
    qkv = torch.randn((2, 3 * 4 * 64), generator=torch.Generator().manual_seed(1)).cuda()
    q = qkv[:, 256:512].view(2, 4, 64)
    lens = torch.tensor([50, 60], dtype=torch.int32, device="cuda")
    want = paged.paged_attention(q.contiguous(), kp, vp, table, lens)
    out = torch.empty((2, 4, 64), device="cuda")
    assert paged.paged_attention(q, kp, vp, table, lens, out=out) is out
    assert same_bits(out, want)


@pytest.mark.parametrize("pool", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-30, 1e-5, 300.0, 1e6])
def test_attention_f32_queries_of_any_size(cuda, pool, size):
    """Split queries keep 24 bits whatever their size; heads of one group differ."""
    c = Cache([90, 40], 2, 16, 128, DTYPES[pool], seed=12)
    q = torch.randn((2, 12, 128), generator=torch.Generator().manual_seed(13))
    q[:, ::2] *= size
    q[0, 5] = 0.0
    check_attention(c, q, [90, 40], scale=min(0.1, 0.5 / size))


@pytest.mark.parametrize("pool,group,dim", [("f32", 1, 128), ("f32", 7, 64), ("bf16", 2, 128), ("bf16", 6, 64), ("f16", 16, 128)])
def test_attention_long_rows_stay_exact(cuda, pool, group, dim):
    """An f32 output over 60000 positions: sums that take many steps, with maxima that
    rise along the row and fall behind it, lose no more than their roundings."""
    from franken_ocr_b200 import paged

    n = 60000
    c = Cache([n, n], 1, 64, dim, DTYPES[pool], seed=17)
    # scores that climb over the first row, and peak early in the second
    q = torch.randn((2, group, dim), generator=torch.Generator().manual_seed(18))
    for r in range(2):
        slope = torch.linspace(0, 0.4, n) if r == 0 else torch.linspace(0.4, 0, n)
        at = torch.arange(n)
        pages = c.table[r].long()[at // 64]
        c.k[pages, 0, at % 64] = (c.k[pages, 0, at % 64].float() + slope[:, None] * q[r, 0]).to(c.dtype)
    out = paged.paged_attention(q.cuda(), *c.cuda(), c.lens.cuda())
    want, _, _ = attention(c, q, [n, n], 1 / math.sqrt(dim))
    # A value's error is a sum of n roundings of either sign, 2^-24 of partial sums
    # that are no larger than about |v| sqrt(n) weights: relative to the output's own
    # size, which is that of |v| sqrt(n) weights too, some 2^-24 sqrt(steps); 512 steps
    # and more a warp would be 2^-19.5.
    rel = float((out.cpu().double() - want).norm() / want.norm())
    assert rel < 2.0 ** -19.5, rel


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1 << 17, 1 << 20])
def test_attention_of_16_bit_queries_over_long_rows(cuda, dtype, dim, n):
    """As many rows as blocks, so that one block sums a whole row of values of one sign:
    no error that grows with the row."""
    from franken_ocr_b200 import paged

    dtype, page, group = DTYPES[dtype], 4096, 4
    rows = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    g = torch.Generator(device="cuda").manual_seed(n + dim)
    k = torch.randn((n // page, 1, page, dim), generator=g, device="cuda").to(dtype)
    v = (1 + torch.randn(k.shape, generator=g, device="cuda").abs() / 2).to(dtype)
    order = torch.randperm(n // page, generator=g, device="cuda")
    q = torch.randn((4, group, dim), generator=g, device="cuda").to(dtype)
    out = paged.paged_attention(q.repeat(rows // 4, 1, 1), k, v, order.int().repeat(rows, 1),
                                torch.full((rows,), n, dtype=torch.int32, device="cuda"))
    assert all(same_bits(out[r], out[r % 4]) for r in range(rows))
    p = torch.softmax(q.view(-1, dim).double() @ k[order, 0].view(n, dim).double().T / math.sqrt(dim), -1)
    want = (p @ v[order, 0].view(n, dim).double()).view(4, group, dim)
    # One rounding to the output's type: half a step at the value. Below it f32 sums of
    # n / 64 tiles a warp and their probabilities, whose roundings are of either sign:
    # 2^-24 sqrt(n / 4) of the value, 2^-15 at 2^20; the probability's two parts leave
    # 2^-17 of each, of either sign too, which the sum over n makes nothing.
    step = torch.exp2(torch.floor(torch.log2(want))) * torch.finfo(dtype).eps
    off = out[:4].double() - want
    below = 2.0 ** -14 * want
    assert bool((off.abs() <= step / 2 + below).all()), float(((off.abs() - step / 2) / want).max())


@pytest.mark.parametrize("pool,group,dim", [("f32", 1, 128), ("bf16", 1, 64), ("bf16", 6, 128), ("f16", 20, 256)])
@pytest.mark.parametrize("heads", [1, 3])
def test_attention_small_and_large_tables_agree(cuda, pool, group, dim, heads):
    """The same rows behind a table of their own size (shared by a cluster of blocks) and
    behind one for long contexts (runs of tiles and a join); lengths of 0 and out of
    range among them."""
    from franken_ocr_b200 import paged

    lens = [300, 0, 1, 33]
    c = Cache(lens, heads, 16, dim, DTYPES[pool], seed=dim)
    q = torch.randn((4, heads * group, dim), generator=torch.Generator().manual_seed(1)).to(DTYPES[pool])
    kp, vp, table = c.cuda()
    wide = torch.full((4, 1 << 16), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    outs, sums = [], []
    for t in (table, wide):
        w = torch.zeros((4, heads, 320), device="cuda")
        outs.append(check_attention(c, q, lens, dev=(kp, vp, t)))
        outs.append(paged.paged_attention(q.cuda(), kp, vp, t, torch.tensor(lens, dtype=torch.int32, device="cuda"), weights=w))
        sums.append(w)
    want, _, bound = attention(c, q, lens, 1 / math.sqrt(dim))
    for out in outs:
        assert bool(((out.cpu().double() - want).abs() <= bound).all())
    for w in sums:
        # every query head's probabilities add up to 1: 300 f32 values below 1 each
        assert torch.allclose(w.sum(-1).cpu(), torch.tensor([[group] * heads if n else [0] * heads for n in lens]).float(),
                              rtol=0, atol=group * 320 * 2.0 ** -20)
    bad = torch.tensor([300, 0, 1, 1 << 21], dtype=torch.int32, device="cuda")
    for t in (table, wide):
        out = paged.paged_attention(q.cuda(), kp, vp, t, bad)
        assert bool(out[3].isnan().all()) and bool((out[1] == 0).all()) and bool(out[0].isfinite().all())


@pytest.mark.parametrize("q_type,pool,group,dim", [("bf16", "bf16", 11, 64), ("f32", "f32", 6, 128), ("f32", "bf16", 2, 256)])
def test_attention_one_long_row_among_many(cuda, q_type, pool, group, dim):
    """A row cut into more pieces than a warp has lanes, with several heads to join."""
    lens = [(3 * r) % 70 for r in range(50)]
    lens[17] = 30000
    c = Cache(lens, 1, 32, dim, DTYPES[pool], seed=31)
    q = torch.randn((50, group, dim), generator=torch.Generator().manual_seed(32)).to(DTYPES[q_type])
    got = check_attention(c, q, lens, weights=True)
    assert same_bits(check_attention(c, q, lens), got)


@pytest.mark.parametrize("q_type,pool,group,dim", [
    ("f32", "f32", 1, 128), ("f32", "f16", 7, 256), ("bf16", "bf16", 2, 64), ("bf16", "bf16", 5, 128),
    ("f16", "f16", 20, 80), ("f32", "bf16", 16, 64), ("f32", "f32", 3, 20), ("bf16", "bf16", 6, 256),
])
def test_attention_many_short_rows(cuda, q_type, pool, group, dim):
    """More (row, head)s than blocks and few positions each: a warp has one to itself.
    Rows with nothing to see and rows that give NaN change none of their neighbours."""
    from franken_ocr_b200 import paged

    rows, heads = 450, 2
    lens = [(7 * r) % 41 for r in range(rows)]
    c = Cache(lens, heads, 8, dim, DTYPES[pool], seed=group)
    q = torch.randn((rows, heads * group, dim), generator=torch.Generator().manual_seed(dim)).to(DTYPES[q_type])
    good = check_attention(c, q, lens, weights=True)
    assert same_bits(check_attention(c, q, lens), good)
    check_attention(c, q, lens, refs=[r % 9 for r in range(rows)], window=6, weights=True)
    kp, vp, table = c.cuda()
    odd = torch.tensor(lens, dtype=torch.int32)
    odd[3::10] = 1 << 20
    odd[4::10] = -5
    if lens[16] > 8:
        table[16, 1] = -1
    w = torch.zeros((rows, heads, 40), device="cuda")
    out = paged.paged_attention(q.cuda(), kp, vp, table, odd.cuda(), weights=w).cpu()
    nan = torch.zeros(rows, dtype=torch.bool)
    nan[3::10] = True
    nan[16] = lens[16] > 8
    zero = odd <= 0
    assert bool(out[nan].isnan().all()) and bool((out[zero] == 0).all())
    rest = ~(nan | zero)
    assert same_bits(out[rest], good.cpu()[rest])
    assert bool((w.cpu()[~rest] == 0).all())
    # an out that begins on no boundary of a wide store
    flat = torch.full((out.numel() + 1,), 7.0, dtype=DTYPES[q_type], device="cuda")
    view = flat[1:].view(out.shape)
    paged.paged_attention(q.cuda(), kp, vp, table, odd.cuda(), out=view)
    assert same_bits(view.cpu()[rest], good.cpu()[rest])
    assert float(flat[0]) == 7


@pytest.mark.parametrize("prefill,ring,more", [(1024, 128, 0), (1000, 37, 500), (1, 1, 300), (300, 128, 7)])
def test_window_over_pages_equals_the_dense_caches(cuda, prefill, ring, more):
    """The R-SWA decode attention of the dense caches (reference block and ring) and the
    paged form of it, where the window is the ring and `more` entries between the two
    have left it."""
    from franken_ocr_b200 import decoder_ops, paged

    heads, dim, page = 10, 128, 16
    n = prefill + more + ring
    g = torch.Generator().manual_seed(prefill)
    k, v = torch.randn((n, heads, dim), generator=g), torch.randn((n, heads, dim), generator=g)
    q = torch.randn((1, heads, dim), generator=g)
    c = Cache([n], heads, page, dim, torch.float32, seed=19)
    kp, vp, table = c.cuda()
    pos = torch.arange(n, dtype=torch.int32)
    paged.paged_write(k.cuda(), v.cuda(), kp, vp, table, pos.cuda(), row=torch.zeros_like(pos).cuda())
    at = pos.long()
    c.k[c.table[0].long()[at // page], :, at % page], c.v[c.table[0].long()[at // page], :, at % page] = k, v
    got = paged.paged_attention(q.cuda(), kp, vp, table, torch.tensor([n], dtype=torch.int32, device="cuda"),
                                ref_lens=torch.tensor([prefill], dtype=torch.int32, device="cuda"), window=ring)[0]
    dense = [t.transpose(0, 1).contiguous().cuda() for t in (k[:prefill], v[:prefill], k[n - ring:], v[n - ring:])]
    want = decoder_ops.attention_decode(q[0].cuda(), dense[0], dense[1], prefill, dense[2], dense[3], ring)
    _, _, bound = attention(c, q, [n], 1 / math.sqrt(dim), [prefill], ring)
    assert bool(((got - want).abs().cpu() <= 2 * bound[0]).all())   # each is within one bound


def test_calls_on_other_streams(cuda):
    """Work goes to the current stream, also two calls at once on two streams."""
    from franken_ocr_b200 import paged

    c = Cache([3000, 900], 2, 16, 128, torch.bfloat16, seed=14)
    kp, vp, table = c.cuda()
    lens = torch.tensor([3000, 900], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(15)
    qs = [torch.randn((2, 8, 128), generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    want = [paged.paged_attention(q, kp, vp, table, lens) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(paged.paged_attention(qs[i], kp, vp, table, lens))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same_bits(o, want[i]) for o in outs[i])
    # a value written on the side stream is seen by the call behind it there
    with torch.cuda.stream(streams[0]):
        q = torch.zeros_like(qs[0])
        torch.cuda._sleep(2_000_000)
        q.copy_(qs[1])
        out = paged.paged_attention(q, kp, vp, table, lens)
    torch.cuda.synchronize()
    assert same_bits(out, want[1])


def test_weights_in_a_replayed_graph(cuda):
    """A captured step adds its weights once a replay, and sees changed lengths."""
    from franken_ocr_b200 import paged

    c = Cache([70, 50], 2, 16, 64, torch.float32, seed=16)
    kp, vp, table = c.cuda()
    q = torch.randn((2, 2, 64), generator=torch.Generator().manual_seed(1)).cuda()
    lens = torch.tensor([70, 50], dtype=torch.int32, device="cuda")
    once = torch.zeros((2, 2, 80), device="cuda")
    paged.paged_attention(q, kp, vp, table, lens, weights=once)
    w = torch.zeros_like(once)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.paged_attention(q, kp, vp, table, lens, weights=w)
    w.zero_()
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.allclose(w, 4 * once, rtol=2.0 ** -20, atol=0)
    lens.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.allclose(w, 4 * once, rtol=2.0 ** -20, atol=0)


def test_attention_is_the_same_every_time_and_in_a_graph(cuda):
    """Repeated calls give the same bits; a captured call follows its inputs, also
    beside another captured call."""
    from franken_ocr_b200 import paged

    c = Cache([4000, 17], 2, 16, 128, torch.bfloat16, seed=10)
    kp, vp, table = c.cuda()
    g = torch.Generator().manual_seed(1)
    qs = [torch.randn((2, 8, 128), generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    lens = torch.tensor([4000, 17], dtype=torch.int32, device="cuda")
    want = [paged.paged_attention(q, kp, vp, table, lens) for q in qs]
    for _ in range(3):
        assert same_bits(paged.paged_attention(qs[0], kp, vp, table, lens), want[0])
    held, graphs, outs = [q.clone() for q in qs], [], []
    for q in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged.paged_attention(q, kp, vp, table, lens))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for _ in range(5):
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert same_bits(outs[0], want[0]) and same_bits(outs[1], want[1])
    held[0].copy_(qs[1])
    lens.copy_(torch.tensor([17, 4], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert same_bits(outs[0], paged.paged_attention(qs[1], kp, vp, table, lens))


def test_calls_without_torchs_internal_short_cuts(cuda, monkeypatch):
    """The public calls in their place give the same; outputs never require a gradient."""
    from franken_ocr_b200 import paged

    c = Cache([70, 50], 2, 16, 64, torch.bfloat16, seed=16)
    kp, vp, table = c.cuda()
    q = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    want = paged.paged_attention(q, kp, vp, table, c.lens.cuda())
    assert not want.requires_grad
    monkeypatch.setattr(paged, "_quick_empty", None)
    monkeypatch.setattr(paged, "_device", torch.cuda.current_device)
    monkeypatch.setattr(paged, "_stream", lambda index: torch.cuda.current_stream(index).cuda_stream)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.paged_attention(q, kp, vp, table, c.lens.cuda())
    torch.cuda.synchronize()
    assert same_bits(got, want)


def test_numbers_that_no_c_type_holds_are_refused(cuda):
    """As ValueErrors that name the call, before anything is allocated by them."""
    from franken_ocr_b200 import beam, paged
    from franken_ocr_b200._lib import FocrError

    c = Cache([70, 50], 2, 16, 64, torch.float32, seed=16)
    kp, vp, table = c.cuda()
    q, lens = torch.zeros((2, 4, 64), device="cuda"), c.lens.cuda()
    w = torch.zeros((2, 2, 80), device="cuda")
    with pytest.raises(FocrError, match="scale must be positive and finite"):   # infinite as f32
        paged.paged_attention(q, kp, vp, table, lens, scale=1e39)
    for kw in (dict(window=1 << 70), dict(scale=10 ** 400)):
        with pytest.raises(ValueError, match="paged_attention: an argument is out of range"):
            paged.paged_attention(q, kp, vp, table, lens, **kw)
    for budget in (1 << 40, 1 << 70, 81):
        with pytest.raises(ValueError, match="paged_evict: the new pages hold fewer entries than the budget"):
            paged.paged_evict(kp, vp, table, lens, w, table.clone(), budget)
    with pytest.raises(ValueError, match="paged_evict: an argument is out of range"):
        paged.paged_evict(kp, vp, table, lens, w, table.clone(), 8, sink=1 << 70)
    x, scores = torch.zeros((1, 40, 9), device="cuda"), torch.zeros((1, 40), device="cuda")
    with pytest.raises(ValueError, match="beam_select: an argument is out of range"):
        beam.beam_select(x, scores, end_token=1 << 31)
    for n in (65, 80, 1 << 40):
        with pytest.raises(FocrError, match=f"beams and n are at most 64, not 40 and {n}"):
            beam.beam_select(x, scores, n)
    assert int(torch.zeros(1, device="cuda")) == 0


def test_attention_offsets_past_32_bits(cuda):
    """A pool of over 4 GB whose last pages hold the row."""
    from franken_ocr_b200 import paged

    pages, page, dim = 140000, 64, 256
    kp = torch.empty((pages, 1, page, dim), dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    c = Cache([150], 1, page, dim, torch.float16, seed=11)
    table = c.table.clone()
    for j in range(3):
        kp[pages - 1 - j] = c.k[int(c.table[0, j])].cuda()
        vp[pages - 1 - j] = c.v[int(c.table[0, j])].cuda()
        table[0, j] = pages - 1 - j
    q = torch.randn((1, 2, dim), generator=torch.Generator().manual_seed(1))
    check_attention(c, q, [150], dev=(kp, vp, table.cuda()))
    # and the write: the last slot of the last page
    x = torch.ones((1, 1, dim), device="cuda")
    paged.paged_write(x, x, kp, vp, table.cuda(), torch.tensor([page - 1], dtype=torch.int32, device="cuda"))
    assert bool((kp[pages - 1, 0, page - 1] == 1).all()) and bool((vp[pages - 1, 0, page - 1] == 1).all())


# ---- eviction --------------------------------------------------------------------

def check_evict(c, w, lens, budget, sink, recent, strided=False):
    from franken_ocr_b200 import paged

    rows, heads, width = w.shape
    small = -(-budget // c.page)
    into = torch.tensor(c.spare[:rows * small], dtype=torch.int32).view(rows, small)
    kp, vp, table = c.cuda()
    dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    dw = w.cuda()
    if strided:
        dw = torch.cat([dw, dw], 2)[:, :, :width]
    kept, new, wo = paged.paged_evict(kp, vp, table, dl, dw, into.cuda(), budget, sink=sink, recent=recent)
    k, v = c.k.clone(), c.v.clone()
    want = torch.full((rows, heads, budget), -1, dtype=torch.int32)
    want_w = torch.zeros_like(w)
    for r, n in enumerate(lens):
        for h in range(heads):
            keep = evict_kept(w[r, h], n, budget, sink, recent)
            want[r, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            for j, p in enumerate(keep):
                src, dst = int(c.table[r, p // c.page]), int(into[r, j // c.page])
                k[dst, h, j % c.page] = c.k[src, h, p % c.page]
                v[dst, h, j % c.page] = c.v[src, h, p % c.page]
                want_w[r, h, j] = w[r, h, p]
    assert torch.equal(kept.cpu(), want)
    assert new.tolist() == [min(n, budget) for n in lens]
    assert same_bits(wo, want_w)
    assert same_bits(kp, k) and same_bits(vp, v)


@pytest.mark.parametrize("pool", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,dim,budget,sink,recent", [(16, 64, 20, 4, 8), (7, 80, 1, 0, 0), (16, 128, 33, 0, 33),
                                                         (1, 64, 10, 10, 0), (24, 64, 64, 1, 30)])
def test_evict_matches_the_definition(cuda, pool, page, dim, budget, sink, recent):
    lens = [1, 0, budget, budget + 1, 150, 149]
    rows = len(lens)
    c = Cache(lens, 3, page, dim, DTYPES[pool], seed=budget, spare=rows * -(-budget // page), strided=page == 7)
    w = torch.rand((rows, 3, 160), generator=torch.Generator().manual_seed(budget))
    check_evict(c, w, lens, budget, sink, recent, strided=page == 24)


def test_evict_ties_infinities_and_nan(cuda):
    lens = [90] * 6
    c = Cache(lens, 2, 16, 64, torch.float32, seed=1, spare=6 * 2)
    g = torch.Generator().manual_seed(2)
    w = torch.zeros((6, 2, 90))
    w[1] = torch.randint(0, 3, (2, 90), generator=g).float()
    w[2] = torch.randint(0, 2, (2, 90), generator=g).float() * -0.0          # -0 and 0 are equal
    w[3] = torch.where(torch.rand((2, 90), generator=g) < 0.8, torch.tensor(math.nan), torch.rand((2, 90), generator=g))
    w[4] = torch.where(torch.rand((2, 90), generator=g) < 0.5, torch.tensor(-math.inf), torch.tensor(math.inf))
    w[5] = -torch.rand((2, 90), generator=g) * 1e-42                          # negative subnormals
    check_evict(c, w, lens, 32, 3, 5)


@pytest.mark.parametrize("n,budget", [(5000, 700), (70000, 3), (40000, 39999), (140000, 9000), (300000, 2000)])
def test_evict_long_rows(cuda, n, budget):
    from franken_ocr_b200 import paged

    heads, page = 2, 64
    g = torch.Generator(device="cuda").manual_seed(n)
    pages, small = -(-n // page), -(-budget // page)
    kp = torch.randn((pages + small, heads, page, 64), generator=g, device="cuda", dtype=torch.float16)
    vp = torch.randn((pages + small, heads, page, 64), generator=g, device="cuda", dtype=torch.float16)
    order = torch.randperm(pages + small, generator=g, device="cuda").int()
    table, into = order[None, :pages], order[None, pages:]
    w = torch.rand((1, heads, n + 3), generator=g, device="cuda")
    w[0, 1] = (w[0, 1] * 4).floor()   # many ties
    sink, recent = min(2, budget), (budget - min(2, budget)) // 2
    kept, lens, wo = paged.paged_evict(kp, vp, table, torch.tensor([n], dtype=torch.int32, device="cuda"), w, into,
                                       budget, sink=sink, recent=recent)
    for h in range(heads):
        keep = torch.tensor(evict_kept(w[0, h].cpu(), n, budget, sink, recent))
        assert torch.equal(kept[0, h].cpu().long(), keep)
        keep = keep.cuda()
        at = torch.arange(budget, device="cuda")
        for pool in (kp, vp):
            assert same_bits(pool[into[0].long()[at // page], h, at % page], pool[table[0].long()[keep // page], h, keep % page])
        assert same_bits(wo[0, h, :budget], w[0, h, keep]) and bool((wo[0, h, budget:] == 0).all())
    assert lens.tolist() == [budget]


def test_evict_in_a_replayed_graph_and_beyond_32_bits(cuda):
    """A captured eviction follows its weights; its pages lie past 4 GB."""
    from franken_ocr_b200 import paged

    pages, page, dim = 140000, 64, 256
    kp = torch.empty((pages, 1, page, dim), dtype=torch.float16, device="cuda")
    vp = torch.empty_like(kp)
    table = torch.tensor([[pages - 1, pages - 2, 3]], dtype=torch.int32, device="cuda")
    into = torch.tensor([[pages - 3]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in table[0].tolist():
        kp[p], vp[p] = torch.randn((1, page, dim), generator=g, device="cuda"), torch.randn((1, page, dim), generator=g, device="cuda")
    lens = torch.tensor([150], dtype=torch.int32, device="cuda")
    w = torch.rand((1, 1, 160), generator=g, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, new, wo = paged.paged_evict(kp, vp, table, lens, w, into, 50, sink=2, recent=7)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        keep = evict_kept(w[0, 0].cpu(), 150, 50, 2, 7)
        assert kept[0, 0].tolist() == keep and new.tolist() == [50]
        keep = torch.tensor(keep, device="cuda")
        for pool in (kp, vp):
            assert same_bits(pool[pages - 3, 0, :50], pool[table[0].long()[keep // page], 0, keep % page])
        w.copy_(torch.rand(w.shape, generator=g, device="cuda"))


@pytest.mark.parametrize("pool", ["f32", "f16", "bf16"])
def test_evict_keeps_lost_entries_lost(cuda, pool):
    """Entries on a page outside the pool give NaN before and after, not what the new page
    held; a new page outside the pool is not written."""
    from franken_ocr_b200 import paged

    c = Cache([64] * 4, 2, 16, 64, DTYPES[pool], seed=3, spare=8)
    kp, vp, table = c.cuda()
    kp, vp = kp.nan_to_num(1.0), vp.nan_to_num(1.0)
    before = kp.clone(), vp.clone()
    table[1, 3], table[2, 2] = -1, kp.shape[0]
    into = torch.tensor(c.spare, dtype=torch.int32, device="cuda").view(4, 2)
    into[3, 1] = -5
    w = torch.zeros((4, 2, 64), device="cuda")
    w[2, 0, 32:48] = 1.0           # of row 2 one head keeps entries of the missing page
    kept, lens, _ = paged.paged_evict(kp, vp, table, c.lens.cuda(), w, into, 20, recent=4)
    assert lens.tolist() == [20] * 4
    for r in range(4):
        for h in range(2):
            for j, p in enumerate(kept[r, h].tolist()):
                at, src = int(into[r, j // 16]), int(table[r, p // 16])
                for new, old in zip((kp, vp), before):
                    if not 0 <= at < kp.shape[0]:
                        continue
                    if 0 <= src < kp.shape[0]:
                        assert same_bits(new[at, h, j % 16], old[src, h, p % 16])
                    else:
                        assert bool(new[at, h, j % 16].isnan().all())
    out = paged.paged_attention(torch.ones((4, 2, 64), device="cuda"), kp, vp, into, lens)
    assert out.isnan().any(-1).tolist() == [[False, False], [True, True], [True, False], [True, True]]
    # nothing else is touched
    same = torch.ones(kp.shape[0], dtype=torch.bool)
    same[[p for p in into.view(-1).tolist() if p >= 0]] = False
    for new, old in zip((kp, vp), before):
        assert same_bits(new.cpu()[same], old.cpu()[same])


def test_evict_lengths_out_of_range_and_bad_pages(cuda):
    from franken_ocr_b200 import paged

    c = Cache([64] * 4, 1, 16, 64, torch.float32, seed=3, spare=8)
    kp, vp, table = c.cuda()
    table[3, 1] = -1
    before = kp.clone()
    into = torch.tensor(c.spare, dtype=torch.int32, device="cuda").view(4, 2)
    w = torch.rand((4, 1, 64), generator=torch.Generator().manual_seed(1)).cuda()
    kept, lens, wo = paged.paged_evict(kp, vp, table, torch.tensor([-1, 65, 1000, 64], dtype=torch.int32, device="cuda"),
                                       w, into, 20, recent=20)
    assert lens.tolist() == [0, 0, 0, 20]
    assert bool((kept[:3] == -1).all()) and bool((wo[:3] == 0).all())
    assert kept[3, 0].tolist() == list(range(44, 64))
    assert same_bits(kp[into[:3].reshape(-1).long()], before[into[:3].reshape(-1).long()])
