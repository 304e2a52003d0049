"""What a server of the decoder calls around its projections when many streams
share one pool of K/V pages and decode with beams: new keys and values written
into pages, attention of each row's new token over its pages, eviction of the
cache's least attended entries, the selection of the next beams over beams and
vocabulary, and the reordering of the beams' pages.

``run`` computes one call in plain torch where ``own`` is false and through the
package's public functions where it is true.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # one decode step of a continuous batch: 64 streams append a token each
        # (the decoder's 10 heads of 128, f32 activations into bf16 pages)
        dict(name="write step 64", op="write", rows=64, tokens=64, prompt=False, kv_heads=10, head_dim=128,
             page=16, src="f32", pool="bf16"),
        # prompts of several streams entering the cache in one padded call
        dict(name="write prompts 12000", op="write", rows=9, tokens=12000, prompt=True, kv_heads=8, head_dim=128,
             page=64, src="bf16", pool="bf16"),
        # one stream of the 12-layer decoder: 1024 prompt rows and a window of
        # 128 behind them, everything in f32: the smallest call
        dict(name="attend 1 stream", op="attend", rows=1, low=1290, high=1290, ref=1024, window=128, q_heads=10,
             kv_heads=10, head_dim=128, page=16, q="f32", pool="f32", weights=False, empty=False),
        # a continuous batch of ragged streams, idle slots among them
        dict(name="attend 64 streams", op="attend", rows=64, low=1, high=4097, ref=0, window=0, q_heads=10,
             kv_heads=10, head_dim=128, page=16, q="f32", pool="bf16", weights=False, empty=True),
        # grouped heads, with the weights that eviction goes by
        dict(name="attend grouped weights", op="attend", rows=32, low=200, high=16385, ref=0, window=0, q_heads=32,
             kv_heads=8, head_dim=128, page=32, q="bf16", pool="bf16", weights=True, empty=False),
        # long documents
        dict(name="attend 131072", op="attend", rows=8, low=131000, high=131072, ref=0, window=0, q_heads=64,
             kv_heads=8, head_dim=128, page=64, q="bf16", pool="bf16", weights=False, empty=False),
        # a batch whose caches go back to their budget, some still below it
        dict(name="evict 16 streams", op="evict", rows=16, low=500, high=4097, budget=1024, sink=4, recent=256,
             kv_heads=10, head_dim=128, page=16, pool="bf16"),
        # long prompts compressed once, right after the prefill
        dict(name="evict 131072", op="evict", rows=2, low=131000, high=131072, budget=8192, sink=16, recent=1024,
             kv_heads=8, head_dim=128, page=64, pool="f16"),
        # one page of OCR decoded with 4 beams over the decoder's vocabulary
        dict(name="select 1x4", op="select", batch=1, beams=4, n=4, vocab=129280, logits="f32", done=False),
        # a batch with 8 beams each, twice as many candidates as beams, some beams ended
        dict(name="select 32x8", op="select", batch=32, beams=8, n=16, vocab=129280, logits="f32", done=True),
        # the beams of one page, all 12 layers
        dict(name="reorder 1x4", op="reorder", batch=1, beams=4, layers=12, low=1290, high=1290, kv_heads=10,
             head_dim=128, page=16, pool="f32", weights=False),
        # a batch of beams that carries the eviction weights along
        dict(name="reorder 32x8 weights", op="reorder", batch=32, beams=8, layers=4, low=300, high=1500, kv_heads=8,
             head_dim=128, page=64, pool="bf16", weights=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["write", "attend", "attend", "attend", "evict", "select", "select", "reorder"])
    heads = rng.choice([1, 2, 4, 5, 8, 10, 16])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256])
    pool = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "write":
        prompt = rng.random() < 0.5
        rows = _log(rng, 1, 16) if prompt else _log(rng, 1, 512)
        return dict(op=op, rows=rows, tokens=_log(rng, rows, 12000) if prompt else rows, prompt=prompt, kv_heads=heads,
                    head_dim=dim, page=page, src=rng.choice(["f32", "f32", pool]), pool=pool)
    if op == "attend":
        size = BYTES[pool] * heads * dim * 2
        rows = _log(rng, 1, 256)
        high = _log(rng, 1, max(2, min(131072, int(3e9 / size / rows))))
        window = rng.choice([0, 0, 0, 128, 1000])
        group = rng.choice([1, 1, 1, 2, 3, 4, 7, 8, 16])
        return dict(op=op, rows=rows, low=min(high, rng.choice([1, high // 2 + 1, high])), high=high,
                    ref=rng.choice([0, 64, 1024]) if window else 0, window=window, q_heads=heads * group, kv_heads=heads,
                    head_dim=dim, page=page, q=rng.choice(["f32", pool]), pool=pool, weights=rng.random() < 0.3,
                    empty=rows > 2 and rng.random() < 0.3)
    if op == "evict":
        size = BYTES[pool] * heads * dim * 2
        rows = _log(rng, 1, 32)
        high = _log(rng, 2, max(4, min(131072, int(1e9 / size / rows))))
        budget = _log(rng, 1, high)
        sink = rng.choice([0, min(4, budget)])
        return dict(op=op, rows=rows, low=rng.choice([1, high // 2 + 1, high]), high=high, budget=budget, sink=sink,
                    recent=int((budget - sink) * rng.choice([0.0, 0.25, 0.5, 1.0])), kv_heads=heads, head_dim=dim,
                    page=page, pool=pool)
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 10, 16])
        vocab = _log(rng, 2, 150000)
        return dict(op=op, batch=_log(rng, 1, max(1, min(64, 33_000_000 // beams // vocab))), beams=beams,
                    n=rng.choice([beams, 2 * beams, beams + 1]), vocab=vocab, logits=rng.choice(["f32", "f32", "f16", "bf16"]),
                    done=rng.random() < 0.5)
    high = _log(rng, 1, 8192)
    batch, beams = _log(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8])
    # the cache is far larger than what is moved: keep the pages within a few GB
    layers = rng.choice([1, 2, 4, 12])
    while layers > 1 and layers * batch * beams * (high + 2 * page) * heads * dim * BYTES[pool] > 1.5e9:
        layers -= 1
    high = max(1, min(high, int(1.5e9 / (layers * batch * beams * heads * dim * BYTES[pool])) - 2 * page))
    return dict(op=op, batch=batch, beams=beams, layers=layers, low=rng.choice([1, high]), high=high, kv_heads=heads,
                head_dim=dim, page=page, pool=pool, weights=rng.random() < 0.4)


# ---- what a user's program holds ----------------------------------------------

def _lens(case, rows):
    """Lengths spread over [low, high]; every seventh stream idle where `empty`."""
    low, high = case["low"], case["high"]
    lens = [low + int((high - low) * ((0.618033988749895 * (i + 1)) % 1.0) + 0.5) for i in range(rows)]
    return [0 if case.get("empty") and i % 7 == 5 else n for i, n in enumerate(lens)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _randn(gen, shape, dtype, scale=1.0):
    """Normal values, drawn in blocks so that a large cache needs no f32 copy of itself."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for part in flat.split(1 << 28):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale))
    return out


def _tables(gen, counts, width, spare=0):
    """Page tables whose pages lie scattered over the pool; -1 behind each row's
    last page. Returns (table, a list of `spare` free pages, pages in the pool)."""
    total = sum(counts) + spare
    order = torch.randperm(max(1, total), generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table, order[at:at + spare], max(1, total)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    if op == "select":
        rows = case["batch"] * case["beams"]
        # a language model's logits: a broad body and a few tokens far above it
        x = torch.randn((rows, case["vocab"]), generator=gen, device="cuda") * 2.0
        x += 4.0 * torch.rand(x.shape, generator=gen, device="cuda").pow_(64)
        s["x"] = x.to(TYPES[case["logits"]]).view(case["batch"], case["beams"], case["vocab"])
        s["scores"] = torch.randn((case["batch"], case["beams"]), generator=gen, device="cuda") * 3.0 - 20.0
        ended = torch.rand(s["scores"].shape, generator=gen, device="cuda") < 0.2
        s["done"] = ended if case["done"] else None
        return s
    heads, dim, page, dtype = case["kv_heads"], case["head_dim"], case["page"], TYPES[case["pool"]]
    if op == "write":
        rows, tokens = case["rows"], case["tokens"]
        if case["prompt"]:
            # prompts behind one another, each stream's prompt entering an
            # empty cache; a twentieth of the tokens is padding, with row -1
            each = [(i + 1) * tokens // rows - i * tokens // rows for i in range(rows)]
            row = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(each)])
            pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in each])
            row[19::20] = -1
            s["row"], s["pos"] = row.cuda(), pos.cuda()
            most = max(each)
        else:
            most = 4096
            s["row"] = None
            s["pos"] = torch.randint(0, most, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        width = most // page + 1
        if case["prompt"]:
            s["table"], _, pages = _tables(gen, [width] * rows, width)
        else:
            # only the page that is written exists in this pool
            s["table"] = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
            s["table"][torch.arange(rows, device="cuda"), (s["pos"] // page).long()] = torch.randperm(
                rows, generator=gen, device="cuda").to(torch.int32)
            pages = rows
        s["k"] = _randn(gen, (tokens, heads, dim), TYPES[case["src"]])
        s["v"] = _randn(gen, (tokens, heads, dim), TYPES[case["src"]])
        s["kp"] = _randn(gen, (pages, heads, page, dim), dtype)
        s["vp"] = _randn(gen, (pages, heads, page, dim), dtype)
        return s
    if op == "reorder":
        rows = case["batch"] * case["beams"]
        # the beams of one entry are equally long
        each = [n for n in _lens(case, case["batch"]) for _ in range(case["beams"])]
        width = case["high"] // page + 2
        s["table"], s["fresh"], pages = _tables(gen, [-(-n // page) for n in each], width, spare=rows)
        s["lens"] = _ints(each)
        shape = (case["layers"], pages, heads, page, dim)
        s["kp"], s["vp"] = _randn(gen, shape, dtype), _randn(gen, shape, dtype)
        s["parent"] = torch.randint(0, case["beams"], (case["batch"], case["beams"]), generator=gen, device="cuda",
                                    dtype=torch.int32)
        s["w"] = None
        if case["weights"]:
            s["w"] = torch.rand((case["layers"], rows, heads, case["high"] + 5), generator=gen, device="cuda")
        return s
    rows = case["rows"]
    lens = _lens(case, rows)
    s["lens"] = _ints(lens)
    if op == "attend":
        width = -(-case["high"] // page)
        s["table"], _, pages = _tables(gen, [-(-n // page) for n in lens], width)
        s["refs"] = _ints([case["ref"]] * rows) if case["ref"] else None
        s["qs"] = _randn(gen, (rows, case["q_heads"], dim), TYPES[case["q"]], 1.5)
        s["w"] = torch.rand((rows, heads, width * page), generator=gen, device="cuda") if case["weights"] else None
    else:
        width, small = -(-case["high"] // page), -(-case["budget"] // page)
        counts = [-(-n // page) for n in lens] + [small] * rows
        both, _, pages = _tables(gen, counts, max(width, small))
        s["table"], s["into"] = both[:rows, :width].contiguous(), both[rows:, :small].contiguous()
        # accumulated probabilities: a heavy tail, and entries that were hardly
        # ever looked at, all with the same value
        w = torch.exp(2.0 * torch.randn((rows, heads, case["high"]), generator=gen, device="cuda") - 4.0)
        s["w"] = torch.where(w < 0.002, torch.zeros_like(w), w)
    shape = (pages, heads, page, dim)
    s["kp"], s["vp"] = _randn(gen, shape, dtype), _randn(gen, shape, dtype)
    return s


# ---- one call ------------------------------------------------------------------

def run(s):
    op = s["op"]
    if own:
        from franken_ocr_b200 import beam, paged

        if op == "write":
            paged.paged_write(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["pos"], row=s["row"])
            return s["kp"], s["vp"]
        if op == "attend":
            out = paged.paged_attention(s["qs"], s["kp"], s["vp"], s["table"], s["lens"], ref_lens=s["refs"],
                                        window=s["window"], weights=s["w"])
            return out if s["w"] is None else (out, s["w"])
        if op == "evict":
            kept, lens, w = paged.paged_evict(s["kp"], s["vp"], s["table"], s["lens"], s["w"], s["into"], s["budget"],
                                              sink=s["sink"], recent=s["recent"])
            return kept, lens, w, s["kp"], s["vp"]
        if op == "select":
            return beam.beam_select(s["x"], s["scores"], n=s["n"], done=s["done"], end_token=1)
        table, lens, w = beam.beam_reorder(s["kp"], s["vp"], s["table"], s["lens"], s["parent"], s["fresh"],
                                           weights=s["w"])
        return [t for t in (table, lens, w, s["kp"], s["vp"]) if t is not None]
    if op == "write":
        return _write(s)
    if op == "attend":
        return _attend(s)
    if op == "evict":
        return _evict(s)
    return _select(s) if op == "select" else _reorder(s)


def _write(s):
    page, pos = s["kp"].shape[2], s["pos"].long()
    row = torch.arange(pos.shape[0], device="cuda") if s["row"] is None else s["row"].long()
    live = row >= 0
    row, pos = row[live], pos[live]
    at = s["table"][row, pos // page].long()
    s["kp"][at, :, pos % page] = s["k"][live].to(s["kp"].dtype)
    s["vp"][at, :, pos % page] = s["v"][live].to(s["vp"].dtype)
    return s["kp"], s["vp"]


def _rows_of(pages, table):
    """[rows, heads, width * page, dim] of the pages that the tables name."""
    x = pages[table.clamp(min=0).long()]
    r, w, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(r, h, w * p, d)


def _attend(s):
    k, v = _rows_of(s["kp"], s["table"]).float(), _rows_of(s["vp"], s["table"]).float()
    rows, heads, span, dim = k.shape
    q = s["qs"].float().view(rows, heads, -1, dim)
    at = torch.arange(span, device="cuda")[None]
    lens = s["lens"][:, None]
    seen = at < lens
    if s["window"]:
        refs = 0 if s["refs"] is None else s["refs"][:, None]
        seen = seen & ((at < refs) | (at >= lens - s["window"]))
    seen = seen[:, None, None, :]
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(dim)
    x = torch.where(seen, x, torch.full_like(x, -torch.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    p = torch.where(seen, p / p.sum(-1, keepdim=True), torch.zeros_like(p))
    out = torch.matmul(p, v).reshape(rows, -1, dim).to(s["qs"].dtype)
    if s["w"] is None:
        return out
    s["w"] += p.sum(2)
    return out, s["w"]


def _evict(s):
    w, lens, budget = s["w"], s["lens"].long()[:, None, None], s["budget"]
    rows, heads, span = w.shape
    page = s["kp"].shape[2]
    at = torch.arange(span, device="cuda")[None, None]
    safe = (at < s["sink"]) | (at >= lens - s["recent"])
    key = torch.where(safe, torch.full_like(w, torch.inf), w)
    key = torch.where(at < lens, key, torch.full_like(w, -torch.inf))
    first = torch.sort(key, dim=-1, descending=True, stable=True).indices
    first = torch.nn.functional.pad(first, (0, max(0, budget - span)))[..., :budget]
    slot = torch.arange(budget, device="cuda")[None, None]
    live = slot < lens
    kept = torch.sort(torch.where(live, first, torch.full_like(first, span)), dim=-1).values
    live = live.expand(kept.shape)
    r, h, j = torch.nonzero(live, as_tuple=True)
    src = kept[r, h, j]
    there, here = s["table"][r, src // page].long(), s["into"][r, j // page].long()
    s["kp"][here, h, j % page] = s["kp"][there, h, src % page]
    s["vp"][here, h, j % page] = s["vp"][there, h, src % page]
    out = torch.zeros_like(w)
    out[r, h, j] = w[r, h, src]
    kept = torch.where(live, kept, torch.full_like(kept, -1)).int()
    return kept, s["lens"].clamp(max=budget), out, s["kp"], s["vp"]


def _select(s):
    x, n = s["x"], s["n"]
    batch, beams, vocab = x.shape
    most = min(n, vocab)
    d = x.double()
    top = d.amax(-1, keepdim=True)
    norm = torch.log(torch.exp(d - top).sum(-1, keepdim=True))
    best, token = torch.sort(x, dim=-1, descending=True, stable=True)
    best, token = best[..., :most].double(), token[..., :most]
    score = s["scores"].double()[..., None] + ((best - top) - norm)
    if s["done"] is not None:
        # an ended beam offers itself once, unchanged
        place = torch.arange(most, device="cuda")[None, None]
        ended = s["done"][..., None]
        itself = torch.where(place == 0, s["scores"].double()[..., None], torch.full_like(score, -torch.inf))
        score = torch.where(ended, itself, score)
        token = torch.where(ended, torch.ones_like(token), token)
    score, token = score.reshape(batch, -1), token.reshape(batch, -1)
    short = max(0, n - score.shape[1])
    score = torch.nn.functional.pad(score, (0, short), value=-torch.inf)
    token = torch.nn.functional.pad(token, (0, short))
    score, at = torch.sort(score, dim=-1, descending=True, stable=True)
    score, at = score[:, :n], at[:, :n]
    live = score > -torch.inf
    parent = torch.where(live, at // most, torch.full_like(at, -1)).int()
    token = torch.where(live, token.gather(1, at), torch.full_like(at, -1)).int()
    return score.float(), parent, token


def _reorder(s):
    batch, beams = s["parent"].shape
    page, width = s["kp"].shape[3], s["table"].shape[1]
    base = torch.arange(batch, device="cuda")[:, None] * beams
    src = (base + s["parent"].long()).view(-1)
    lens = s["lens"][src]
    last = (lens // page).long()
    column = torch.arange(width, device="cuda")[None]
    table = torch.where(column < last[:, None], s["table"][src], torch.full_like(s["table"], -1))
    table = torch.where(column == last[:, None], s["fresh"][:, None], table)
    tail = s["table"][src, last].long().clamp(min=0)
    slot = torch.arange(page, device="cuda")[None]
    row, j = torch.nonzero(slot < (lens.long() % page)[:, None], as_tuple=True)
    here = s["fresh"].long()[row]
    s["kp"][:, here, :, j] = s["kp"][:, tail[row], :, j]
    s["vp"][:, here, :, j] = s["vp"][:, tail[row], :, j]
    if s["w"] is None:
        return [table, lens, s["kp"], s["vp"]]
    at = torch.arange(s["w"].shape[3], device="cuda")[None, None, None]
    w = torch.where(at < lens[None, :, None, None], s["w"][:, src], torch.zeros_like(s["w"]))
    return [table, lens, w, s["kp"], s["vp"]]


# ---- what a call cannot do without ------------------------------------------------

def work(case):
    op = case["op"]
    if op == "select":
        rows = case["batch"] * case["beams"]
        return {"bytes": rows * case["vocab"] * BYTES[case["logits"]] + 12 * case["batch"] * case["n"],
                "flops": 4.0 * rows * case["vocab"]}
    heads, dim, page, size = case["kv_heads"], case["head_dim"], case["page"], BYTES[case["pool"]]
    if op == "write":
        live = case["tokens"] - (case["tokens"] // 20 if case["prompt"] else 0)
        return {"bytes": 2 * live * heads * dim * (BYTES[case["src"]] + size) + 12 * case["tokens"], "flops": 0}
    if op == "reorder":
        lens = [n for n in _lens(case, case["batch"]) for _ in range(case["beams"])]
        moved = sum(n % page for n in lens)
        total = case["layers"] * 2 * moved * heads * dim * size * 2 + 8 * len(lens) * (case["high"] // page + 2)
        if case["weights"]:
            total += case["layers"] * heads * (sum(lens) + len(lens) * (case["high"] + 5)) * 4
        return {"bytes": total, "flops": 0}
    lens = _lens(case, case["rows"])
    if op == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        read = sum(lens) * heads * 4
        return {"bytes": read + kept * heads * (dim * size * 4 + 4) + case["rows"] * heads * case["high"] * 4, "flops": 0}
    if case["window"]:
        lens = [min(n, case["ref"]) + max(0, n - max(min(n, case["ref"]), n - case["window"])) for n in lens]
    seen = sum(lens)
    total = seen * heads * dim * size * 2 + 2 * case["rows"] * case["q_heads"] * dim * BYTES[case["q"]] + 4 * seen // page
    if case["weights"]:
        total += seen * heads * 8
    return {"bytes": total, "flops": 4.0 * seen * case["q_heads"] * dim}


# ---- the definitions, in 64 bits ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "select":
        # log p = x - log sum exp x, the candidates of one entry ranked together
        scores, parents, tokens = [], [], []
        for b in range(case["batch"]):
            found = []
            for i in range(case["beams"]):
                total = float(s["scores"][b, i])
                if s["done"] is not None and bool(s["done"][b, i]):
                    found.append((-total, i, 0, 1))
                    continue
                x = s["x"][b, i].double()
                p = x - torch.logsumexp(x, 0)
                value = torch.topk(x, min(case["n"], case["vocab"])).values[-1]
                for t in torch.nonzero(x >= value)[:, 0].tolist()[:20000]:
                    found.append((-(total + float(p[t])), i, -float(x[t]), t))
            found = sorted(found)[:case["n"]]
            missing = case["n"] - len(found)
            scores.append([-f[0] for f in found] + [-math.inf] * missing)
            parents.append([f[1] for f in found] + [-1] * missing)
            tokens.append([f[3] for f in found] + [-1] * missing)
        return torch.tensor(scores, dtype=torch.float64), torch.tensor(parents), torch.tensor(tokens)
    if op == "attend":
        dim, page, group = case["head_dim"], case["page"], case["q_heads"] // case["kv_heads"]
        out = torch.zeros((case["rows"], case["q_heads"], dim), dtype=torch.float64, device="cuda")
        w = None if s["w"] is None else s["w"].double()
        for r, n in enumerate(s["lens"].tolist()):
            at = list(range(n))
            if case["window"]:
                at = [j for j in at if j < case["ref"] or j >= n - case["window"]]
            if not at:
                continue
            at = torch.tensor(at, device="cuda")
            pages = s["table"][r].long()[at // page]
            for h in range(case["kv_heads"]):
                k, v = s["kp"][pages, h, at % page].double(), s["vp"][pages, h, at % page].double()
                p = torch.softmax(s["qs"][r, h * group:(h + 1) * group].double() @ k.T / math.sqrt(dim), -1)
                out[r, h * group:(h + 1) * group] = p @ v
                if w is not None:
                    w[r, h, at] += p.sum(0)
        return out if w is None else (out, w)
    kp, vp, page = s["kp"].double(), s["vp"].double(), case["page"]
    if op == "write":
        row = list(range(case["tokens"])) if s["row"] is None else s["row"].tolist()
        table, pos = s["table"].tolist(), s["pos"].tolist()
        live = [t for t, r in enumerate(row) if r >= 0]
        here = torch.tensor([table[row[t]][pos[t] // page] for t in live], device="cuda")
        slot = torch.tensor([pos[t] % page for t in live], device="cuda")
        kp[here, :, slot], vp[here, :, slot] = s["k"][live].double(), s["v"][live].double()
        return kp, vp
    if op == "evict":
        budget = case["budget"]
        kept = torch.full((case["rows"], case["kv_heads"], budget), -1)
        w = torch.zeros_like(s["w"], dtype=torch.float64)
        lens = s["lens"].tolist()
        for r, n in enumerate(lens):
            for h in range(case["kv_heads"]):
                if n <= budget:
                    keep = torch.arange(n)
                else:
                    end = n - case["recent"]
                    middle = s["w"][r, h, case["sink"]:end].double().cpu()
                    order = sorted(zip((-middle).tolist(), range(case["sink"], end)))
                    chosen = [j for _, j in order[:budget - case["sink"] - case["recent"]]]
                    keep = torch.tensor(sorted(list(range(case["sink"])) + chosen + list(range(end, n))))
                kept[r, h, :len(keep)] = keep
                keep = keep.cuda()
                to = torch.arange(len(keep), device="cuda")
                there, here = s["table"][r].long()[keep // page], s["into"][r].long()[to // page]
                kp[here, h, to % page], vp[here, h, to % page] = kp[there, h, keep % page], vp[there, h, keep % page]
                w[r, h, to] = s["w"][r, h, keep].double()
        return kept, torch.tensor([min(n, budget) for n in lens]), w, kp, vp
    beams, rows = case["beams"], case["batch"] * case["beams"]
    parent, lens, old = s["parent"].view(-1).tolist(), s["lens"].tolist(), s["table"].tolist()
    fresh, new = s["fresh"].tolist(), []
    w = None if s["w"] is None else torch.zeros_like(s["w"], dtype=torch.float64)
    for i in range(rows):
        p = i // beams * beams + parent[i]
        full, rest = divmod(lens[p], page)
        new.append(old[p][:full] + [fresh[i]] + [-1] * (len(old[p]) - full - 1))
        if rest:
            kp[:, fresh[i], :, :rest] = kp[:, old[p][full], :, :rest]
            vp[:, fresh[i], :, :rest] = vp[:, old[p][full], :, :rest]
        if w is not None:
            w[:, i, :, :lens[p]] = s["w"][:, p, :, :lens[p]].double()
    got = [torch.tensor(new), torch.tensor([lens[i // beams * beams + parent[i]] for i in range(rows)]), w, kp, vp]
    return [t for t in got if t is not None]
