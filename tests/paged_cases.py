"""Plain 64-bit forms of the paged-cache and beam operators on the host, and
caches with poison wherever a call must not look."""
import math

import numpy as np
import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#: half a step of each type, relative to the value
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in DTYPES.values()}


class Cache:
    """Pools with scattered pages. Slots that hold no entry are NaN, table
    entries that name no page are out of range on either side."""

    def __init__(self, lens, kv_heads, page, dim, dtype, seed=0, capacity=None, spare=0, scale=1.0,
                 strided=False):
        g = torch.Generator().manual_seed(seed)
        self.page, self.heads, self.dim, self.dtype = page, kv_heads, dim, dtype
        rows = len(lens)
        counts = [-(-n // page) for n in lens]
        self.width = -(-(capacity or max(max(lens), 1)) // page)
        total = sum(counts) + spare + 1
        order = torch.randperm(total, generator=g).tolist()
        self.spare = [order.pop() for _ in range(spare)]
        self.table = torch.full((rows, self.width), 2**31 - 1, dtype=torch.int32)
        self.table[:, 1::2] = -7
        if strided:  # K and V of a page beside one another, heads apart
            both = torch.full((total, kv_heads, 2, page, dim), math.nan, dtype=dtype)
            self.k, self.v = both[:, :, 0], both[:, :, 1]
        else:
            self.k = torch.full((total, kv_heads, page, dim), math.nan, dtype=dtype)
            self.v = self.k.clone()
        for r, n in enumerate(lens):
            for j in range(counts[r]):
                self.table[r, j] = order.pop()
                live = min(page, n - j * page)
                shape = (kv_heads, live, dim)
                at = int(self.table[r, j])
                self.k[at, :, :live] = (torch.randn(shape, generator=g) * scale).to(dtype)
                self.v[at, :, :live] = torch.randn(shape, generator=g).to(dtype)
        self.lens = torch.tensor(lens, dtype=torch.int32)

    def cuda(self):
        """The device's copy: k, v with this cache's strides, and the table."""
        def up(x):
            y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
            return y.copy_(x)
        if self.k.stride()[1] != self.page * self.dim:
            base = torch.empty((self.k.shape[0], self.heads, 2, self.page, self.dim), dtype=self.dtype,
                               device="cuda")
            base[:, :, 0], base[:, :, 1] = self.k, self.v
            return base[:, :, 0], base[:, :, 1], self.table.cuda()
        return up(self.k), up(self.v), self.table.cuda()

    def row(self, r, positions, which="k"):
        """[heads, positions, dim] in 64 bits."""
        pool = self.k if which == "k" else self.v
        positions = torch.as_tensor(positions, dtype=torch.long)
        pages = self.table[r].long()[positions // self.page]
        return pool[pages, :, positions % self.page].double().permute(1, 0, 2)


def visible(n, ref=0, window=0):
    if not window:
        return list(range(max(n, 0)))
    return [j for j in range(n) if j < ref or j >= n - window]


def attention(cache, q, lens, scale, refs=None, window=0):
    """(out, probabilities summed over a kv head's query heads as {(r, h): (positions, p)},
    a bound on the kernel's error): f64."""
    rows, q_heads, dim = q.shape
    group = q_heads // cache.heads
    out = torch.zeros((rows, q_heads, dim), dtype=torch.float64)
    bound = torch.zeros((rows, q_heads, dim), dtype=torch.float64)
    probs = {}
    eps = 2.0 ** -24
    for r in range(rows):
        at = visible(int(lens[r]), 0 if refs is None else int(refs[r]), window)
        if not at:
            continue
        k, v = cache.row(r, at), cache.row(r, at, "v")
        for h in range(cache.heads):
            qs = q[r, h * group:(h + 1) * group].double()
            s = scale * qs @ k[h].T
            p = torch.softmax(s, -1)
            out[r, h * group:(h + 1) * group] = p @ v[h]
            probs[r, h] = (at, p.sum(0))
            # A score is a dot of dim products and one product with the scale:
            # (dim + 2) roundings of sums no larger than scale * |q| . |k|. A
            # probability is exp of a difference of two scores (2^-22 for the
            # exponential, and 2^-24 of its argument, which is no larger than the
            # scores' span); numerator and denominator add n terms each. With a
            # 16-bit query a probability enters the product as two parts of 8
            # bits or more, which leaves 2^-18 of it.
            ds = (dim + 2) * eps * (scale * qs.abs() @ k[h].abs().T).amax(-1, keepdim=True)
            span = s.amax(-1, keepdim=True) - s.amin(-1, keepdim=True)
            rel = 2 * ds + 2 * (len(at) + 16) * eps + 2.0 ** -21 + 2 * eps * span
            if q.dtype != torch.float32:
                rel = rel + 2.0 ** -18
            bound[r, h * group:(h + 1) * group] = rel * (p @ v[h].abs()) + 1e-30
    bound = bound + out.abs() * HALF_STEP[q.dtype]
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half the smallest subnormal
    return out, probs, bound


def evict_kept(w, n, budget, sink, recent):
    """The kept positions of one row and head."""
    if n <= budget:
        return list(range(n))
    middle = [(-math.inf if math.isnan(x) else x, -j) for j, x in enumerate(w[:n].tolist())]
    middle = middle[sink:n - recent]
    # NaN below every number, -inf included
    nan = [math.isnan(float(w[-j])) for _, j in middle]
    order = sorted(range(len(middle)), key=lambda i: (nan[i], -middle[i][0], -middle[i][1]))
    chosen = [-middle[i][1] for i in order[:budget - sink - recent]]
    return sorted(list(range(sink)) + chosen + list(range(n - recent, n)))


def select(logits, scores, n, done=None, end=1):
    """Per entry the ranked (score, beam, token), by the definition."""
    batch, beams, vocab = logits.shape
    big = float(np.finfo(np.float32).max)
    out = []
    for b in range(batch):
        found = []
        for i in range(beams):
            cum = float(scores[b, i])
            if not math.isfinite(cum):
                continue
            if done is not None and bool(done[b, i]):
                found.append((-cum, i, 0.0, end))
                continue
            x = logits[b, i].double().numpy()
            x = np.where(np.isposinf(x), big, x)
            ok = np.isfinite(x)
            if not ok.any():
                continue
            m = x[ok].max()
            norm = math.log(np.exp(x[ok] - m).sum())
            for t in np.argsort(np.where(ok, -x, np.inf), kind="stable")[:n]:
                if ok[t]:
                    found.append((-(cum + ((x[t] - m) - norm)), i, -x[t], int(t)))
        found.sort()
        out.append([(-f[0], f[1], f[3]) for f in found[:n]])
    return out
