"""The paged cache's operators in 64 bits, from their formulas, entry by entry; shared by its tests."""

from __future__ import annotations

import torch

DEV = torch.device("cuda", 0)


class Batch:
    """Sequences with `counts` new tokens and `lengths` entries over a pool of NaN, in pages of any order; the dense
    keys and values of every entry (`keys[s]`, `values[s]` [entries, kv_heads, head_dim]) and a pool that holds
    them (`fill`)."""

    def __init__(self, counts, lengths, kv_heads, head_dim, page, dtype, seed=0, spare=2, layers=None, width=None):
        from linnet_amd.torch.paged import PagedCache

        self.counts, self.lengths_list, self.page, self.dtype = list(counts), list(lengths), page, dtype
        self.kv_heads, self.head_dim = kv_heads, head_dim
        g = torch.Generator().manual_seed(seed)
        self.g = g
        need = [-(-max(n, 0) // page) for n in lengths]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.pages = total
        width = max(need + [1]) if width is None else width
        rows, at = [], 0
        for n in need:
            rows.append((order[at : at + n] + [-1] * width)[:width])
            at += n
        self.rows = rows
        self.tables = torch.tensor(rows, dtype=torch.int32).reshape(len(rows), width).to(DEV)
        self.lengths = torch.tensor(self.lengths_list, dtype=torch.int32, device=DEV)
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        self.starts_list = starts
        self.starts = torch.tensor(starts, dtype=torch.int32, device=DEV)
        self.tokens = starts[-1]
        lead = (total,) if layers is None else (layers, total)
        k = torch.full((*lead, kv_heads, head_dim // 8, page, 8), float("nan"), dtype=dtype)
        v = torch.full((*lead, kv_heads, page // 8, head_dim, 8), float("nan"), dtype=dtype)
        self.cache = PagedCache(k.to(DEV), v.to(DEV))
        self.keys = [self.random(max(n, 0), kv_heads, head_dim) for n in lengths]
        self.values = [self.random(max(n, 0), kv_heads, head_dim) for n in lengths]

    def random(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype)

    def fill(self):
        """Every entry into the pool, entry by entry."""
        k, v = self.cache.k.cpu(), self.cache.v.cpu()
        for row, keys, values in zip(self.rows, self.keys, self.values):
            for e in range(keys.shape[0]):
                p, place = row[e // self.page] if e // self.page < len(row) else -1, e % self.page
                if 0 <= p < k.shape[0]:
                    k[p, :, :, place] = keys[e].view(self.kv_heads, -1, 8)
                    v[p, :, place // 8, :, place % 8] = values[e]
        self.cache.k.copy_(k)
        self.cache.v.copy_(v)
        return self

    def there(self, s, e):
        """Whether entry e of sequence s has a page in the pool."""
        row = self.rows[s]
        return 0 <= e // self.page < len(row) and 0 <= row[e // self.page] < self.pages


def entry_of(cache_k, cache_v, page, place):
    """An entry's key and value [kv_heads, head_dim] out of a pool on the CPU."""
    return cache_k[page, :, :, place].flatten(1), cache_v[page, :, place // 8, :, place % 8]


def paths_of(parents, window):
    """Each node's path (itself first) and depth, of one sequence's parents."""
    paths = []
    for i in range(len(parents)):
        path, j = [], i
        while j >= 0:
            path.append(j)
            j = parents[j] if 0 <= parents[j] < j else -1
        paths.append((path[:window] if window else path, len(path) - 1))
    return paths


def seen_of(batch, s, window, parents=None):
    """[new tokens, entries]: which entries of sequence s its new tokens see."""
    n, length = batch.counts[s], max(batch.lengths_list[s], 0)
    base = length - n
    entries = torch.arange(length)
    there = torch.tensor([batch.there(s, e) for e in range(length)], dtype=torch.bool)
    seen = torch.zeros(n, length, dtype=torch.bool)
    paths = paths_of(parents, window) if parents is not None else None
    for i in range(n):
        if paths is None:
            seen[i] = (entries <= base + i) & ((entries > base + i - window) if window else True)
        elif i < 256:
            path, depth = paths[i]
            seen[i] = (entries < base) & ((entries > base + depth - window) if window else True)
            for j in path:
                if base + j >= 0:
                    seen[i, base + j] = True
    return seen & there


def attention(batch, q, scale=None, window=0, sinks=None, parents=None):
    """(out, tolerance) [tokens, heads * head_dim] in 64 bits. The tolerance, from the kernel's arithmetic:
    each weight is rounded to 16 bits (u = eps / 2 relative; f16 below its least normal number, 2^-25 of a
    weight of 1 or more), the output too; scores are f32 sums of head_dim products; exp2 and its argument are
    f32; sums over n entries are f32."""
    hd, heads = batch.head_dim, q.shape[1] // batch.head_dim
    group = heads // batch.kv_heads
    scale = hd**-0.5 if scale is None else scale
    u = torch.finfo(batch.dtype).eps / 2
    out = torch.zeros(q.shape[0], heads, hd, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for s, n in enumerate(batch.counts):
        if n == 0:
            continue
        first = batch.starts_list[s]
        seen = seen_of(batch, s, window, None if parents is None else parents[first : first + n])
        x = q[first : first + n].double().cpu().view(n, heads, hd)
        for h in range(heads):
            k, v = batch.keys[s][:, h // group].double(), batch.values[s][:, h // group].double()
            score = (x[:, h] @ k.t()) * scale
            score = torch.where(seen, score, -torch.inf)
            top = score.amax(-1, keepdim=True) if score.shape[1] else torch.full((n, 1), -torch.inf, dtype=torch.float64)
            if sinks is not None:
                top = torch.maximum(top, sinks[h].double().cpu())
            e = torch.where(seen, torch.exp(score - torch.where(top == -torch.inf, 0.0, top)), 0.0)
            total = e.sum(-1, keepdim=True)
            some = seen.any(-1, keepdim=True)
            if sinks is not None:
                total = total + torch.exp(sinks[h].double().cpu() - top)
            w = torch.where(some, e / torch.where(some, total, 1.0), 0.0)
            # Values that a row does not see count nothing, whatever they are.
            o = torch.stack([torch.where(w[i][:, None] > 0, w[i][:, None] * v, 0.0).sum(0) for i in range(n)])
            size = torch.stack([torch.where(w[i][:, None] > 0, w[i][:, None] * v.abs(), 0.0).sum(0) for i in range(n)])
            out[first : first + n, h] = o
            dots = (x[:, h].abs() @ k.abs().t() * scale).where(seen, torch.tensor(0.0, dtype=torch.float64))
            worst = dots.amax(-1, keepdim=True) if dots.shape[1] else torch.zeros(n, 1, dtype=torch.float64)
            d = 2.0**-24 * (worst * (hd + 4) + 8 + 2 * v.shape[0])
            tol[first : first + n, h] = size * (u + 2 * d) + u * o.abs()
            if batch.dtype == torch.float16 and v.shape[0]:
                finite = torch.where(v.isfinite(), v.abs(), 0.0)
                tol[first : first + n, h] += v.shape[0] * 2.0**-25 * finite.amax() / torch.where(some, total.clamp(min=1e-30), 1.0).clamp(min=1.0) + 2.0**-24
    return out.flatten(1), tol.flatten(1)


def compare(what, got, want, tol):
    got = got.double().cpu()
    odd = ~want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN elsewhere"
    assert torch.equal(got[odd & ~want.isnan()], want[odd & ~want.isnan()]), f"{what}: infinities"
    err = torch.where(odd, 0.0, (got - want).abs())
    ratio = (err / tol.where(~odd, torch.tensor(1.0, dtype=torch.float64)).clamp(min=1e-30)).max().item() if err.numel() else 0.0
    print(f"{what}: largest error {err.max().item() if err.numel() else 0.0:.3e}, of its tolerance {ratio:.3f}", flush=True)
    assert ratio <= 1.0
