"""The KV cache in pages on the GPU: append, attention, drafted trees and keep against their formulas in 64
bits (tests/paged_reference.py), over pools whose unused places hold NaN."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from linnet_amd import LinnetError
from linnet_amd.torch import paged
from tests.paged_reference import DEV, Batch, attention, compare, entry_of

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


# ------------------------------------------------------------------ append


def _turned(x, norm, eps, cos, sin):
    """One token's heads [heads, head_dim] in 64 bits, and the size of what its sums add."""
    x = x.double()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double().cpu()
    size = x.abs()
    if cos is None:
        return x, size
    r = cos.shape[-1]
    a, b, c, s = x[:, :r], x[:, r : 2 * r], cos.double(), sin.double()
    turned = torch.cat([a * c - b * s, b * c + a * s, x[:, 2 * r :]], dim=-1)
    both = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), x[:, 2 * r :].abs()], dim=-1)
    return turned, both


def _append(batch, heads, half, norm, positions=None, table=None, strided=True, seed=0, extra=0, out=None):
    hd, kvh, tokens = batch.head_dim, batch.kv_heads, batch.tokens + extra
    x = batch.random(tokens, (heads + 2 * kvh) * hd + (8 if strided else 0)).to(DEV)
    q, k, v = x[:, : heads * hd], x[:, heads * hd : (heads + kvh) * hd], x[:, (heads + kvh) * hd : (heads + 2 * kvh) * hd]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cos = sin = None
    if half:
        rows = max([1, *batch.lengths_list]) if table is None else table
        angle = torch.rand(rows, half, generator=batch.g, dtype=torch.float64) * 6.28
        cos, sin = angle.cos().float().to(DEV), angle.sin().float().to(DEV)
    norms = [(1 + 0.2 * torch.randn(hd, generator=batch.g)).to(DEV) if norm else None for _ in range(2)]
    given = None if positions is None else torch.tensor(positions, dtype=torch.int32, device=DEV)
    before = batch.cache.k.cpu(), batch.cache.v.cpu()
    got = paged.paged_append(q, k, v, cos, sin, batch.cache, batch.tables, batch.lengths, batch.starts, positions=given,
                             q_norm=norms[0], k_norm=norms[1], eps=1e-5, out=out)
    torch.cuda.synchronize()
    u, f32 = torch.finfo(batch.dtype).eps / 2, 2.0**-24
    want = torch.zeros(tokens, heads * hd, dtype=torch.float64)
    tol = torch.zeros_like(want)
    k_want, v_want = (t.clone() for t in before)
    k_tol = torch.zeros(k_want.shape, dtype=torch.float64)
    k_exact = k_want.double()
    for s, n in enumerate(batch.counts):
        for i in range(n):
            t, e = batch.starts_list[s] + i, batch.lengths_list[s] - n + i
            p = e if positions is None else positions[t]
            if half and not 0 <= p < cos.shape[0]:
                continue
            # A head's sum of squares, root, three products and a sum: under (head_dim + 16) roundings of f32.
            args = (cos[p].cpu(), sin[p].cpu()) if half else (None, None)
            y, size = _turned(q[t].cpu().view(heads, hd), norms[0], 1e-5, *args)
            want[t], tol[t] = y.flatten(), (u * y.abs() + size * f32 * (hd + 16)).flatten() + 2.0**-25
            if batch.there(s, e):
                page, place = batch.rows[s][e // batch.page], e % batch.page
                y, size = _turned(k[t].cpu().view(kvh, hd), norms[1], 1e-5, *args)
                k_exact[page, :, :, place] = y.view(kvh, -1, 8)
                k_tol[page, :, :, place] = (u * y.abs() + size * f32 * (hd + 16)).view(kvh, -1, 8) + 2.0**-25
                v_want[page, :, place // 8, :, place % 8] = v[t].cpu().view(kvh, hd)
    compare("q", got[: batch.tokens], want[: batch.tokens], tol[: batch.tokens])
    compare("k", batch.cache.k, k_exact, k_tol)
    assert torch.equal(batch.cache.v.cpu().view(torch.int16), v_want.view(torch.int16))
    return got


APPENDS = [
    # counts, lengths, heads, kv_heads, head_dim, page, dtype, half, norm
    ([1], [1], 4, 1, 128, 64, BF16, 64, False),
    ([1], [700], 32, 8, 128, 64, BF16, 64, True),
    ([1] * 5, [1, 16, 17, 33, 64], 8, 2, 64, 16, F16, 32, True),
    ([7, 8, 9, 0, 1], [7, 16, 25, 5, 1], 6, 2, 128, 16, BF16, 32, True),
    ([130, 3], [130, 131], 5, 5, 64, 32, F16, 16, False),
    ([33, 64], [200, 64], 3, 1, 128, 128, F16, 0, True),
    ([20, 20], [33, 41], 1, 1, 64, 16, BF16, 8, False),
    ([900, 1, 61], [905, 30, 61], 11, 4, 128, 64, BF16, 64, True),
    ([700, 400], [700, 400], 13, 4, 64, 16, F16, 16, False),
    ([1] * 70 + [9] + [0] * 3 + [2] * 70, [5] * 70 + [60] + [0] * 3 + [2] * 70, 2, 1, 64, 16, BF16, 32, False),
]


@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_append(case) -> None:
    counts, lengths, heads, kvh, hd, page, dtype, half, norm = case
    print(case, flush=True)
    for strided in (True, False):
        _append(Batch(counts, lengths, kvh, hd, page, dtype, seed=1), heads, half, norm, strided=strided)


def test_append_positions_of_a_tree_and_past_the_tables() -> None:
    batch = Batch([6, 2], [20, 9], 2, 64, 16, BF16, seed=2)
    _append(batch, 4, 32, True, positions=[14, 15, 15, 16, -1, 17, 40, 39], table=40)


def test_append_entries_without_a_page_and_before_the_first() -> None:
    batch = Batch([40, 5, 3], [60, 2, 30], 2, 64, 16, BF16, seed=3)
    batch.rows[0][2], batch.rows[2][1] = -1, 10**6
    batch.tables = torch.tensor(batch.rows, dtype=torch.int32, device=DEV)
    _append(batch, 4, 32, False)
    # No table reaches the new entries; and a pool of no pages.
    batch = Batch([3, 4], [64, 20], 2, 64, 16, BF16, seed=4, width=1)
    _append(batch, 4, 32, False)
    empty = paged.PagedCache.empty(0, 2, 64, 16)
    x = torch.randn(1, 128, device=DEV).to(BF16)
    got = paged.paged_append(x, x, x, None, None, empty, torch.zeros(1, 0, dtype=torch.int32, device=DEV),
                             torch.ones(1, dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV))
    assert torch.equal(got, x)


def test_append_leaves_rows_of_no_sequence() -> None:
    batch = Batch([2, 1], [9, 17], 2, 64, 16, BF16, seed=5)
    got = _append(batch, 4, 32, False, extra=13)
    assert torch.equal(got[3:], torch.zeros_like(got[3:]))
    out = torch.full((16, 256), 7.0, dtype=BF16, device=DEV)
    got = _append(batch, 4, 32, False, extra=13, out=out)
    assert got is out and torch.equal(got[3:], torch.full_like(got[3:], 7.0))


def test_append_in_place_and_without_rotation() -> None:
    batch = Batch([20], [20], 2, 128, 32, F16, seed=6)
    q, k, v = batch.random(20, 512).to(DEV), batch.random(20, 256).to(DEV), batch.random(20, 256).to(DEV)
    cos, sin = torch.rand(20, 64, device=DEV), torch.rand(20, 64, device=DEV)
    want = paged.paged_append(q, k, v, cos, sin, batch.cache, batch.tables, batch.lengths, batch.starts)
    got = paged.paged_append(q, k, v, cos, sin, batch.cache, batch.tables, batch.lengths, batch.starts, out=q)
    assert got is q and torch.equal(got, want)
    plain = paged.paged_append(q, k, v, None, None, batch.cache, batch.tables, batch.lengths, batch.starts)
    assert torch.equal(plain, q)
    for e in (0, 7, 8, 19):
        key, value = entry_of(batch.cache.k, batch.cache.v, batch.rows[0][0], e)
        assert torch.equal(key.flatten(), k[e]) and torch.equal(value.flatten(), v[e])


# ------------------------------------------------------------------ attention


ATTENDS = [
    # counts, lengths, heads, kv_heads, head_dim, page, dtype, window, sinks
    ([1], [1], 4, 1, 128, 64, BF16, 0, False),
    ([1], [1], 1, 1, 64, 16, F16, 0, True),
    ([1], [31], 8, 2, 128, 16, BF16, 0, False),
    ([1], [129], 32, 8, 128, 64, BF16, 0, True),
    ([1], [1500], 8, 2, 64, 128, F16, 0, False),
    ([1] * 6, [1, 2, 100, 256, 257, 900], 16, 2, 128, 16, BF16, 0, False),
    ([1] * 3, [500, 70, 1], 10, 2, 64, 32, BF16, 64, True),
    ([1, 1], [300, 40], 40, 1, 128, 32, F16, 0, False),
    ([1, 1], [300, 40], 17, 1, 64, 16, F16, 33, False),
    ([3, 8, 1], [3, 200, 77], 8, 2, 128, 64, F16, 0, True),
    ([5, 6], [5, 400], 6, 3, 64, 16, BF16, 5, False),
    ([40], [40], 4, 1, 128, 64, BF16, 0, False),
    ([200], [200], 8, 2, 64, 16, F16, 0, True),
    ([130], [390], 6, 2, 128, 32, BF16, 0, False),
    ([65, 1, 0, 33, 2], [65, 300, 12, 90, 2], 8, 2, 128, 16, BF16, 0, False),
    ([65, 1, 0, 33, 2], [100, 300, 12, 90, 2], 5, 5, 64, 64, F16, 40, True),
    ([300], [300], 3, 1, 128, 128, BF16, 70, False),
    ([257, 1], [700, 1], 40, 1, 64, 32, BF16, 0, False),
    ([100], [100], 28, 4, 128, 16, F16, 1, False),
    ([300], [420], 7, 7, 64, 16, BF16, 0, True),
    ([300, 20], [420, 900], 10, 1, 128, 64, F16, 0, False),
]


def _attend(batch, heads, window=0, sinks=False, max_queries=None, scale=None, parents=None, extra=0, sharp=2.0):
    q = (sharp * torch.randn(batch.tokens + extra, heads * batch.head_dim, generator=batch.g)).to(batch.dtype).to(DEV)
    sink = torch.randn(heads, generator=batch.g).to(DEV) if sinks else None
    kinds = dict(max_queries=max_queries, scale=scale, window=window, sinks=sink)
    if parents is None:
        got = paged.paged_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts, **kinds)
    else:
        flat = torch.tensor(parents + [0] * extra, dtype=torch.int32, device=DEV)
        got = paged.paged_tree_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts, flat, **kinds)
    torch.cuda.synchronize()
    want, tol = attention(batch, q, scale, window, sink, parents)
    compare(f"attention max_queries={max_queries}", got, want, tol)
    return got


@pytest.mark.parametrize("case", ATTENDS, ids=str)
def test_attention(case) -> None:
    counts, lengths, heads, kvh, hd, page, dtype, window, sinks = case
    print(case, flush=True)
    batch = Batch(counts, lengths, kvh, hd, page, dtype, seed=11).fill()
    # What the caller says of the batch decides the kernels: each gives the same within its rounding.
    for most in (None, max(counts), 1):
        _attend(batch, heads, window, sinks, max_queries=most)


def test_attention_of_rows_that_see_nothing() -> None:
    """Fewer entries than new tokens, none at all, sequences without new tokens, entries without a page, rows of no
    sequence: zeros, and what is there counts."""
    for sinks in (False, True):
        batch = Batch([3, 2, 0, 40, 1], [2, 0, 50, 35, 20], 2, 64, 16, BF16, seed=21)
        batch.rows[3][1], batch.rows[4] = -1, [10**9, -5, -(2**31)]
        batch.tables = torch.tensor([(row + [-1] * 4)[:4] for row in batch.rows], dtype=torch.int32, device=DEV)
        batch.rows = batch.tables.tolist()
        batch.fill()
        got = _attend(batch, 8, sinks=sinks, extra=70)
        assert not got[:1].any() and not got[3:5].any() and not got[45:].any() and got[5:45].any()
        out = torch.full_like(got, 5.0)
        q = torch.randn(got.shape, device=DEV).to(BF16)
        paged.paged_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts, out=out)
        assert torch.equal(out[46:], torch.full_like(out[46:], 5.0)) and not (out[:46] == 5.0).all(-1).any()


@pytest.mark.parametrize("most", [None, 1])
def test_attention_of_a_pool_or_tables_of_nothing(most) -> None:
    """No pages, tables of no width, no sequences, lengths past the tables."""
    q = torch.randn(50, 256, device=DEV).to(BF16)
    i32 = dict(dtype=torch.int32, device=DEV)
    for pages, width, sequences in ((0, 3, 2), (4, 0, 2), (4, 3, 0)):
        cache = paged.PagedCache.empty(pages, 2, 64, 16)
        tables, lengths = torch.zeros(sequences, width, **i32), torch.full((sequences,), 30, **i32)
        starts = torch.tensor([0, 30, 50][: sequences + 1], **i32)
        got = paged.paged_attention(q, cache, tables, lengths, starts, max_queries=most)
        assert got.shape == q.shape and not got.any()
    batch = Batch([2, 30], [40, 64], 2, 64, 16, BF16, seed=22, width=2).fill()
    _attend(batch, 4, max_queries=most)


def test_attention_scales_and_far_scores() -> None:
    """Scores whose exponentials lie far apart, and a scale of the caller's."""
    for hd, most in ((64, None), (128, None), (128, 1)):
        batch = Batch([50, 1], [130, 500], 2, hd, 16, BF16, seed=23).fill()
        _attend(batch, 8, max_queries=most, sharp=30.0)
        _attend(batch, 8, max_queries=most, scale=0.7)
        _attend(batch, 8, max_queries=most, scale=1e-6)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("most", [None, 1])
def test_attention_keeps_infinities_and_nan_to_the_rows_that_see_them(dtype, most) -> None:
    for counts, lengths, heads, kvh, hd, window in (([70, 3], [150, 40], 4, 2, 128, 0), ([70, 3], [150, 40], 3, 1, 64, 20),
                                                    ([2, 1], [300, 33], 8, 1, 64, 0)):
        batch = Batch(counts, lengths, kvh, hd, 16, dtype, seed=24)
        inf, nan = float("inf"), float("nan")
        for e, d, what in ((-1, 5, nan), (-2, 9, inf), (-2, 40, -inf), (-1, 9, -inf), (-1, 63, inf)):
            batch.values[0][e, 0, d] = what
        batch.values[1][20, :, 7] = inf
        if counts[0] == 70:
            batch.values[0][-40, 0, 3], batch.values[0][-36, 0, 3] = inf, -inf
            batch.values[0][-50, kvh - 1, 30] = nan
            batch.keys[0][-3, 0, 0] = nan  # all rows that see it
        batch.fill()
        q = (2 * torch.randn(batch.tokens, heads * hd, generator=batch.g)).to(dtype).to(DEV)
        got = paged.paged_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts, max_queries=most, window=window)
        keys = batch.keys[0].clone()
        batch.keys[0] = torch.where(keys.isnan(), torch.zeros_like(keys), keys)
        want, tol = attention(batch, q, window=window)
        group = heads // kvh
        if counts[0] == 70:
            for i in (67, 68, 69):
                want[i, : group * hd], tol[i, : group * hd] = nan, nan
        for i in range(batch.tokens):  # a tolerance that an infinity is part of: the values there are compared as they are
            tol[i] = torch.where(tol[i].isfinite(), tol[i], 0.0)
        compare(f"{dtype} {counts} most={most}", got, want, tol)


# ------------------------------------------------------------------ drafted trees


def _random_parents(counts, g, chain=False):
    parents = []
    for n in counts:
        for i in range(n):
            r = torch.randint(0, 100, (1,), generator=g).item()
            parents.append(-1 if i == 0 or r < 10 else i - 1 if chain else torch.randint(max(0, i - 6), i, (1,), generator=g).item())
    return parents


TREES = [
    # counts, lengths, heads, kv_heads, head_dim, page, dtype, window, sinks
    ([1], [1], 4, 1, 128, 64, BF16, 0, False),
    ([5], [5], 4, 1, 64, 16, F16, 0, True),
    ([7, 2], [30, 200], 4, 2, 128, 16, BF16, 0, False),
    ([24], [500], 8, 2, 128, 64, BF16, 0, False),
    ([60, 33, 1, 0, 17], [60, 100, 40, 8, 300], 8, 2, 64, 16, F16, 0, True),
    ([256], [300], 2, 1, 128, 32, BF16, 0, False),
    ([130, 64], [140, 333], 6, 2, 64, 128, BF16, 0, False),
    ([40, 9], [90, 9], 4, 1, 64, 16, F16, 3, True),
    ([6, 40], [300, 41], 4, 2, 128, 16, BF16, 30, False),
]


@pytest.mark.parametrize("case", TREES, ids=str)
def test_tree_attention(case) -> None:
    counts, lengths, heads, kvh, hd, page, dtype, window, sinks = case
    print(case, flush=True)
    batch = Batch(counts, lengths, kvh, hd, page, dtype, seed=31).fill()
    for most in (None, max(counts), 1):
        for chain in (False, True):
            _attend(batch, heads, window, sinks, max_queries=most, parents=_random_parents(counts, batch.g, chain))


def test_tree_attention_of_any_parents() -> None:
    """Parents that are no earlier node follow the context, nodes past the 256th give zeros, fewer entries than nodes."""
    batch = Batch([12, 300], [20, 290], 2, 64, 16, BF16, seed=32).fill()
    parents = [-1, 1, 5, 2**31 - 1, -(2**31), 3, 5, 6, 7, 200, 9, 10] + [i - 1 for i in range(300)]
    for most in (None, 1):
        got = _attend(batch, 4, parents=parents, max_queries=most, extra=5)
        assert not got[12 + 256 :].any() and not got[12:22].any() and got[22:268].any(-1).all()


def test_tree_attention_keeps_odd_values_to_the_rows_that_see_them() -> None:
    for most in (None, 1):
        batch = Batch([9, 70], [100, 90], 2, 64, 16, F16, seed=33)
        parents = [-1, 0, 0, 1, 2, 2, 3, -1, 7] + [-1] + [i // 2 for i in range(69)]
        batch.values[0][91 + 2, 0, 5] = float("inf")
        batch.values[1][20 + 3, 1, 9] = float("nan")
        batch.fill()
        q = torch.randn(79, 256, generator=batch.g).to(F16).to(DEV)
        flat = torch.tensor(parents, dtype=torch.int32, device=DEV)
        got = paged.paged_tree_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts, flat, max_queries=most)
        want, tol = attention(batch, q, parents=parents)
        compare("tree", got, want, torch.where(tol.isfinite(), tol, 0.0))
        assert got[[2, 4, 5], 5].isinf().all() and got[[0, 1, 3, 6, 7, 8], 5].isfinite().all()


# ------------------------------------------------------------------ keep


def _kept(batch, kept):
    """The pool and the lengths that follow, entry by entry."""
    k, v = batch.cache.k.cpu().clone(), batch.cache.v.cpu().clone()
    k0, v0 = k.clone(), v.clone()
    lengths = []
    for s, n in enumerate(batch.counts):
        base, last, number = batch.lengths_list[s] - n, -1, 0
        for j, node in enumerate(kept[s]):
            if not last < node < n or node < 0:
                break
            last, number = node, j + 1
            a, b = base + node, base + j
            if batch.there(s, a) and batch.there(s, b):
                pa, ia, pb, ib = batch.rows[s][a // batch.page], a % batch.page, batch.rows[s][b // batch.page], b % batch.page
                k[..., pb, :, :, ib, :] = k0[..., pa, :, :, ia, :]
                v[..., pb, :, ib // 8, :, ib % 8] = v0[..., pa, :, ia // 8, :, ia % 8]
        lengths.append(max(base + number, 0))
    return k, v, lengths


@pytest.mark.parametrize(("hd", "page", "dtype", "layers"), [(64, 16, BF16, None), (128, 32, F16, 3), (64, 128, F16, 2), (128, 64, BF16, None)],
                         ids=str)
def test_keep(hd, page, dtype, layers) -> None:
    counts, lengths = [24, 9, 0, 1, 200, 5, 12], [40, 9, 30, 17, 333, 64, 40]
    batch = Batch(counts, lengths, 3, hd, page, dtype, seed=41, layers=layers)
    batch.rows[5][0] = batch.rows[6][-1] = -1
    batch.tables = torch.tensor(batch.rows, dtype=torch.int32, device=DEV)
    batch.cache.k.copy_(torch.randn(batch.cache.k.shape, generator=batch.g))
    batch.cache.v.copy_(torch.randn(batch.cache.v.shape, generator=batch.g))
    paths = [[0, 2, 3, 7, 11, 23], [1, 3, 3, 4], [0], [0], list(range(1, 200, 2)), [4], [5, 2, 9]]
    for width in (100, 3, 0):
        kept = [(p + [-1] * width)[:width] for p in paths]
        k, v, want = _kept(batch, kept)
        given = torch.tensor(kept, dtype=torch.int32, device=DEV).reshape(len(counts), width)
        got = paged.paged_keep(batch.cache, batch.tables, batch.lengths, batch.starts, given)
        assert got.tolist() == want and batch.lengths.tolist() == lengths
        assert torch.equal(batch.cache.k.cpu(), k) and torch.equal(batch.cache.v.cpu(), v)


# ------------------------------------------------------------------ together


def _cause(q, keys, values):
    """The last row's causal attention over dense keys and values [entries, kv_heads, head_dim] in 64 bits."""
    group = q.shape[0] // keys.shape[1]
    k, v = keys.double().repeat_interleave(group, 1), values.double().repeat_interleave(group, 1)
    w = torch.softmax(torch.einsum("hd,ehd->he", q.double().contiguous(), k.contiguous()) * q.shape[1] ** -0.5, -1)
    return torch.einsum("he,ehd->hd", w, v)


def test_a_run_of_prompt_draft_keep_and_step() -> None:
    """A prompt of two sequences, a drafted tree over it, its accepted path kept, the next token: after each,
    the same as attention over the dense history."""
    g = torch.Generator().manual_seed(51)
    heads, kvh, hd, page = 8, 2, 64, 16
    cache = paged.PagedCache.empty(24, kvh, hd, page)
    cache.k.fill_(float("nan")), cache.v.fill_(float("nan"))
    tables = torch.randperm(24, generator=g).int().view(2, 12).to(DEV)
    cos, sin = torch.rand(200, 32, generator=g).to(DEV), torch.rand(200, 32, generator=g).to(DEV)
    history = [([], []), ([], [])]  # rotated keys, values of each sequence
    lengths = [0, 0]

    def rotate(x, p):
        a, b = x[..., :32].float(), x[..., 32:].float()
        return torch.cat([a * cos[p].cpu() - b * sin[p].cpu(), b * cos[p].cpu() + a * sin[p].cpu()], -1).to(BF16)

    def add(counts, parents=None):
        """One call's new tokens: appended, attended; returns per token (queries, keys, values, output)."""
        starts = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device=DEV)
        x = torch.randn(sum(counts), (heads + 2 * kvh) * hd, generator=g).to(BF16)
        q, k, v = x.to(DEV).split([heads * hd, kvh * hd, kvh * hd], 1)
        now = torch.tensor([lengths[s] + counts[s] for s in range(2)], dtype=torch.int32, device=DEV)
        places, positions = [], []
        for s in range(2):
            for i in range(counts[s]):
                depth = i
                if parents is not None:
                    depth, j = 0, parents[s][i]
                    while j >= 0:
                        depth, j = depth + 1, parents[s][j]
                places.append((s, i))
                positions.append(lengths[s] + depth)
        pos = torch.tensor(positions, dtype=torch.int32, device=DEV) if parents is not None else None
        qr = paged.paged_append(q, k, v, cos, sin, cache, tables, now, starts, positions=pos)
        if parents is None:
            out = paged.paged_attention(qr, cache, tables, now, starts, max_queries=max(counts))
        else:
            flat = torch.tensor(parents[0] + parents[1], dtype=torch.int32, device=DEV)
            out = paged.paged_tree_attention(qr, cache, tables, now, starts, flat, max_queries=max(counts))
        rows = []
        for t, (s, i) in enumerate(places):
            rows.append((rotate(x[t, : heads * hd].view(heads, hd), positions[t]),
                         rotate(x[t, heads * hd : (heads + kvh) * hd].view(kvh, hd), positions[t]), x[t, (heads + kvh) * hd :].view(kvh, hd),
                         out[t].cpu().view(heads, hd)))
        return places, rows, now, starts

    def check(got, q, keys, values):
        want = _cause(q, torch.stack(keys), torch.stack(values))
        # Queries and keys may part by a rounding from those of this test's rotation, which shifts scores by 2^-7 or so.
        assert (got.double() - want).abs().max() <= 0.05, (got.double() - want).abs().max()

    for counts in ([37, 50], [1, 1]):
        places, rows, now, _ = add(counts)
        for (s, i), (q, k, v, got) in zip(places, rows):
            history[s][0].append(k), history[s][1].append(v)
            check(got, q, *history[s])
        lengths = now.tolist()
    parents = [[-1, 0, 0, 1, 2, 4, 5], [-1, -1, 1, 2, 0]]
    kept = [[0, 2, 4, 5], [1, 2]]
    places, rows, now, starts = add([7, 5], parents)
    for (s, i), (q, k, v, got) in zip(places, rows):
        path, j = [], i
        while j >= 0:
            path.append(j)
            j = parents[s][j]
        nodes = [places.index((s, p)) for p in path[::-1]]
        check(got, q, history[s][0] + [rows[t][1] for t in nodes], history[s][1] + [rows[t][2] for t in nodes])
    new = paged.paged_keep(cache, tables, now, starts, torch.tensor([kept[0], kept[1] + [-1, -1]], dtype=torch.int32, device=DEV))
    for s in range(2):
        for node in kept[s]:
            t = places.index((s, node))
            history[s][0].append(rows[t][1]), history[s][1].append(rows[t][2])
    lengths = new.tolist()
    assert lengths == [len(history[0][0]), len(history[1][0])]
    places, rows, now, _ = add([1, 3])
    for (s, i), (q, k, v, got) in zip(places, rows):
        history[s][0].append(k), history[s][1].append(v)
        check(got, q, *history[s])


def test_captured_calls_follow_the_batch_on_the_device() -> None:
    """A captured append and attention replayed as the lengths grow, beside another graph of the same kind and eager
    calls: every replay gives the eager call's bits."""
    batch = Batch([1, 1, 0], [100, 41, 7], 2, 128, 16, BF16, seed=61, spare=8)
    batch.fill()
    tables = torch.cat([batch.tables, torch.full((3, 4), -1, dtype=torch.int32, device=DEV)], 1)
    g = batch.g
    cos, sin = torch.rand(200, 64, generator=g).to(DEV), torch.rand(200, 64, generator=g).to(DEV)
    x = torch.randn(3, 12 * 128, generator=g).to(BF16).to(DEV)
    lengths, starts = batch.lengths.clone(), torch.tensor([0, 1, 2, 2], dtype=torch.int32, device=DEV)

    def step(cache):
        q, k, v = x.split([8 * 128, 2 * 128, 2 * 128], 1)
        q = paged.paged_append(q, k, v, cos, sin, cache, tables, lengths, starts)
        return paged.paged_attention(q, cache, tables, lengths, starts, max_queries=1), paged.paged_attention(q, cache, tables, lengths, starts)

    other = paged.PagedCache(batch.cache.k.clone(), batch.cache.v.clone())
    step(batch.cache), step(other)
    torch.cuda.synchronize()
    graphs = []
    for cache in (batch.cache, other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(cache)
        graphs.append((graph, outs))
    for turn in range(4):
        x.copy_(torch.randn(x.shape, generator=g))
        spare = paged.PagedCache(batch.cache.k.clone(), batch.cache.v.clone())
        want = step(spare)
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(batch.cache.k.nan_to_num(), spare.k.nan_to_num())
        lengths[:2] += 1


def test_calls_on_another_stream_and_of_strided_operands() -> None:
    batch = Batch([20, 1], [50, 300], 2, 64, 16, BF16, seed=62).fill()
    q = torch.randn(21, 512, generator=batch.g).to(BF16).to(DEV)
    want = paged.paged_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = paged.paged_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts)
    stream.synchronize()
    assert torch.equal(got, want)
    wide = torch.zeros(21, 1000, dtype=BF16, device=DEV)
    wide[:, 3:515] = q
    strided_tables = torch.stack([batch.tables, batch.tables], 2)[:, :, 0]
    for x in (wide[:, 3:515], q.t().contiguous().t(), torch.cat([q, q], 1)[:, 512:]):
        assert torch.equal(paged.paged_attention(x, batch.cache, strided_tables, batch.lengths, batch.starts), want)
    one = paged.paged_attention(q[:1].expand(21, 512), batch.cache, batch.tables, batch.lengths, batch.starts)
    assert torch.equal(one, paged.paged_attention(q[:1].repeat(21, 1), batch.cache, batch.tables, batch.lengths, batch.starts))


def test_offsets_past_32_bits() -> None:
    """A pool of over 4 GiB of keys, a sequence's pages at its end."""
    kvh, hd, page = 8, 128, 64
    pages = (9 << 29) // (kvh * hd * page * 2)
    cache = paged.PagedCache.empty(pages, kvh, hd, page)
    small = Batch([40, 1], [150, 70], kvh, hd, page, BF16, seed=63).fill()
    n = small.cache.k.shape[0]
    cache.k[pages - n :] = small.cache.k
    cache.v[pages - n :] = small.cache.v
    tables = torch.where(small.tables >= 0, small.tables + (pages - n), -1).int()
    q = torch.randn(41, 2 * kvh * hd, generator=small.g).to(BF16).to(DEV)
    x = torch.randn(41, 2 * kvh * hd, generator=small.g).to(BF16).to(DEV)
    for most in (None, 1):
        want = paged.paged_attention(q, small.cache, small.tables, small.lengths, small.starts, max_queries=most)
        assert torch.equal(paged.paged_attention(q, cache, tables, small.lengths, small.starts, max_queries=most), want)
    k, v = x.split([kvh * hd, kvh * hd], 1)
    kept = torch.tensor([[3, 9, 30], [0, -1, -1]], dtype=torch.int32, device=DEV)
    for pool, at in ((cache, tables), (small.cache, small.tables)):
        paged.paged_append(q, k, v, None, None, pool, at, small.lengths, small.starts)
        paged.paged_keep(pool, at, small.lengths, small.starts, kept)
    assert torch.equal(cache.k[pages - n :].nan_to_num(), small.cache.k.nan_to_num())
    assert torch.equal(cache.v[pages - n :].nan_to_num(), small.cache.v.nan_to_num())


def test_long_context_in_many_parts() -> None:
    """One token over a context that is split many ways, against 64 bits."""
    for heads, kvh, hd, n, dtype in ((4, 1, 128, 40000, BF16), (8, 1, 64, 70001, F16)):
        batch = Batch([1], [1], kvh, hd, 128, dtype, seed=64)
        pages = -(-n // 128)
        k, v = torch.randn(pages, kvh, hd // 8, 128, 8, device=DEV).to(dtype), torch.randn(pages, kvh, 16, hd, 8, device=DEV).to(dtype)
        tables = torch.randperm(pages, device=DEV).int()[None]
        cache = paged.PagedCache(k, v)
        q = (2 * torch.randn(1, heads * hd, generator=batch.g)).to(dtype).to(DEV)
        got = paged.paged_attention(q, cache, tables, torch.tensor([n], dtype=torch.int32, device=DEV),
                                    torch.tensor([0, 1], dtype=torch.int32, device=DEV))
        t = tables[0].long()
        kd = k[t][:, 0].permute(0, 2, 1, 3).reshape(-1, hd)[:n].double()
        vd = v[t][:, 0].permute(0, 1, 3, 2).reshape(-1, hd)[:n].double()
        x = q.view(heads, hd).double()
        w = torch.softmax(x @ kd.t().contiguous() * hd**-0.5, -1)
        want, size = w @ vd, w @ vd.abs()
        u = torch.finfo(dtype).eps / 2
        # As in the reference's tolerance; a wave's sums here are of at most n entries.
        worst = (x.abs() @ kd.abs().t().contiguous() * hd**-0.5).max().item()
        tol = size * (u + 2.0**-23 * (worst * (hd + 4) + 8 + 2 * n / 64)) + u * want.abs() + 2.0**-24
        compare(f"{n} entries", got.view(heads, hd), want.cpu(), tol.cpu())


def test_refusals() -> None:
    batch = Batch([2], [5], 2, 64, 16, BF16, seed=65)
    q, kv = torch.zeros(2, 256, dtype=BF16, device=DEV), torch.zeros(2, 128, dtype=BF16, device=DEV)
    cache, tables, lengths, starts = batch.cache, batch.tables, batch.lengths, batch.starts
    cos = torch.zeros(9, 32, device=DEV)
    append = [q, kv, kv, cos, cos, cache, tables, lengths, starts]

    def refused(call, *args, match, **kinds):
        with pytest.raises(LinnetError, match=match):
            call(*args, **kinds)

    def but(args, at, value):
        return args[:at] + [value] + args[at + 1 :]

    refused(paged.paged_append, *but(append, 0, q.half()), match="as the cache is")
    refused(paged.paged_append, *but(append, 0, q[:, :250]), match="heads")
    refused(paged.paged_append, *but(append, 1, kv[:1]), match="k and v")
    refused(paged.paged_append, *but(append, 3, None), match="come together")
    refused(paged.paged_append, *but(append, 3, cos[:, :16]), match="float32")
    refused(paged.paged_append, *but(but(append, 3, cos[:, :4]), 4, cos[:, :4]), match="angles")
    refused(paged.paged_append, *but(append, 7, lengths.long()), match="lengths")
    refused(paged.paged_append, *but(append, 8, lengths), match="starts")
    refused(paged.paged_append, *but(append, 6, tables.long()), match="tables")
    refused(paged.paged_append, *append, positions=lengths, match="positions")
    refused(paged.paged_append, *append, q_norm=torch.ones(64, device=DEV, dtype=BF16), match="q_norm")
    refused(paged.paged_append, *append, out=q[:1], match="out")
    refused(paged.paged_append, *but(append, 0, q.cpu()), match="GPU tensors")
    refused(paged.paged_append, *but(append, 5, paged.PagedCache.empty(2, 2, 64, 16, layers=2)), match="one layer")
    attend = [q, cache, tables, lengths, starts]
    refused(paged.paged_attention, *but(attend, 0, q[:, :192]), match="multiple of 2")
    refused(paged.paged_attention, *attend, max_queries=0, match="max_queries")
    refused(paged.paged_attention, *attend, window=-1, match="window")
    refused(paged.paged_attention, *attend, scale=0.0, match="scale")
    refused(paged.paged_attention, *attend, sinks=torch.zeros(3, device=DEV), match="sinks")
    refused(paged.paged_attention, *attend, out=q.t().contiguous().t(), match="out")
    refused(paged.paged_attention, *but(attend, 0, q.float().requires_grad_().to(BF16)), match="gradient")
    refused(paged.paged_tree_attention, *attend, lengths, match="parents")
    refused(paged.paged_keep, cache, tables, lengths, starts, lengths, match="kept")
    with torch.no_grad():
        paged.paged_attention(q.float().requires_grad_().to(BF16), *attend[1:])
    empty = paged.paged_attention(q[:0], *attend[1:])
    assert empty.shape == (0, 256)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("sink", [False, True])
def test_attention_f16_keeps_a_long_tail_of_small_weights(new, sink) -> None:
    print("tail", new, sink, flush=True)
    entries, hd, page = 1 << 17, 64, 64
    pages = entries // page
    k = torch.zeros(pages, 1, hd // 8, page, 8, dtype=F16, device=DEV)
    v = torch.ones(pages, 1, page // 8, hd, 8, dtype=F16, device=DEV)
    k[0, 0, 0, 0, 0] = 1  # entry 0: score 17.75 of value 0; the others 0 of value 1, weights of 2^-25.6 each
    v[0, 0, 0, :, 0] = 0
    q = torch.zeros(new, hd, dtype=F16, device=DEV)
    q[:, 0] = 17.75
    ints = lambda *n: torch.tensor(n, dtype=torch.int32, device=DEV)  # noqa: E731
    sinks = torch.tensor([17.75], device=DEV) if sink else None
    got = paged.paged_attention(q, paged.PagedCache(k, v), torch.arange(pages, dtype=torch.int32, device=DEV)[None], ints(entries),
                                ints(0, new), scale=1.0, sinks=sinks).double().cpu()
    seen = torch.arange(entries - new, entries, dtype=torch.float64)  # entries but the first that a row sees
    tail = seen * torch.tensor(-17.75, dtype=torch.float64).exp()
    want = (tail / (tail + (2 if sink else 1)))[:, None].expand(-1, hd)
    # A weight below f16's normal numbers is off by half of 2^-24 / 2^7 of the largest, each one the same; the output
    # by half a step; sums and exponents in f32 by under 2^-16 of it.
    tol = entries * 2.0**-32 + want * (2.0**-11 + 2.0**-16)
    err = (got - want).abs()
    print(f"largest error {err.max().item():.2e} of {tol.max().item():.2e}", flush=True)
    assert (err <= tol).all()


PARTS = [case for case in ATTENDS if sum(case[0]) <= 70] + [
    # joined one head of a token a wave, and four
    ([1] * 41, [40 + 9 * i for i in range(41)], 9, 3, 64, 16, BF16, 0, True),
    ([1] * 69 + [0, 1], [20 + 11 * i for i in range(69)] + [7, 3], 32, 8, 128, 32, BF16, 0, True),
    ([2] * 70, [2 + 9 * i for i in range(70)], 18, 6, 64, 16, F16, 0, False),
]


@pytest.mark.parametrize("case", PARTS, ids=lambda case: f"{len(case[0])}-{case[1][0]}-{case[2:]}")
def test_attention_in_parts(case) -> None:
    """The same over tables of 4096 entries: the entries are divided by what the tables can hold."""
    counts, lengths, heads, kvh, hd, page, dtype, window, sinks = case
    print(case, flush=True)
    batch = Batch(counts, lengths, kvh, hd, page, dtype, seed=41, width=4096 // page).fill()
    for most in (None, max(counts)):
        _attend(batch, heads, window, sinks, max_queries=most)


@pytest.mark.parametrize("case", [case for case in TREES if sum(case[0]) <= 140], ids=str)
def test_tree_attention_in_parts(case) -> None:
    counts, lengths, heads, kvh, hd, page, dtype, window, sinks = case
    print(case, flush=True)
    batch = Batch(counts, lengths, kvh, hd, page, dtype, seed=42, width=4096 // page).fill()
    for most in (None, max(counts)):
        _attend(batch, heads, window, sinks, max_queries=most, parents=_random_parents(counts, batch.g))


@pytest.mark.parametrize("most", [None, 2])
def test_attention_in_parts_keeps_infinities_and_nan_to_the_rows_that_see_them(most) -> None:
    print("odd values in parts", most, flush=True)
    inf, nan = float("inf"), float("nan")
    batch = Batch([2, 1], [300, 140], 1, 64, 16, BF16, seed=43, width=256)
    for e, d, what in ((-1, 5, nan), (-1, 9, -inf), (10, 40, inf), (200, 40, inf), (200, 50, -inf), (20, 50, inf)):
        batch.values[0][e, 0, d] = what
    batch.fill()
    q = (2 * torch.randn(3, 512, generator=batch.g)).to(BF16).to(DEV)
    got = paged.paged_attention(q, batch.cache, batch.tables, batch.lengths, batch.starts, max_queries=most)
    want, tol = attention(batch, q)
    compare(f"most={most}", got, want, torch.where(tol.isfinite(), tol, 0.0))
    rows = got.view(3, 8, 64)
    assert rows[:2, :, 40].isinf().all() and rows[:2, :, 50].isnan().all() and rows[0, :, [5, 9]].isfinite().all()


def test_of_thousands_of_sequences() -> None:
    """More than 64 times 64 sequences, many of them without new tokens: each workgroup finds its own."""
    print("4200 sequences", flush=True)
    counts = [(i * 7) % 3 if i % 50 else 0 for i in range(4200)]
    counts[4100] = 45
    lengths = [n + (i * 5) % 9 for i, n in enumerate(counts)]
    _append(Batch(counts, lengths, 1, 64, 16, BF16, seed=44), 1, 8, False)
    batch = Batch(counts, lengths, 1, 64, 16, BF16, seed=44).fill()
    for most in (None, 2):
        _attend(batch, 1, max_queries=most, extra=3)


def test_captured_trees_follow_the_batch_on_the_device() -> None:
    """Append, tree attention and keep in one graph, in two graphs whose replays take turns, against the eager calls'
    bits while parents, paths and lengths change."""
    print("captured trees", flush=True)
    batch = Batch([9, 40, 0], [50, 300, 5], 2, 64, 16, BF16, seed=45, layers=2)
    g = batch.g
    batch.cache.k.copy_(torch.randn(batch.cache.k.shape, generator=g)), batch.cache.v.copy_(torch.randn(batch.cache.v.shape, generator=g))
    cos, sin = torch.rand(400, 32, generator=g).to(DEV), torch.rand(400, 32, generator=g).to(DEV)
    x = torch.randn(52, 12 * 64, generator=g).to(BF16).to(DEV)
    positions, parents = torch.zeros(52, dtype=torch.int32, device=DEV), torch.zeros(52, dtype=torch.int32, device=DEV)
    kept = torch.zeros(3, 6, dtype=torch.int32, device=DEV)
    lengths, starts = batch.lengths.clone(), batch.starts.clone()

    def step(cache):
        q, k, v = x.split([8 * 64, 2 * 64, 2 * 64], 1)
        pool = cache.layer(1)
        q = paged.paged_append(q, k, v, cos, sin, pool, batch.tables, lengths, starts, positions=positions)
        out = paged.paged_tree_attention(q, pool, batch.tables, lengths, starts, parents, max_queries=40)
        return out, paged.paged_keep(cache, batch.tables, lengths, starts, kept)

    copies = [paged.PagedCache(batch.cache.k.clone(), batch.cache.v.clone()) for _ in range(3)]
    for cache in copies:
        step(cache)
    torch.cuda.synchronize()
    graphs = []
    for cache in copies[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(cache)
        graphs.append((graph, outs))
    for turn in range(4):
        x.copy_(torch.randn(x.shape, generator=g))
        positions.copy_(torch.randint(0, 400, (52,), generator=g))
        parents.copy_(torch.tensor(_random_parents([9, 40, 3], g)))
        kept.copy_(torch.tensor([[0, 2, 5, 8, -1, -1], [1, 2, 7 + turn, 20, 33, 39], [0, 1, 2, 3, 4, 5]]))
        want = step(copies[2])
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, outs), cache in zip(graphs, copies):
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
            assert torch.equal(cache.k, copies[2].k) and torch.equal(cache.v, copies[2].v)
        lengths.copy_(torch.tensor([50 - turn, 299 - 13 * turn, 5]))


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize(("tokens", "heads", "kvh", "hd", "page", "width"),
                         [(50, 4, 2, 64, 16, 8), (64, 4, 2, 64, 16, 0), (300, 4, 2, 128, 64, 2048), (1000, 40, 1, 64, 128, 3), (1, 1, 1, 128, 16, 5)])
def test_attention_of_no_sequences(tokens, heads, kvh, hd, page, width, tree) -> None:
    """Tokens of which none has a sequence give zeros, or with `out` leave its rows, whatever the tables could hold."""
    print("no sequences", tokens, heads, kvh, hd, page, width, tree, flush=True)
    i32 = dict(dtype=torch.int32, device=DEV)
    cache = paged.PagedCache.empty(4, kvh, hd, page)
    tables, lengths, starts = torch.zeros(0, width, **i32), torch.zeros(0, **i32), torch.zeros(1, **i32)
    parents = torch.full((tokens,), -1, **i32)
    q = torch.randn(tokens, heads * hd, device=DEV).to(BF16)
    for most in (None, 1, 33, 200):
        for window in (0, 20):
            for out in (None, torch.full_like(q, 3.0)):
                kinds = dict(max_queries=most, window=window, out=out)
                if tree:
                    got = paged.paged_tree_attention(q, cache, tables, lengths, starts, parents, **kinds)
                else:
                    got = paged.paged_attention(q, cache, tables, lengths, starts, **kinds)
                torch.cuda.synchronize()
                assert torch.equal(got, torch.zeros_like(q) if out is None else torch.full_like(q, 3.0))


@pytest.mark.parametrize("width", [None, 256])
@pytest.mark.parametrize(("counts", "lengths", "heads", "kvh", "hd", "window", "sinks"),
                         [([300], [500], 4, 2, 64, 0, False), ([290, 3, 257], [420, 40, 600], 2, 2, 128, 0, True),
                          ([300], [2000], 3, 1, 64, 1500, False), ([700, 1], [900, 300], 1, 1, 64, 0, True)])
def test_tree_nodes_past_the_256th_after_a_context(counts, lengths, heads, kvh, hd, window, sinks, width) -> None:
    """They see nothing, the entries before the draft neither; the nodes before them what they saw."""
    print("long drafts", counts, lengths, heads, kvh, hd, window, sinks, width, flush=True)
    batch = Batch(counts, lengths, kvh, hd, 16, BF16, seed=34, width=width).fill()
    parents = _random_parents(counts, batch.g)
    for most in (None, 1):
        got = _attend(batch, heads, window, sinks, max_queries=most, parents=parents)
        for first, n in zip(batch.starts_list, counts):
            assert got[first : first + min(n, 256)].any(-1).all() and not got[first + min(n, 256) : first + n].any()


@pytest.mark.parametrize(("new", "heads", "width"), [(1, 4, 256), (1, 4, 4096), (1, 300, 256), (1, 520, 2048), (1, 5000, 256), (40, 4, 256)])
def test_odd_values_of_parts_without_weight_reach_their_rows(new, heads, width) -> None:
    """Infinities and NaNs in parts whose weights are 0 beside another part's: no dimension that has one is a number
    in the rows that see them, and the others are as without them."""
    print("odd values in parts without weight", new, heads, width, flush=True)
    batch = Batch([new, 1], [4000, 1300], 1, 64, 16, BF16, seed=46, width=width)
    for s, n in ((0, new), (1, 1)):  # scores 300 of the sequence's first new entry, 0 of all before it
        batch.keys[s].zero_()
        batch.keys[s][-n, 0, 0] = 20
    inf, nan = float("inf"), float("nan")
    for e, d, what in ((10, 5, nan), (700, 6, inf), (1500, 7, -inf)):
        batch.values[0][e, 0, d] = what
    batch.fill()
    q = torch.zeros(new + 1, heads, 64, dtype=BF16, device=DEV)
    q[:, :, 0] = 15
    got = paged.paged_attention(q.view(new + 1, -1), batch.cache, batch.tables, batch.lengths, batch.starts, scale=1.0)
    got = got.view(new + 1, heads, 64).cpu()
    odd = [5, 6, 7]
    assert not got[:new, :, odd].isfinite().any()
    rest = [d for d in range(64) if d not in odd]
    # The one entry has all of the weight (the others' sum is below 4000 e^-300): its value, exactly, to the first new token.
    assert torch.equal(got[0][:, rest], batch.values[0][-new, 0, rest].expand(heads, -1))
    assert got[:, :, rest].isfinite().all() and torch.equal(got[new], batch.values[1][-1, 0].expand(heads, -1))


def test_duals_of_forward_mode_are_refused() -> None:
    """No tangent is dropped; inside a level of forward mode, calls without one are as outside of it."""
    print("duals", flush=True)
    batch = Batch([2], [5], 2, 64, 16, BF16, seed=66).fill()
    cache, batch_of = batch.cache, (batch.tables, batch.lengths, batch.starts)
    q, kv = torch.randn(2, 256, generator=batch.g).to(BF16).to(DEV), torch.randn(2, 128, generator=batch.g).to(BF16).to(DEV)
    cos, norm, sinks = torch.rand(9, 32, device=DEV), torch.ones(64, device=DEV), torch.zeros(4, device=DEV)
    parents, kept = torch.tensor([-1, 0], dtype=torch.int32, device=DEV), torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
    append = dict(q=q, k=kv, v=kv, cos=cos, sin=cos, q_norm=norm, k_norm=norm)

    def calls():
        return (paged.paged_append(cache=cache, tables=batch_of[0], lengths=batch_of[1], starts=batch_of[2], **append),
                paged.paged_attention(q, cache, *batch_of, sinks=sinks), paged.paged_tree_attention(q, cache, *batch_of, parents),
                paged.paged_keep(cache, *batch_of, kept))

    def refused(call, *args, **kinds):
        with torch.no_grad(), pytest.raises(LinnetError, match="tangent"):
            call(*args, **kinds)

    want = calls()
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        assert all(torch.equal(a, b) for a, b in zip(calls(), want))
        for name in append:
            refused(paged.paged_append, cache=cache, tables=batch_of[0], lengths=batch_of[1], starts=batch_of[2],
                    **(append | {name: dual(append[name])}))
        refused(paged.paged_append, cache=cache, tables=batch_of[0], lengths=batch_of[1], starts=batch_of[2], out=dual(q.clone()), **append)
        for call, more in ((paged.paged_attention, ()), (paged.paged_tree_attention, (parents,))):
            refused(call, dual(q), cache, *batch_of, *more)
            refused(call, q, cache, *batch_of, *more, sinks=dual(sinks))
            refused(call, q, cache, *batch_of, *more, out=dual(q.clone()))
        for pool in (paged.PagedCache(dual(cache.k), cache.v), paged.PagedCache(cache.k, dual(cache.v))):
            refused(paged.paged_append, cache=pool, tables=batch_of[0], lengths=batch_of[1], starts=batch_of[2], **append)
            refused(paged.paged_attention, q, pool, *batch_of)
            refused(paged.paged_keep, pool, *batch_of, kept)
    refused(torch.func.jvp, lambda x: paged.paged_attention(x, cache, *batch_of), (q,), (q,))


def test_attention_of_a_workspace_at_its_bound() -> None:
    """A mixed batch whose tables could hold more parts than the workspace has room for."""
    print("workspace at its bound", flush=True)
    counts, lengths = [1] * 128, [1 + (37 * i) % 200 for i in range(128)]
    counts[40], counts[70], counts[71] = 20, 3, 16
    for s, n in ((40, 300), (70, 1900), (71, 700), (90, 2600)):
        lengths[s] = n
    batch = Batch(counts, lengths, 16, 64, 128, BF16, seed=47, width=1024).fill()
    assert paged._workspace(128, 1024, 128, batch.tokens, 16, 16, 64, batch.tokens, 0) == 124 * 128 * 16 * 16 * 66  # 128 parts: 2^28 and more
    _attend(batch, 16, sinks=True)
