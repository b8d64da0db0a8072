"""Operators of a KV cache in pages: new tokens appended to it (queries' and keys' norms and the rotary
embedding on the way), attention over it for single tokens, chunks and prompts of a ragged batch, attention
of drafted trees, and the move of an accepted path to where the sequence goes on. Each case is one call as a
program that serves a decoder makes it, through `linnet_amd.torch.paged`; beside it stands the same in
elementary torch operations.

The cache: K [pages, kv_heads, head_dim/8, page, 8] and V [pages, kv_heads, page/8, head_dim, 8]; entry i of
a sequence lies in page tables[sequence, i / page] at place i % page. A batch: `starts` [sequences + 1], where
each sequence's new tokens begin among all new tokens, and `lengths`, its entries with the new ones.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # One sequence's next token in a decoder of 32 query and 8 KV heads: latency.
        _append("append_one_token", "single", 1, 1, 1023, 32, 8, 128, 64, "bf16", False, 128),
        # A decode batch of a model with norms of queries and keys, half of each head rotated.
        _append("append_batch64", "single", 64, 64, 40000, 16, 4, 64, 16, "f16", True, 32),
        # Three prompts in one call.
        _append("append_prompts", "several", 3, 8191, 0, 32, 8, 128, 64, "bf16", True, 128),
        # One token over a context of 1024, latency.
        _attend("attend_one_token", "single", 1, 1, 1023, 32, 8, 128, 64, "bf16", 0, False),
        # A decode batch of contexts of different lengths.
        _attend("attend_batch64", "single", 64, 64, 230000, 32, 8, 128, 64, "bf16", 0, False),
        # One token over a long context, small heads with a sink each.
        _attend("attend_long", "single", 1, 1, 131000, 64, 8, 64, 128, "f16", 0, True),
        # Prompts from their first token on.
        _attend("attend_prompts", "several", 3, 8191, 0, 32, 8, 128, 64, "bf16", 0, False),
        # A chunk of one prompt among decoding sequences, in a layer that looks back 128 tokens and has sinks.
        _attend("attend_mixed_window", "mixed", 33, 2031, 60000, 64, 8, 64, 16, "bf16", 128, True),
        # One sequence's drafted tree.
        _tree("tree_one", 1, 24, 1000, 32, 8, 128, 64, "bf16"),
        # Drafted trees of a batch.
        _tree("tree_batch16", 16, 900, 70000, 32, 8, 128, 64, "bf16"),
        # The accepted path of one sequence, in every layer's cache.
        _keep("keep_one", 32, 1, 24, 100, 8, 128, 64, "bf16"),
        # The accepted paths of a batch.
        _keep("keep_batch48", 32, 48, 2700, 4000, 8, 128, 64, "bf16"),
    ]


def _append(name, mode, sequences, tokens, context, heads, kv_heads, head_dim, page, dtype, norm, rotated):
    return dict(name=name, kind="append", mode=mode, sequences=sequences, tokens=tokens, context=context, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, norm=norm, rotated=rotated)


def _attend(name, mode, sequences, tokens, context, heads, kv_heads, head_dim, page, dtype, window, sinks):
    return dict(name=name, kind="attend", mode=mode, sequences=sequences, tokens=tokens, context=context, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, window=window, sinks=sinks)


def _tree(name, sequences, tokens, context, heads, kv_heads, head_dim, page, dtype):
    return dict(name=name, kind="tree", mode="several", sequences=sequences, tokens=tokens, context=context, heads=heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype)


def _keep(name, layers, sequences, tokens, context, kv_heads, head_dim, page, dtype):
    return dict(name=name, kind="keep", mode="several", layers=layers, sequences=sequences, tokens=tokens, context=context,
                kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype)


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "tree", "tree", "keep"])
    head_dim, page, dtype = rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8]) if kind != "keep" else kv_heads
    if kind == "append":
        sequences = _log(rng, 1, 256)
        tokens = sequences if rng.random() < 0.5 else min(8191, sequences * _log(rng, 2, 4096))
        case = _append("", "single" if tokens == sequences else "several", sequences, tokens, _log(rng, 1, 60000), heads, kv_heads,
                       head_dim, page, dtype, rng.random() < 0.5, rng.choice([head_dim, head_dim, head_dim // 2]))
    elif kind == "attend":
        mode = rng.choice(["single", "single", "several", "several", "mixed"])
        window = rng.choice([0, 0, 0, 100, 1000])
        if mode == "single":
            sequences = _log(rng, 1, 128)
            context = min(sequences * _log(rng, 1, 130000), 230000)
            tokens = sequences
        elif mode == "several":
            sequences = _log(rng, 1, 8)
            tokens = min(8191, sequences * _log(rng, 2, 4096))
            context = 0 if rng.random() < 0.5 else _log(rng, 1, 16000)
            # No more work than the listed prompts' (the longest sequences are about twice the shortest).
            while heads * head_dim * tokens * (context + tokens) > 5e10 * sequences:
                tokens, context = max(2 * sequences, tokens * 2 // 3), context * 2 // 3
        else:
            sequences = rng.randint(2, 48)
            tokens = sequences - 1 + _log(rng, 2, 1000)
            context = sequences * _log(rng, 1, 2000)
        case = _attend("", mode, sequences, tokens, context, heads, kv_heads, head_dim, page, dtype, window, rng.random() < 0.3)
    elif kind == "tree":
        sequences = _log(rng, 1, 24)
        case = _tree("", sequences, sequences * rng.randint(2, 40), min(sequences * _log(rng, 1, 60000), 70000), heads, kv_heads,
                     head_dim, page, dtype)
    else:
        sequences = _log(rng, 1, 48)
        case = _keep("", rng.randint(1, 32), sequences, sequences * rng.randint(2, 40), sequences * _log(rng, 1, 100), kv_heads,
                     head_dim, page, dtype)
    del case["name"]
    return case


# ------------------------------------------------------------------ sizes


def _spread(total, parts, spread=2.0):
    """`total` in `parts` of up to about 1 + `spread` times each other's size, always the same."""
    weight = [1 + spread * ((i * 0.61803398875) % 1) for i in range(parts)]
    ends = [0.0]
    for w in weight:
        ends.append(ends[-1] + w)
    ends = [round(total * e / ends[-1]) for e in ends]
    return [b - a for a, b in zip(ends, ends[1:])]


def _sizes(case):
    """(new tokens, entries with them) of each sequence."""
    sequences, tokens = case["sequences"], case["tokens"]
    if case["mode"] == "mixed":
        counts = [1] * sequences
        counts[sequences // 2] = tokens - sequences + 1
    else:
        counts = _spread(tokens, sequences, 0.0 if case["mode"] == "single" else 0.5 if case["kind"] in ("tree", "keep") else 2.0)
    return counts, [c + n for c, n in zip(_spread(case["context"], sequences), counts)]


# ------------------------------------------------------------------ inputs


def _generator(seed, salt):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + salt)


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _batch(case, g):
    """tables, lengths, starts: the pages of each sequence in any order, -1 past its last."""
    counts, lengths = _sizes(case)
    pages = [-(-n // case["page"]) for n in lengths]
    total = max(1, sum(pages))
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    width, at, rows = max(1, max(pages)), 0, []
    for n in pages:
        rows.append(order[at : at + n] + [-1] * (width - n))
        at += n
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    make = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return make(rows), make(lengths), make(starts), total


def _cache(case, g, pages):
    dtype, lead = DTYPES[case["dtype"]], (case["layers"],) if "layers" in case else ()
    shape = (*lead, pages, case["kv_heads"])
    k = _normal(g, *shape, case["head_dim"] // 8, case["page"], 8, dtype=dtype)
    v = _normal(g, *shape, case["page"] // 8, case["head_dim"], 8, dtype=dtype)
    return k, v


def _parents(case, rng):
    """A tree for each sequence: each node's parent among its earlier ones, -1 for the context's last token."""
    parents = []
    for n in _sizes(case)[0]:
        parents.append([-1 if i == 0 or rng.random() < 0.1 else rng.randrange(max(0, i - 8), i) for i in range(n)])
    return parents


def prepare(case, seed):
    kind = case["kind"]
    g = _generator(seed, {"append": 1, "attend": 2, "tree": 3, "keep": 4}[kind])
    tables, lengths, starts, pages = _batch(case, g)
    k_cache, v_cache = _cache(case, g, pages)
    counts = _sizes(case)[0]
    state = dict(kind=kind, case=case, tables=tables, lengths=lengths, starts=starts, k_cache=k_cache, v_cache=v_cache,
                 most=max(counts))
    dtype, head_dim, tokens = DTYPES[case["dtype"]], case["head_dim"], case["tokens"]
    if kind == "append":
        heads, kv_heads = case["heads"], case["kv_heads"]
        # Column slices of one projection's output, with a few larger channels.
        joined = torch.randn(tokens, (heads + 2 * kv_heads) * head_dim, generator=g, device="cuda")
        joined[:, ::61] *= 4
        joined = joined.to(dtype)
        state["q"], state["k"], state["v"] = joined.split([heads * head_dim, kv_heads * head_dim, kv_heads * head_dim], dim=1)
        half = case["rotated"] // 2
        angle = torch.arange(max(_sizes(case)[1]), device="cuda", dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
        state["cos"], state["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        state["q_norm"] = state["k_norm"] = None
        if case["norm"]:
            state["q_norm"] = 1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda")
            state["k_norm"] = 1 + 0.1 * torch.randn(head_dim, generator=g, device="cuda")
    elif kind == "keep":
        rng = random.Random(int(seed))
        paths = []
        for parents in _parents(case, rng):
            node, path = (rng.randrange(len(parents)) if parents else -1), []
            while node >= 0:
                path.append(node)
                node = parents[node]
            paths.append(path[::-1])
        width = max(1, max(len(p) for p in paths))
        state["kept"] = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32, device="cuda")
    else:
        # Queries that make some entries count more than others, as trained ones do.
        state["q"] = (2 * torch.randn(tokens, case["heads"] * head_dim, generator=g, device="cuda")).to(dtype)
        state["window"] = case.get("window", 0)
        state["sinks"] = torch.randn(case["heads"], generator=g, device="cuda") if case.get("sinks") else None
        state["parents"] = None
        if kind == "tree":
            flat = [p for parents in _parents(case, random.Random(int(seed))) for p in parents]
            state["parents"] = torch.tensor(flat, dtype=torch.int32, device="cuda")
        # Sequences of one new token and of several, which the plain form takes each as one padded batch.
        state["groups"] = [torch.tensor(ids, device="cuda") for ids in ([i for i, n in enumerate(counts) if n == 1],
                                                                        [i for i, n in enumerate(counts) if n > 1]) if ids]
        state["group_most"] = [(max(counts[i] for i in ids), max(_sizes(case)[1][i] for i in ids)) for ids in
                               ([i for i, n in enumerate(counts) if n == 1], [i for i, n in enumerate(counts) if n > 1]) if ids]
    if own:
        from linnet_amd.torch import paged

        state["cache"] = paged.PagedCache(k_cache, v_cache)
    return state


# ------------------------------------------------------------------ the plain form


def _entries(tables, lengths, starts, tokens):
    """(sequence, entry) of each new token."""
    at = torch.arange(tokens, device=starts.device)
    sequence = torch.searchsorted(starts.long(), at, right=True) - 1
    return sequence, (lengths - starts[1:]).long()[sequence] + at


def _head_rows(x, head_dim, norm, cos, sin):
    """x [tokens, heads * head_dim] by heads in 32 bits, normed and rotated."""
    y = x.unflatten(-1, (-1, head_dim)).float()
    if norm is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * norm
    half = cos.shape[-1]
    a, b = y[..., :half], y[..., half : 2 * half]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half :]], dim=-1)


def _append_plain(s):
    page, head_dim = s["case"]["page"], s["case"]["head_dim"]
    sequence, entry = _entries(s["tables"], s["lengths"], s["starts"], s["q"].shape[0])
    cos, sin = s["cos"][entry], s["sin"][entry]
    dtype = s["q"].dtype
    q = _head_rows(s["q"], head_dim, s["q_norm"], cos, sin).to(dtype)
    k = _head_rows(s["k"], head_dim, s["k_norm"], cos, sin).to(dtype)
    pages, place = s["tables"].long()[sequence, entry // page], entry % page
    s["k_cache"][pages, :, :, place] = k.unflatten(-1, (-1, 8))
    s["v_cache"][pages, :, place // 8, :, place % 8] = s["v"].unflatten(-1, (-1, head_dim))
    return dict(q=q.flatten(1), k_cache=s["k_cache"], v_cache=s["v_cache"])


def _ancestors(parents, starts, most):
    """[sequences, most, most]: whether node i is j or below it; and each node's depth [sequences, most]."""
    counts = starts[1:] - starts[:-1]
    node = torch.arange(most, device=starts.device)
    flat = (starts[:-1, None] + node).clamp(max=parents.shape[0] - 1).long()
    up = torch.where(node < counts[:, None], parents[flat].long(), -1)
    # Row `most` stands for "no node". Each round doubles the number of steps taken towards the root.
    step = torch.nn.functional.one_hot(torch.where(up < 0, most, up), most + 1)[..., :most].float()
    reach = torch.eye(most, device=starts.device) + step
    for _ in range(max(1, (most - 1).bit_length())):
        step = torch.bmm(step, step)
        reach = (reach + torch.bmm(step, reach) > 0).float()
    return reach > 0, reach.sum(-1).long() - 1


def _attend_plain(s):
    case = s["case"]
    page, head_dim, heads, kv_heads = case["page"], case["head_dim"], case["heads"], case["kv_heads"]
    out = torch.zeros_like(s["q"])
    for ids, (most, longest) in zip(s["groups"], s["group_most"]):
        lengths, first = s["lengths"][ids].long(), s["starts"][ids].long()
        counts = s["starts"][ids + 1].long() - first
        tables = s["tables"][ids, : -(-longest // page)].long().clamp(min=0)
        batch, room = tables.shape[0], tables.shape[1] * page
        # [batch, kv_heads, head_dim, entries] and [batch, kv_heads, entries, head_dim].
        k = s["k_cache"][tables].permute(0, 2, 3, 5, 1, 4).reshape(batch, kv_heads, head_dim, room).float()
        v = s["v_cache"][tables].permute(0, 2, 1, 3, 5, 4).reshape(batch, kv_heads, room, head_dim).float()
        node = torch.arange(most, device=ids.device)
        live = node < counts[:, None]
        row = torch.where(live, first[:, None] + node, first[:, None])
        q = s["q"][row].float().view(batch, most, kv_heads, -1, head_dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, head_dim)
        score = torch.matmul(q, k).mul_(head_dim**-0.5).view(batch, kv_heads, -1, most, room)
        base, entry = (lengths - counts)[:, None, None], torch.arange(room, device=ids.device)
        if s["parents"] is None:
            at = base + node[:, None]
            seen = entry <= at
            if s["window"]:
                seen = seen & (entry > at - s["window"])
        else:
            reach, _ = _ancestors(s["parents"], s["starts"], most)
            drafted = (entry - base).clamp(0, most - 1).expand(-1, most, -1)
            seen = (entry < base) | ((entry < lengths[:, None, None]) & reach[ids].gather(-1, drafted))
        score.masked_fill_(~seen[:, None, None], -torch.inf)
        top = score.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            sinks = s["sinks"].view(1, kv_heads, -1, 1, 1)
            top = torch.maximum(top, sinks)
        weight = score.sub_(top).exp_()
        total = weight.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            total = total + torch.exp(sinks - top)
        y = torch.matmul(weight.view(batch, kv_heads, -1, room), v).view(batch, kv_heads, -1, most, head_dim) / total
        out[row[live]] = y.permute(0, 3, 1, 2, 4).reshape(batch, most, -1)[live].to(out.dtype)
    return out


def _keep_plain(s):
    page, kept = s["case"]["page"], s["kept"].long()
    base = s["lengths"].long() - (s["starts"][1:] - s["starts"][:-1]).long()
    number = (kept >= 0).sum(-1)
    j = torch.arange(kept.shape[1], device=kept.device)
    # Places past a path's end move its first node again.
    j = torch.where(j < number[:, None], j, 0)
    source = base[:, None] + kept.gather(1, j).clamp(min=0)
    target = base[:, None] + j
    tables = s["tables"].long()
    from_page, to_page = tables.gather(1, source // page), tables.gather(1, target // page)
    a, b = source % page, target % page
    k = s["k_cache"][:, from_page, :, :, a]
    v = s["v_cache"][:, from_page, :, a // 8, :, a % 8]
    s["k_cache"][:, to_page, :, :, b] = k
    s["v_cache"][:, to_page, :, b // 8, :, b % 8] = v
    return dict(lengths=(base + number).int(), k_cache=s["k_cache"], v_cache=s["v_cache"])


# ------------------------------------------------------------------ a pass


def run(state):
    kind = state["kind"]
    if own:
        from linnet_amd.torch import paged

        s = state
        if kind == "append":
            q = paged.paged_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["cache"], s["tables"], s["lengths"], s["starts"],
                                   q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
            return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
        if kind == "attend":
            return paged.paged_attention(s["q"], s["cache"], s["tables"], s["lengths"], s["starts"], max_queries=s["most"],
                                         window=s["window"], sinks=s["sinks"])
        if kind == "tree":
            return paged.paged_tree_attention(s["q"], s["cache"], s["tables"], s["lengths"], s["starts"], s["parents"],
                                              max_queries=s["most"])
        lengths = paged.paged_keep(s["cache"], s["tables"], s["lengths"], s["starts"], s["kept"])
        return dict(lengths=lengths, k_cache=s["k_cache"], v_cache=s["v_cache"])
    if kind == "append":
        return _append_plain(state)
    if kind == "keep":
        return _keep_plain(state)
    return _attend_plain(state)


def work(case):
    kind, kv_heads, head_dim, tokens = case["kind"], case["kv_heads"], case["head_dim"], case["tokens"]
    counts, lengths = _sizes(case)
    if kind == "keep":
        moved = sum(min(n, 1 + math.log2(n + 1)) for n in counts)
        return {"bytes": case["layers"] * moved * 2 * 2 * kv_heads * head_dim * 2, "flops": 0}
    heads = case["heads"]
    if kind == "append":
        return {"bytes": tokens * ((heads + 2 * kv_heads) * head_dim * 4 + case["rotated"] * 4),
                "flops": tokens * (heads + kv_heads) * (3 * case["rotated"] + (4 * head_dim if case["norm"] else 0))}
    window = case.get("window", 0)
    read = pairs = 0
    for n, whole in zip(counts, lengths):
        base = whole - n
        if kind == "tree":
            read += whole
            pairs += n * base + sum(min(i + 1, 1 + math.log2(i + 1)) for i in range(n))
        elif window:
            read += min(whole, n + window - 1)
            full = max(0, n - max(0, window - 1 - base))  # rows that see a whole window
            pairs += full * window + (n - full) * base + (n - full) * (n - full + 1) // 2
        else:
            read += whole
            pairs += n * base + n * (n + 1) // 2
    return {"bytes": 2 * tokens * heads * head_dim * 2 + read * kv_heads * head_dim * 4, "flops": 4 * head_dim * heads * pairs}


# ------------------------------------------------------------------ the same in 64 bits


def _turn(x, norm, cos, sin):
    """One token's heads [heads, head_dim] in 64 bits: each pair (i, i + r) as a complex number times e^(i angle)."""
    if norm is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * norm.double()
    r = cos.shape[-1]
    pair = torch.complex(x[..., :r], x[..., r : 2 * r]) * torch.complex(cos.double(), sin.double())[:, None]
    return torch.cat([pair.real, pair.imag, x[..., 2 * r :]], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    kind, page = case["kind"], case["page"]
    counts, lengths = _sizes(case)
    pages = s["tables"].tolist()
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    first = 0
    if kind == "append":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(counts):
            rows, entries = slice(first, first + n), torch.arange(lengths[i] - n, lengths[i], device="cuda")
            first += n
            cos, sin = s["cos"][entries], s["sin"][entries]
            q, k, v = (s[name][rows].double().reshape(n, -1, case["head_dim"]) for name in ("q", "k", "v"))
            out[rows] = _turn(q, s["q_norm"], cos, sin).flatten(1)
            k = _turn(k, s["k_norm"], cos, sin)
            for p in range((lengths[i] - n) // page, -(-lengths[i] // page)):
                here = (entries // page == p).nonzero()[:, 0]
                if here.numel() == 0:
                    continue
                lo, hi = int(entries[here[0]]) % page, int(entries[here[-1]]) % page + 1
                a, b = int(here[0]), int(here[-1]) + 1
                k_cache[pages[i][p], :, :, lo:hi] = k[a:b].unflatten(-1, (-1, 8)).permute(1, 2, 0, 3)
                dense = v_cache[pages[i][p]].permute(0, 1, 3, 2).reshape(case["kv_heads"], page, -1)
                dense[:, lo:hi] = v[a:b].transpose(0, 1)
                v_cache[pages[i][p]] = dense.view(case["kv_heads"], page // 8, 8, -1).transpose(2, 3)
        return dict(q=out, k_cache=k_cache, v_cache=v_cache)
    if kind == "keep":
        kept = s["kept"].tolist()
        for i, n in enumerate(counts):
            base = lengths[i] - n
            for j, node in enumerate(kept[i]):  # ascending, so no entry is moved before it is read
                if node < 0:
                    break
                a, b = divmod(base + node, page), divmod(base + j, page)
                k_cache[:, pages[i][b[0]], :, :, b[1]] = k_cache[:, pages[i][a[0]], :, :, a[1]].clone()
                v_cache[:, pages[i][b[0]], :, b[1] // 8, :, b[1] % 8] = v_cache[:, pages[i][a[0]], :, a[1] // 8, :, a[1] % 8].clone()
        return dict(lengths=None, k_cache=k_cache, v_cache=v_cache)
    if kind == "tree":
        flat = s["parents"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    for i, n in enumerate(counts):
        rows, whole, base = slice(first, first + n), lengths[i], lengths[i] - n
        used = pages[i][: -(-whole // page)]
        k = torch.cat([k_cache[p].transpose(1, 2).flatten(2) for p in used], dim=1)[:, :whole]
        v = torch.cat([v_cache[p].transpose(2, 3).flatten(1, 2) for p in used], dim=1)[:, :whole]
        place = torch.arange(whole, device="cuda")
        if kind == "tree":
            hidden = torch.ones(n, whole, dtype=torch.bool)
            hidden[:, :base] = False
            for node in range(n):
                up = node
                while up >= 0:
                    hidden[node, base + up] = False
                    up = flat[first + up]
            hidden = hidden.cuda()
        else:
            last = base + torch.arange(n, device="cuda")[:, None]
            hidden = place > last
            if s["window"]:
                hidden |= place + s["window"] <= last
        for h in range(heads):
            q = s["q"][rows, h * case["head_dim"] : (h + 1) * case["head_dim"]].double()
            score = (q @ k[h // group].t().contiguous() / math.sqrt(case["head_dim"])).masked_fill(hidden, -math.inf)
            if s["sinks"] is not None:
                sink = s["sinks"][h].double().expand(n, 1)
                weight = torch.softmax(torch.cat([score, sink], dim=1), dim=1)[:, :whole]
            else:
                weight = torch.softmax(score, dim=1)
            out[rows, h * case["head_dim"] : (h + 1) * case["head_dim"]] = weight @ v[h // group]
        first += n
    return out
