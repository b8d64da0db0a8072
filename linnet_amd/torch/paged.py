"""A KV cache in pages and what a serving decoder does with it (`csrc/paged_append.hip`,
`csrc/paged_attention.hip`), bf16 or f16: new tokens appended to it (`paged_append`: the norms of
queries and keys and the rotary embedding on the way), attention over it for single tokens, chunks and
prompts in one call (`paged_attention`), the attention of drafted trees (`paged_tree_attention`)
and the move of an accepted path to where its sequence goes on (`paged_keep`).

A batch is three int32 tensors on the device: `tables` [sequences, width], the page ids of each
sequence in order (anything outside the pool, -1 say: no page); `lengths` [sequences], the entries of
each sequence, its new tokens among them; `starts` [sequences + 1], ascending from 0: tokens
`starts[s]` .. `starts[s + 1] - 1` of the call are the last entries of sequence s. The kernels read
them on the device, with bounds checked, so a captured call follows them as they change; tokens from
`starts[-1]` on (the padding of a captured batch) belong to no sequence. An entry without a page is
neither read nor written.

The reference keeps one contiguous cache of one length in its generated module
(`python/linnet/src/linnet/torch/compiled.py:430-503`). Every call enqueues on the current stream and
returns; the kernels record no gradient, and inputs that require one or have a tangent of forward mode
are refused.
"""

from __future__ import annotations

import ctypes
import dataclasses
import functools

import torch
from torch.autograd import forward_ad

from .. import _lib
from ..errors import LinnetError
from .kernels import _aligned, _code, _on_gpu

PAGES = (16, 32, 64, 128)  # entries a page may hold
TREE_NODES = 256  # of a drafted tree
_MOST_TOKENS = 1 << 24  # new tokens of a batch


@dataclasses.dataclass(frozen=True, eq=False)
class PagedCache:
    """The pool of one layer, or of several: `k` [(layers,) pages, kv_heads, head_dim/8, page, 8] and `v`
    [(layers,) pages, kv_heads, page/8, head_dim, 8], bf16 or f16, contiguous. Entry e of a sequence
    lies in its e / page-th page at place e % page: `k[p, h, :, place, :]` is its key (in order),
    `v[p, h, place // 8, :, place % 8]` its value. head_dim 64 or 128, page 16, 32, 64 or 128."""

    k: torch.Tensor
    v: torch.Tensor

    def __post_init__(self) -> None:
        k, v = self.k, self.v
        if k.dim() not in (5, 6) or v.dim() != k.dim():
            raise LinnetError(f"PagedCache: k and v are [(layers,) pages, kv_heads, ...], got {tuple(k.shape)} and {tuple(v.shape)}")
        *lead, kv_heads, eighths, page, eight = k.shape
        if eight != 8 or tuple(v.shape) != (*lead, kv_heads, page // 8, 8 * eighths, 8):
            raise LinnetError("PagedCache: k is [.., kv_heads, head_dim/8, page, 8] and v [.., kv_heads, page/8, head_dim, 8], got "
                              f"{tuple(k.shape)} and {tuple(v.shape)}")
        if page not in PAGES or 8 * eighths not in (64, 128):
            raise LinnetError(f"PagedCache: a page holds 16, 32, 64 or 128 entries and head_dim is 64 or 128, got {page} and {8 * eighths}")
        if kv_heads < 1 or lead[0] < 1 and len(lead) == 2:
            raise LinnetError("PagedCache: no KV heads or no layers")
        if k.dtype != v.dtype or k.device != v.device:
            raise LinnetError("PagedCache: k and v are of one dtype on one device")
        code = _code(k.dtype, "PagedCache")
        if not (k.is_contiguous() and v.is_contiguous()) or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise LinnetError("PagedCache: k and v are contiguous and 16-byte aligned")
        # What each call passes on: (pages, page, kv_heads, head_dim, dtype code, layers).
        object.__setattr__(self, "_sizes", (lead[-1], page, kv_heads, 8 * eighths, code, lead[0] if len(lead) == 2 else 0))

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page: int = 64, dtype: torch.dtype = torch.bfloat16,
              device: torch.device | str = "cuda", layers: int | None = None) -> PagedCache:
        """An uninitialised pool (of `layers` layers). Nothing of it is read before it is written."""
        lead = (pages, kv_heads) if layers is None else (layers, pages, kv_heads)
        return cls(torch.empty(*lead, head_dim // 8, page, 8, dtype=dtype, device=device),
                   torch.empty(*lead, page // 8, head_dim, 8, dtype=dtype, device=device))

    def layer(self, i: int) -> PagedCache:
        """The pool of layer i of several (a view)."""
        if self.k.dim() != 6:
            raise LinnetError("PagedCache.layer: a pool of one layer")
        return PagedCache(self.k[i], self.v[i])


# A call's host time is longer than a decode step's kernels here (10 us against 4), so the checks below are the
# direct forms.
_INT32, _FLOAT32 = torch.int32, torch.float32
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _launch(index: int, name: str, *args: object) -> None:
    """Calls entry point `name` on the current stream of device `index`, its last argument."""
    if index == _current_device():
        _lib.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, _raw_stream(index))


def _records(what: str) -> None:
    raise LinnetError(f"{what}: records no gradient, and an input requires one")


def _tangents(what: str, *tensors: torch.Tensor | None) -> None:
    """Refuses duals, whose tangents the kernels would drop (asked only inside a level of forward mode)."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise LinnetError(f"{what}: records no gradient in forward mode, and an input has a tangent")


def _ints(what: str, name: str, t: torch.Tensor, count: int) -> torch.Tensor:
    if t.dtype is not _INT32 or t.dim() != 1 or t.numel() != count:
        raise LinnetError(f"{what}: {name} is [{count}] int32, got {list(t.shape)} {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _batch(what: str, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor) -> tuple:
    if tables.dtype is not _INT32 or tables.dim() != 2:
        raise LinnetError(f"{what}: tables is [sequences, width] int32, got {list(tables.shape)} {tables.dtype}")
    sequences, width = tables.shape
    return (tables if tables.is_contiguous() else tables.contiguous(), _ints(what, "lengths", lengths, sequences),
            _ints(what, "starts", starts, sequences + 1), sequences, width)


def _rows(what: str, name: str, t: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, int, int, int]:
    """`t` [tokens, width] as the kernels read it (rows of contiguous values, whole 16 bytes apart; column slices
    of a joined projection as they are, anything else copied), its row stride, tokens and width."""
    if t.dtype is not dtype or t.dim() != 2:
        raise LinnetError(f"{what}: {name} is [tokens, width] {dtype} as the cache is, got {list(t.shape)} {t.dtype}")
    rows, width = t.shape
    stride, step = t.stride()
    if rows <= 1:
        stride = width
    if step != 1 or stride % 8 or stride < width or t.data_ptr() % 16:
        t = _aligned(t)
        stride = width
    return t, stride, rows, width


def _floats(what: str, name: str, t: torch.Tensor, count: int) -> torch.Tensor:
    if t.dtype is not _FLOAT32 or t.dim() != 1 or t.numel() != count:
        raise LinnetError(f"{what}: {name} is [{count}] float32, got {list(t.shape)} {t.dtype}")
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else _aligned(t)


def _out(what: str, out: torch.Tensor, rows: int, width: int, dtype: torch.dtype) -> torch.Tensor:
    if out.dtype is not dtype or out.shape != (rows, width) or not out.is_contiguous() or out.data_ptr() % 16:
        raise LinnetError(f"{what}: out is a contiguous, 16-byte aligned [{rows}, {width}] {dtype}, got {list(out.shape)} {out.dtype}")
    return out


def _one_layer(what: str, cache: PagedCache) -> tuple:
    sizes = cache._sizes
    if sizes[5]:
        raise LinnetError(f"{what}: takes one layer's pool (`cache.layer(i)`)")
    return sizes


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor | None, sin: torch.Tensor | None,
                 cache: PagedCache, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
                 positions: torch.Tensor | None = None, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                 eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """The new tokens' keys and values into the cache, and their queries ready for it: q [tokens,
    heads*head_dim], k and v [tokens, kv_heads*head_dim] (the cache's dtype; column slices of a joined
    projection are read in place). Per head, with `q_norm` / `k_norm` (f32 [head_dim]) first `x *
    rsqrt(mean(x^2) + eps) * norm`; then the rotary embedding of the pairs (i, i + half) by `cos`, `sin`
    (f32 [positions, half], as `decode.rope_tables` gives; half a multiple of 8 up to head_dim / 2; both
    None: no rotation), all in f32 and rounded once. A token's position is `positions` ([tokens] int32: those
    of a drafted tree, say), else its entry. Returns the queries [tokens, heads*head_dim]
    (`out`, if given; it may be q itself).

    A token whose position has no row of the tables is not stored and its queries are zeros. Tokens of no
    sequence give zeros, or with `out` leave its rows as they were. Two sequences may share pages, but not
    the places of their new entries."""
    pages, page, kv_heads, head_dim, code, _ = _one_layer("paged_append", cache)
    k_cache, v_cache = cache.k, cache.v
    index = q.get_device()
    if not (0 <= index == k.get_device() == v.get_device() == k_cache.get_device() == tables.get_device() == lengths.get_device()
            == starts.get_device()) or any(t is not None and t.get_device() != index for t in (cos, sin, positions, q_norm, k_norm, out)):
        _on_gpu("paged_append", q, k, v, k_cache, tables, lengths, starts, cos, sin, positions, q_norm, k_norm, out)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_cache.requires_grad
                                    or v_cache.requires_grad or any(t is not None and t.requires_grad
                                                                    for t in (cos, sin, q_norm, k_norm, out))):
        _records("paged_append")
    if forward_ad._current_level >= 0:
        _tangents("paged_append", q, k, v, k_cache, v_cache, cos, sin, q_norm, k_norm, out)
    dtype = k_cache.dtype
    tables, lengths, starts, sequences, width = _batch("paged_append", tables, lengths, starts)
    q, q_stride, tokens, columns = _rows("paged_append", "q", q, dtype)
    k, k_stride, k_rows, k_columns = _rows("paged_append", "k", k, dtype)
    v, v_stride, v_rows, v_columns = _rows("paged_append", "v", v, dtype)
    heads = columns // head_dim
    if columns != heads * head_dim or not k_columns == v_columns == kv_heads * head_dim or not k_rows == v_rows == tokens:
        raise LinnetError(f"paged_append: q is [tokens, heads*{head_dim}], k and v [tokens, {kv_heads * head_dim}], got "
                          f"{list(q.shape)}, {list(k.shape)} and {list(v.shape)}")
    table = half = 0
    at_cos = at_sin = at_positions = at_q_norm = at_k_norm = None
    if cos is not None and sin is not None:
        if cos.dtype is not _FLOAT32 or sin.dtype is not _FLOAT32 or cos.dim() != 2 or cos.shape != sin.shape:
            raise LinnetError(f"paged_append: cos and sin are [positions, half] float32, got {list(cos.shape)} {cos.dtype} and "
                              f"{list(sin.shape)} {sin.dtype}")
        table, half = cos.shape
        if half == 0 or half % 8 or 2 * half > head_dim:
            raise LinnetError(f"paged_append: tables of {half} angles (a multiple of 8, at most {head_dim // 2})")
        cos, sin = _aligned(cos), _aligned(sin)
        at_cos, at_sin = cos.data_ptr(), sin.data_ptr()
    elif cos is not sin:
        raise LinnetError("paged_append: cos and sin come together")
    if positions is not None:
        positions = _ints("paged_append", "positions", positions, tokens)
        at_positions = positions.data_ptr()
    if q_norm is not None:
        q_norm = _floats("paged_append", "q_norm", q_norm, head_dim)
        at_q_norm = q_norm.data_ptr()
    if k_norm is not None:
        k_norm = _floats("paged_append", "k_norm", k_norm, head_dim)
        at_k_norm = k_norm.data_ptr()
    fill = out is None
    if fill:
        out = q.new_empty((tokens, columns))
    else:
        out = _out("paged_append", out, tokens, columns, dtype)
    _launch(index, "lnq_paged_append", q.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride, at_cos, at_sin, table,
            half, at_positions, at_q_norm, at_k_norm, eps, out.data_ptr(), columns, fill, k_cache.data_ptr(), v_cache.data_ptr(),
            tables.data_ptr(), lengths.data_ptr(), starts.data_ptr(), sequences, width, pages, page, tokens, heads, kv_heads, head_dim,
            code)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace(*sizes: int) -> int:
    floats = ctypes.c_int64(0)
    _lib.call("lnq_paged_attention_workspace", *sizes, ctypes.byref(floats))
    return floats.value


def _attend(what: str, q: torch.Tensor, cache: PagedCache, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
            parents: torch.Tensor | None, max_queries: int | None, scale: float | None, window: int | None,
            sinks: torch.Tensor | None, out: torch.Tensor | None) -> torch.Tensor:
    pages, page, kv_heads, head_dim, code, _ = _one_layer(what, cache)
    k_cache = cache.k
    index = q.get_device()
    if not (0 <= index == k_cache.get_device() == tables.get_device() == lengths.get_device() == starts.get_device()) or any(
            t is not None and t.get_device() != index for t in (parents, sinks, out)):
        _on_gpu(what, q, k_cache, tables, lengths, starts, parents, sinks, out)
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or cache.v.requires_grad or any(
            t is not None and t.requires_grad for t in (sinks, out))):
        _records(what)
    if forward_ad._current_level >= 0:
        _tangents(what, q, k_cache, cache.v, sinks, out)
    dtype = k_cache.dtype
    tables, lengths, starts, sequences, width = _batch(what, tables, lengths, starts)
    q, q_stride, tokens, columns = _rows(what, "q", q, dtype)
    heads = columns // head_dim
    if heads == 0 or columns != heads * head_dim or heads % kv_heads:
        raise LinnetError(f"{what}: q is [tokens, heads*{head_dim}], heads a multiple of {kv_heads}, got {list(q.shape)}")
    most = tokens if max_queries is None else int(max_queries)
    if most < 1 and tokens > 0:
        raise LinnetError(f"{what}: max_queries of {most}")
    at_parents = at_sinks = at_work = None
    if parents is not None:
        parents = _ints(what, "parents", parents, tokens)
        at_parents = parents.data_ptr()
    if sinks is not None:
        sinks = _floats(what, "sinks", sinks, heads)
        at_sinks = sinks.data_ptr()
    scale = head_dim**-0.5 if scale is None else float(scale)
    if not 1e-9 <= scale <= 1e9:
        raise LinnetError(f"{what}: the scale is a positive number, not {scale}")
    window = int(window) if window else 0
    fill = out is None
    if fill:
        out = q.new_empty((tokens, columns))
    else:
        out = _out(what, out, tokens, columns, dtype)
    if tokens == 0:
        return out
    floats = _workspace(sequences, width, page, tokens, heads, kv_heads, head_dim, most, window)
    if floats:
        work = q.new_empty((floats,), dtype=_FLOAT32)
        at_work = work.data_ptr()
    _launch(index, "lnq_paged_attention", q.data_ptr(), q_stride, k_cache.data_ptr(), cache.v.data_ptr(), out.data_ptr(), columns,
            fill, tables.data_ptr(), lengths.data_ptr(), starts.data_ptr(), at_parents, at_sinks, at_work, floats, sequences, width,
            pages, page, tokens, heads, kv_heads, head_dim, most, window, scale, code)
    return out


def paged_attention(q: torch.Tensor, cache: PagedCache, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
                    max_queries: int | None = None, scale: float | None = None, window: int | None = None,
                    sinks: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Grouped-query attention of the new tokens' queries q [tokens, heads*head_dim] (as `paged_append` returns
    them, their keys and values in the cache): `softmax(scale q K^T) V` over the entries up to each
    token's own, the last `window` of them with one (0 or None: all); scale head_dim^-0.5 unless given. `sinks`
    (f32 [heads]) add e^sink to each row's sum. Returns [tokens, heads*head_dim] (`out`, if given, which shares
    no memory with the inputs).

    `max_queries`, the most new tokens of a sequence, where the caller knows it, spares the kernels for longer
    ones: 1 for a decode step. Sequences with more are computed all the same. A row that sees no entry, or
    only ones whose score is -inf, gives zeros; infinities and NaNs of a value reach the rows that see its entry
    and no other (an infinity as it is, or as NaN where its weight beside the row's others is 0); tokens of no
    sequence give zeros, or with `out` leave its rows as they were.

    Long contexts of few rows are split over the chip by what the tables can hold. Tables much wider than the
    sequences (131072 entries for some thousands) make a decode step slower and its workspace larger, up to 1 GiB:
    pass the columns that are in use (`tables[:, :n]`, contiguous; in a captured step one of a few widths)."""
    return _attend("paged_attention", q, cache, tables, lengths, starts, None, max_queries, scale, window, sinks, out)


def paged_tree_attention(q: torch.Tensor, cache: PagedCache, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
                         parents: torch.Tensor, max_queries: int | None = None, scale: float | None = None,
                         window: int | None = None, sinks: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """`paged_attention` where each sequence's new tokens are a drafted tree of up to 256 nodes: `parents` [tokens]
    int32 holds each node's parent, an earlier node of its sequence counted from 0, or any other number (-1)
    where it follows the entry before the draft. A node sees the entries before the draft, its ancestors
    and itself; its position is their number, and `window` counts along that path. (`paged_append` of a
    tree takes the nodes' positions.) `max_queries` is at most 256; nodes past the 256th give zeros."""
    if max_queries is not None and max_queries > TREE_NODES:
        raise LinnetError(f"paged_tree_attention: a tree has at most {TREE_NODES} nodes, max_queries is {max_queries}")
    return _attend("paged_tree_attention", q, cache, tables, lengths, starts, parents, max_queries, scale, window, sinks, out)


def paged_keep(cache: PagedCache, tables: torch.Tensor, lengths: torch.Tensor, starts: torch.Tensor,
               kept: torch.Tensor) -> torch.Tensor:
    """The accepted path of each sequence's drafted tokens to where the sequence goes on, in every layer of the pool
    in one launch. `kept` [sequences, path] int32 holds a path's nodes in ascending order, as a path from the
    root has them; it ends at the first number that is no later node of the draft (-1). Node kept[s, j] moves to the
    place of node j. Returns the new lengths ([sequences] int32): the entries before the draft and the path's. The
    places after those hold what they held."""
    pages, page, kv_heads, head_dim, _, layers = cache._sizes
    index = cache.k.get_device()
    _on_gpu("paged_keep", cache.k, tables, lengths, starts, kept)
    if torch.is_grad_enabled() and (cache.k.requires_grad or cache.v.requires_grad):
        _records("paged_keep")
    if forward_ad._current_level >= 0:
        _tangents("paged_keep", cache.k, cache.v)
    tables, lengths, starts, sequences, width = _batch("paged_keep", tables, lengths, starts)
    if kept.dim() != 2:
        raise LinnetError(f"paged_keep: kept is [sequences, path] int32, got {list(kept.shape)}")
    if kept.dtype is not _INT32 or kept.shape[0] != sequences:
        raise LinnetError(f"paged_keep: kept is [{sequences}, path] int32, got {list(kept.shape)} {kept.dtype}")
    kept = kept if kept.is_contiguous() else kept.contiguous()
    new = torch.empty_like(lengths)
    if sequences == 0:
        return new
    _launch(index, "lnq_paged_keep", cache.k.data_ptr(), cache.v.data_ptr(), layers or 1, pages * kv_heads * page * head_dim,
            tables.data_ptr(), lengths.data_ptr(), starts.data_ptr(), kept.data_ptr(), kept.shape[1], new.data_ptr(), sequences,
            width, pages, page, _MOST_TOKENS, kv_heads, head_dim)
    return new
