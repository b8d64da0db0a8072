"""The KV cache in pages without a GPU: what the C ABI refuses before it touches a device, what the wrappers
refuse, and the workspace's size."""

from __future__ import annotations

import ctypes
import itertools

import pytest
import torch

from linnet_amd import LinnetError, _lib
from linnet_amd.torch import paged

NULL = ctypes.c_void_p(0)
FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4104)


def _status(name: str, *args: object) -> tuple[int, str]:
    status = getattr(_lib.load(), name)(*args)
    return status, _lib.last_error()


def _append(**change: object) -> tuple:
    args = dict(q=FAKE, q_stride=512, k=FAKE, k_stride=256, v=FAKE, v_stride=256, cos=FAKE, sin=FAKE, table=10, half=32,
                positions=NULL, q_norm=NULL, k_norm=NULL, eps=1e-6, q_out=FAKE, q_out_stride=512, fill=0, k_cache=FAKE,
                v_cache=FAKE, tables=FAKE, lengths=FAKE, starts=FAKE, sequences=2, width=4, pages=8, page=16, tokens=3, heads=8,
                kv_heads=4, head_dim=64, dtype=0, stream=NULL)
    assert set(change) <= set(args)
    return tuple((args | change).values())


def _attend(**change: object) -> tuple:
    args = dict(q=FAKE, q_stride=512, k_cache=FAKE, v_cache=FAKE, out=FAKE, out_stride=512, fill=0, tables=FAKE, lengths=FAKE,
                starts=FAKE, parents=NULL, sinks=NULL, workspace=FAKE, workspace_floats=1 << 40, sequences=2, width=4, pages=8,
                page=16, tokens=3, heads=8, kv_heads=4, head_dim=64, max_queries=3, window=0, scale=0.1, dtype=0, stream=NULL)
    assert set(change) <= set(args)
    return tuple((args | change).values())


def _keep(**change: object) -> tuple:
    args = dict(k_cache=FAKE, v_cache=FAKE, layers=2, layer_step=8 * 4 * 16 * 64, tables=FAKE, lengths=FAKE, starts=FAKE, kept=FAKE,
                path=3, lengths_out=FAKE, sequences=2, width=4, pages=8, page=16, tokens=3, kv_heads=4, head_dim=64, stream=NULL)
    assert set(change) <= set(args)
    return tuple((args | change).values())


BATCHES = [(dict(page=24), "16, 32, 64 or 128"), (dict(sequences=-1), "sequences"), (dict(sequences=1 << 21), "sequences"),
           (dict(tokens=-1), "new tokens"), (dict(tokens=1 << 25), "new tokens"), (dict(pages=-1), "pages"),
           (dict(width=-1), "2^30"), (dict(width=1 << 27), "2^30"), (dict(head_dim=96), "64 or 128")]


@pytest.mark.parametrize(("change", "message"), BATCHES + [
    (dict(dtype=2), "not bf16 or f16"), (dict(kv_heads=0), "bad heads"), (dict(heads=-1), "bad heads"), (dict(half=4), "multiple of 8"),
    (dict(half=40), "at most head_dim / 2"), (dict(table=-1), "bad tables"), (dict(k=NULL), "null"), (dict(q=NULL), "null"),
    (dict(cos=NULL), "null"), (dict(tables=NULL), "null"), (dict(starts=NULL), "null"), (dict(v_cache=NULL), "null"),
    (dict(q=ODD), "aligned"), (dict(k_cache=ODD), "aligned"), (dict(q_stride=516), "whole 16 bytes"), (dict(q_stride=504), "shorter"),
    (dict(k_stride=0), "shorter"), (dict(tokens=1 << 24, heads=65536, sequences=1), "too large"),
    (dict(tokens=1 << 24, heads=64, q_stride=4096, q_out_stride=4096), "too large"),
])
def test_append_refuses(change: dict, message: str) -> None:
    status, error = _status("lnq_paged_append", *_append(**change))
    assert status == _lib.LNQ_ERROR and message in error, error


@pytest.mark.parametrize(("change", "message"), BATCHES + [
    (dict(dtype=2), "not bf16 or f16"), (dict(kv_heads=3), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"),
    (dict(max_queries=-1), "queries"), (dict(window=-1), "window"), (dict(window=1 << 31), "window"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q=NULL), "null"), (dict(out=NULL), "null"), (dict(lengths=NULL), "null"), (dict(k_cache=NULL), "null"),
    (dict(q=ODD), "aligned"), (dict(out=ODD), "aligned"), (dict(v_cache=ODD), "aligned"), (dict(q_stride=516), "whole 16 bytes"),
    (dict(out_stride=0), "shorter"), (dict(workspace_floats=3, width=1000), "floats"), (dict(workspace=NULL, width=1000), "floats"),
    (dict(tokens=1 << 24, heads=1024), "too many"), (dict(tokens=1 << 24, sequences=1 << 20, heads=64, kv_heads=64), "too many"),
    (dict(sequences=1 << 20, width=1 << 15, heads=64, kv_heads=64), "too many"), (dict(scale=1e10), "scale"), (dict(scale=1e-10), "scale"),
])
def test_attention_refuses(change: dict, message: str) -> None:
    status, error = _status("lnq_paged_attention", *_attend(**change))
    assert status == _lib.LNQ_ERROR and message in error, error


@pytest.mark.parametrize(("change", "message"), BATCHES + [
    (dict(kv_heads=0), "bad shape"), (dict(layers=0), "bad shape"), (dict(path=-1), "bad shape"), (dict(layer_step=64), "overlap"),
    (dict(k_cache=NULL), "null"), (dict(kept=NULL), "null"), (dict(lengths_out=NULL), "null"), (dict(v_cache=ODD), "aligned"),
    (dict(layers=65536, kv_heads=65536, layer_step=1 << 50), "too large"), (dict(layers=1024, sequences=1 << 15), "too large"),
])
def test_keep_refuses(change: dict, message: str) -> None:
    status, error = _status("lnq_paged_keep", *_keep(**change))
    assert status == _lib.LNQ_ERROR and message in error, error


def test_calls_of_nothing_are_fine() -> None:
    assert _status("lnq_paged_append", *_append(tokens=0))[0] == _lib.LNQ_OK
    assert _status("lnq_paged_attention", *_attend(tokens=0))[0] == _lib.LNQ_OK
    assert _status("lnq_paged_keep", *_keep(sequences=0))[0] == _lib.LNQ_OK


def _floats(sequences, width, page, tokens, heads, kv_heads, head_dim, most, window=0) -> int:
    floats = ctypes.c_int64(-1)
    status, error = _status("lnq_paged_attention_workspace", sequences, width, page, tokens, heads, kv_heads, head_dim, most, window,
                            ctypes.byref(floats))
    assert status == _lib.LNQ_OK, error
    return floats.value


def test_workspace_stays_small() -> None:
    """Parts are kept where entries are split, which they are where rows are few."""
    assert _floats(1, 2, 64, 1, 32, 8, 128, 1) == 0 or _floats(1, 2, 64, 1, 32, 8, 128, 1) <= 32 * 130
    assert _floats(1, 2048, 64, 1, 32, 8, 128, 1) <= 256 * 32 * 130
    assert _floats(512, 512, 64, 512, 32, 8, 128, 1) <= 64 * 512 * 32 * 130
    # A long prompt alone: its own rows are not split (the few-row kernel's are).
    assert _floats(1, 128, 64, 8192, 32, 8, 128, 8192) <= 256 * 32 * 16 * 130
    # A window bounds what there is to split.
    assert _floats(1, 2048, 64, 1, 32, 8, 128, 1, 128) <= 4 * 32 * 130


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize(("heads", "kv_heads"), [(1, 1), (4, 2), (40, 1), (32, 8), (64, 64)])
def test_no_sequences_have_no_parts(heads: int, kv_heads: int, head_dim: int) -> None:
    """Tokens of no sequence are only cleared: whatever the tables could hold, no kernel looks for a sequence of theirs."""
    for width, page in ((0, 16), (3, 16), (8, 16), (2048, 64), (1 << 23, 128)):
        for tokens in (1, 16, 50, 64, 300, 8191):
            for most in (0, 1, 2, 33, tokens, 1 << 20):
                for window in (0, 1, 128):
                    assert _floats(0, width, page, tokens, heads, kv_heads, head_dim, most, window) == 0, (width, page, tokens, most, window)


def test_workspace_has_a_bound() -> None:
    """No batch that is taken needs more than 1 GiB, however wide its tables."""
    floats, taken = ctypes.c_int64(-1), 0
    call = _lib.load().lnq_paged_attention_workspace
    for head_dim, page, width in itertools.product((64, 128), (16, 128), (1, 10, 64, 1024, 8192, 1 << 23)):
        for sequences in [3, 700] + [1 << i for i in range(21)]:
            for kv_heads, group in itertools.product((1, 2, 8, 64, 4096), (1, 2, 4, 8, 16, 17, 32, 40)):
                for most, window in ((1, 0), (2, 0), (16, 0), (33, 0), (2000, 0), (2000, 5000)):
                    sizes = (sequences, width, page, sequences + most, kv_heads * group, kv_heads, head_dim, most, window)
                    if call(*sizes, ctypes.byref(floats)) == _lib.LNQ_OK:
                        taken += 1
                        assert 0 <= floats.value <= 1 << 28, sizes
    assert taken > 10000
    # What lies within the bound is divided as it would be without one.
    assert _floats(256, 2048, 64, 256, 32, 8, 128, 1) == 128 * 256 * 32 * 130


CPU = dict(dtype=torch.bfloat16, device="cpu")


def test_cache_shapes() -> None:
    cache = paged.PagedCache.empty(3, 2, 64, 16, **CPU)
    assert cache.k.shape == (3, 2, 8, 16, 8) and cache.v.shape == (3, 2, 2, 64, 8)
    stack = paged.PagedCache.empty(3, 2, 128, 32, torch.float16, "cpu", layers=4)
    assert stack.k.shape == (4, 3, 2, 16, 32, 8) and stack.layer(3).v.shape == (3, 2, 4, 128, 8)
    with pytest.raises(LinnetError, match="one layer"):
        cache.layer(0)
    k, v = cache.k, cache.v
    for bad in ((k[0, 0, 0], v), (k, v[:, :1]), (k, v.half()), (k.float(), v.float()), (k.transpose(0, 1).contiguous().transpose(0, 1), v),
                (torch.zeros(3, 2, 8, 24, 8).bfloat16(), torch.zeros(3, 2, 3, 64, 8).bfloat16()),
                (torch.zeros(3, 2, 12, 16, 8).bfloat16(), torch.zeros(3, 2, 2, 96, 8).bfloat16()),
                (torch.zeros(0, 3, 2, 8, 16, 8).bfloat16(), torch.zeros(0, 3, 2, 2, 64, 8).bfloat16())):
        with pytest.raises(LinnetError):
            paged.PagedCache(*bad)


def test_wrappers_refuse_cpu_tensors() -> None:
    cache = paged.PagedCache.empty(3, 2, 64, 16, **CPU)
    q, kv = torch.zeros(2, 256, **CPU), torch.zeros(2, 128, **CPU)
    tables, lengths, starts = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(LinnetError, match="GPU tensors"):
        paged.paged_append(q, kv, kv, None, None, cache, tables, lengths, starts)
    with pytest.raises(LinnetError, match="GPU tensors"):
        paged.paged_attention(q, cache, tables, lengths, starts)
    with pytest.raises(LinnetError, match="GPU tensors"):
        paged.paged_tree_attention(q, cache, tables, lengths, starts, starts)
    with pytest.raises(LinnetError, match="GPU tensors"):
        paged.paged_keep(cache, tables, lengths, starts, tables)
    with pytest.raises(LinnetError, match="at most 256"):
        paged.paged_tree_attention(q, cache, tables, lengths, starts, starts, max_queries=257)
