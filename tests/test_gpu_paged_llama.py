"""The int4 Llama-shaped stack over a KV cache in pages (`Int4Llama.paged_step`) against the same stack over its own
contiguous caches: prompts, single tokens of sequences at different lengths, a drafted tree and its accepted path.
Both round q, k, v and the attention's output to bf16 and part in the order of their f32 sums, the paged form also
in the weights rounded to bf16 for their product with V; over two layers the logits agree to the bound the
contiguous step is held to against its own reference (3e-2 of the largest logit)."""

from __future__ import annotations

import pytest
import torch

from linnet_amd.llama import Int4Llama
from linnet_amd.torch import kernels, paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
SMALL = dict(layers=2, hidden=512, heads=8, kv_heads=2, ffn=1536, vocab=1000)


def _x(rows, seed):
    return (torch.randn(rows, 512, generator=torch.Generator().manual_seed(seed)) * 0.5).to(torch.bfloat16).to(DEV)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _close(got, want):
    err, scale = (got.float() - want.float()).abs().max().item(), want.float().abs().max().item()
    print(f"logits max abs err {err:.3e}, rel to max|logit| {err / scale:.3e}", flush=True)
    assert got.shape == want.shape and err <= 3e-2 * scale


def _dense(model, history):
    """The logits after each token of `history` [n, hidden], one sequence over the contiguous caches."""
    logits = [model.prefill(history[:1])]
    for t in range(1, history.shape[0]):
        logits.append(model.step(history[t : t + 1]))
        model.set_position(t + 1)
    return torch.cat(logits)


@pytest.mark.parametrize("page", [16, 64])
def test_paged_steps_match_the_contiguous_caches(page) -> None:
    model = Int4Llama(torch, kernels, DEV, batch=1, seed=5, ctx=64, spare=64, **SMALL)
    prompts = [_x(37, 1), _x(5, 2), _x(70, 3)]
    more = [_x(3, 11), _x(3, 12), _x(3, 13)]
    want = [_dense(model, torch.cat([p, m])) for p, m in zip(prompts, more)]
    cache = model.paged_cache(24, page)
    width = 128 // page
    tables = torch.randperm(24, generator=torch.Generator().manual_seed(4)).int()[: 3 * width].view(3, -1)[:, :width].to(DEV)
    lengths = [0, 0, 0]

    def step(parts, last=True, **kinds):
        counts = [p.shape[0] for p in parts]
        starts = [0]
        for s, n in enumerate(counts):
            lengths[s] += n
            starts.append(starts[-1] + n)
        rows = torch.tensor([e - 1 for e in starts[1:]], device=DEV) if last else None
        return model.paged_step(torch.cat(parts), cache, tables, _i32(lengths), _i32(starts), rows=rows, **kinds)

    # A prompt whole, one in two chunks beside it, and single tokens.
    got = step([prompts[0], prompts[1], prompts[2][:33]])
    _close(got[0], want[0][36]), _close(got[1], want[1][4]), _close(got[2], want[2][32])
    got = step([more[0][:1], more[1][:1], prompts[2][33:]], last=False)
    _close(got[0], want[0][37]), _close(got[1], want[1][5]), _close(got[2:], want[2][33:70])
    got = step([more[0][1:2], more[1][1:2], more[2][:1]], max_queries=1)
    _close(got[0], want[0][38]), _close(got[1], want[1][6]), _close(got[2], want[2][70])


def test_a_drafted_tree_and_its_accepted_path() -> None:
    """Two sequences draft trees; every node's logits are those of its path decoded alone, and after the accepted
    paths are kept the next tokens' too."""
    model = Int4Llama(torch, kernels, DEV, batch=1, seed=6, ctx=64, spare=64, **SMALL)
    prompts, drafts, last = [_x(20, 1), _x(33, 2)], [_x(7, 3), _x(4, 4)], [_x(1, 5), _x(1, 6)]
    parents = [[-1, 0, 0, 1, 2, 4, 4], [-1, -1, 1, 2]]
    kept = [[0, 2, 4, 6], [1, 2, 3, -1]]
    cache = model.paged_cache(8, 16)
    tables = torch.tensor([[5, 2, 7, 0], [1, 6, 3, 4]], dtype=torch.int32, device=DEV)
    model.paged_step(torch.cat(prompts), cache, tables, _i32([20, 33]), _i32([0, 20, 53]))
    positions = []
    paths = []
    for s in range(2):
        for i in range(len(parents[s])):
            path, j = [], i
            while j >= 0:
                path.append(j)
                j = parents[s][j]
            paths.append((s, path[::-1]))
            positions.append(prompts[s].shape[0] + len(path) - 1)
    flat = _i32(parents[0] + parents[1])
    lengths, starts = _i32([27, 37]), _i32([0, 7, 11])
    got = model.paged_step(torch.cat(drafts), cache, tables, lengths, starts, parents=flat, positions=_i32(positions), max_queries=7)
    for t, (s, path) in enumerate(paths):
        _close(got[t], _dense(model, torch.cat([prompts[s], drafts[s][path]]))[-1])
    lengths = paged.paged_keep(cache, tables, lengths, starts, _i32(kept))
    assert lengths.tolist() == [24, 36]
    got = model.paged_step(torch.cat(last), cache, tables, lengths + 1, _i32([0, 1, 2]), max_queries=1)
    for s in range(2):
        path = [n for n in kept[s] if n >= 0]
        _close(got[s], _dense(model, torch.cat([prompts[s], drafts[s][path], last[s]]))[-1])


def test_paged_step_replays_as_a_graph() -> None:
    """A captured step of a padded batch follows tables, lengths and starts: replays give the eager step's logits."""
    model = Int4Llama(torch, kernels, DEV, batch=1, seed=7, ctx=64, spare=64, **SMALL)
    cache, spare = model.paged_cache(12, 16), model.paged_cache(12, 16)
    tables = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4)
    lengths, starts = _i32([10, 20, 0]), _i32([0, 10, 30, 30])
    x = _x(30, 1)
    for pool in (cache, spare):
        model.paged_step(x, pool, tables, lengths, starts)
    lengths, starts, x = _i32([11, 21, 0]), _i32([0, 1, 2, 2]), _x(3, 2)
    model.paged_step(x, spare, tables, lengths, starts, max_queries=1)  # (warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.paged_step(x, cache, tables, lengths, starts, max_queries=1)
    for turn in range(4):
        x.copy_(_x(3, 10 + turn))
        graph.replay()
        torch.cuda.synchronize()
        want = model.paged_step(x, spare, tables, lengths, starts, max_queries=1)
        assert torch.equal(out[:2], want[:2])
        lengths[:2] += 1
        if turn == 1:  # a sequence leaves, another begins
            lengths.copy_(_i32([lengths[0].item(), 0, 1]))
            starts.copy_(_i32([0, 1, 1, 2]))
        elif turn == 2:
            lengths[2] += 1
            lengths[1] = 0
