"""The experts' router on the GPU (`lnq_expert_route`) against the oracle's rows in f64: the same
experts, every one, and weights within an f32 rounding: half a step, 2^-24 relative, of a
quotient whose 64-bit terms err by less than 1e-13."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from linnet_amd import LinnetError
from linnet_amd.torch import kernels
from oracle import route

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _same(got: tuple[torch.Tensor, torch.Tensor], logits: torch.Tensor, top: int, bias: torch.Tensor | None = None, **kw) -> None:
    want_experts, want_weights = route.expert_route(logits.float().cpu().numpy(), top,
                                                    None if bias is None else bias.cpu().numpy(), **kw)
    experts, weights = got[0].cpu().numpy(), got[1].double().cpu().numpy()
    assert got[0].dtype == torch.int64 and got[1].dtype == torch.float32
    bad = (experts != want_experts).any(-1)
    assert not bad.any(), f"rows {np.nonzero(bad)[0][:5]}: {experts[bad][:2]} for {want_experts[bad][:2]}"
    assert np.array_equal(np.isnan(weights), np.isnan(want_weights))
    fine = ~np.isnan(want_weights)
    off = np.abs(weights - want_weights)[fine]
    assert (off <= (2.0 ** -24 + 1e-12) * np.abs(want_weights[fine]) + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize(("rows", "count", "top", "groups", "group_top", "group_best", "biased"), [
    (1, 1, 1, 1, 1, 1, False), (5, 8, 8, 1, 1, 1, True), (33, 32, 4, 1, 1, 2, False), (9, 60, 6, 1, 1, 1, True),
    (40, 64, 6, 8, 3, 1, False), (31, 96, 6, 4, 2, 2, False), (29, 128, 8, 4, 1, 2, True), (65, 256, 8, 8, 4, 2, True),
    (7, 160, 6, 8, 3, 1, True), (3, 384, 12, 1, 1, 1, True), (5, 1000, 64, 1, 1, 1, False), (6, 1024, 64, 64, 8, 2, True),
    (4, 64, 3, 64, 3, 1, True), (4, 66, 2, 33, 2, 2, True)])
def test_route_is_the_oracles(rows, count, top, groups, group_top, group_best, biased, score, dtype) -> None:
    print(f"route {rows} x {count} top={top} groups={groups}/{group_top}/{group_best} {score} {dtype} bias={biased}", flush=True)
    g = torch.Generator().manual_seed(rows * 1000 + count)
    logits = torch.randn(rows, count, generator=g).to(dtype).to(DEV)
    bias = (0.1 * torch.randn(count, generator=g)).to(DEV) if biased else None
    for renormalize, scale in ((True, 2.5), (False, 1.0)):
        kw = dict(score=score, groups=groups, group_top=group_top, group_best=group_best, renormalize=renormalize, scale=scale)
        _same(kernels.expert_route(logits, top, bias, **kw), logits, top, bias, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_ties_go_to_the_lower_index(score: str, biased: bool) -> None:
    """Rows of few distinct values, and biases of few: equal choices everywhere."""
    g = torch.Generator().manual_seed(4)
    logits = torch.randint(-1, 2, (64, 128), generator=g).to(torch.bfloat16).to(DEV)
    logits[0] = 0
    bias = (0.25 * torch.randint(0, 2, (128,), generator=g)).float().to(DEV) if biased else None
    for groups, group_top, best in ((1, 1, 1), (8, 3, 1), (8, 3, 2)):
        kw = dict(score=score, groups=groups, group_top=group_top, group_best=best)
        _same(kernels.expert_route(logits, 8, bias, **kw), logits, 8, bias, **kw)


@pytest.mark.parametrize("best", [1, 2])
def test_groups_that_only_64_bits_tell_apart(best: int) -> None:
    """Groups whose scores differ by less than f32 holds, tie, underflow f32 or pass its largest value."""
    count, groups = 64, 8
    bias = torch.zeros(count)
    logits = torch.full((6, count), -3.0)
    for g in range(groups):
        logits[0, 8 * g] = 1.0 + (g * 5 % 8) * 2.0 ** -23  # neighbours in f32; their scores closer still
        logits[0, 8 * g + 1] = 0.5 + (g * 3 % 8) * 2.0 ** -24
        logits[1, 8 * g] = 2.0
        logits[2, 8 * g] = -120.0 - (g * 3 % 8)
    logits[2, 0::8] -= 30
    logits[3] = -100.0 - 0.25 * torch.arange(count)
    logits[4, :8], logits[4, 32:40] = -float("inf"), -float("inf")
    logits[5] = torch.linspace(-1, 1, count).flip(0)
    for top in (1, 6):
        for score in ("softmax", "sigmoid"):
            kw = dict(score=score, groups=groups, group_top=3, group_best=best)
            _same(kernels.expert_route(logits.to(DEV), top, **kw), logits, top, **kw)
            for b in (bias, bias + 3.0e38, bias + 1024.0):
                _same(kernels.expert_route(logits.to(DEV), top, b.to(DEV), **kw), logits, top, b, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("count", [1, 7, 64])
def test_groups_of_one(count: int, score: str) -> None:
    """A group of one expert goes by that expert, also with the default `group_best` of 2."""
    print(f"groups of one, {count} experts {score}", flush=True)
    g = torch.Generator().manual_seed(count)
    logits = torch.randn(9, count, generator=g).to(DEV)
    bias = (0.3 * torch.randn(count, generator=g)).to(DEV)
    top = min(2, count)
    for b in (None, bias):
        got = kernels.expert_route(logits, top, b, score=score, groups=count, group_top=top)
        _same(got, logits, top, b, score=score)
        _same(got, logits, top, b, score=score, groups=count, group_top=top)


def test_no_experts_and_no_rows() -> None:
    for lead in ((), (2,), (2, 3)):
        with pytest.raises(LinnetError, match="0 experts"):
            kernels.expert_route(torch.empty(*lead, 0, device=DEV), 1)
    for lead in ((0,), (0, 2), (2, 0), (2, 0, 3)):
        experts, weights = kernels.expert_route(torch.empty(*lead, 8, device=DEV), 3)
        assert experts.shape == weights.shape == (*lead, 3)


def test_neighbours_in_the_last_bit() -> None:
    """Choices one f32 step apart, as logits and through the bias: 64 bits tell them apart."""
    g = torch.Generator().manual_seed(6)
    base = torch.randn(200, 1, generator=g)
    logits = base.repeat(1, 32)
    steps = torch.randint(-2, 3, (200, 32), generator=g)
    logits = (logits.view(torch.int32) + steps.int()).view(torch.float32).to(DEV)
    for score in ("softmax", "sigmoid"):
        _same(kernels.expert_route(logits, 6, score=score), logits, 6, score=score)
        bias = torch.zeros(32, device=DEV)
        _same(kernels.expert_route(logits, 6, bias, score=score), logits, 6, bias, score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_rows(score: str) -> None:
    """-inf logits are never chosen; rows that leave fewer than `top`, or nothing, hold -1 and 0;
    the type's lowest value is a logit like others; NaN and +inf rows are NaN."""
    g = torch.Generator().manual_seed(2)
    inf = float("inf")
    logits = torch.randn(12, 40, generator=g)
    logits[0] = -inf
    logits[1, 2:] = -inf
    logits[2, ::2] = -inf
    logits[3] = torch.finfo(torch.float32).min
    logits[4, 5] = torch.finfo(torch.float32).min
    logits[5, 7] = float("nan")
    logits[6, 9] = inf
    logits[7, :39] = -inf
    logits[8] = torch.finfo(torch.float32).max
    logits[9, 3:9] = 30.0
    logits = logits.to(DEV)
    bias = 0.1 * torch.randn(40, generator=g)
    bias[11], bias[12], bias[13] = -inf, inf, float("nan")
    for b in (None, bias.to(DEV)):
        for kw in (dict(), dict(groups=4, group_top=2, group_best=2), dict(groups=8, group_top=3, group_best=1),
                   dict(renormalize=False)):
            _same(kernels.expert_route(logits, 6, b, score=score, **kw), logits, 6, b, score=score, **kw)


def test_shapes_and_strides() -> None:
    wide = torch.randn(3, 4, 48, device=DEV)
    logits = wide[..., 8:40]
    experts, weights = kernels.expert_route(logits, 3)
    assert experts.shape == weights.shape == (3, 4, 3)
    _same((experts.view(12, 3), weights.view(12, 3)), logits.reshape(12, 32), 3)
    rows = wide.view(12, 48)
    for view in (rows[:, 1:33], rows[::2, 3:35], rows[:, ::2], rows[:1].expand(5, 48), torch.randn(32, 7, device=DEV).t()):
        _same(kernels.expert_route(view, 3), view, 3)
    empty = kernels.expert_route(torch.zeros(0, 8, device=DEV), 2)
    assert empty[0].shape == (0, 2)


def test_refusals() -> None:
    logits = torch.zeros(2, 12, device=DEV)
    for call, message in [
        (lambda: kernels.expert_route(logits, 0), "choices a row"),
        (lambda: kernels.expert_route(logits, 13), "choices a row"),
        (lambda: kernels.expert_route(torch.zeros(2, 100, device=DEV), 65), "choices a row"),
        (lambda: kernels.expert_route(logits, 4, groups=4, group_top=1), "choices a row"),
        (lambda: kernels.expert_route(logits, 1, groups=5), "groups"),
        (lambda: kernels.expert_route(logits, 1, groups=4, group_top=5), "groups"),
        (lambda: kernels.expert_route(logits, 1, groups=4, group_best=3), "groups"),
        (lambda: kernels.expert_route(torch.zeros(2, 1025, device=DEV), 1), "experts"),
        (lambda: kernels.expert_route(logits, 1, score="tanh"), "softmax or sigmoid"),
        (lambda: kernels.expert_route(logits, 1, torch.zeros(11, device=DEV)), "bias"),
        (lambda: kernels.expert_route(logits, 1, torch.zeros(12, device=DEV, dtype=torch.bfloat16)), "bias"),
        (lambda: kernels.expert_route(logits.double(), 1), "dtype"),
        (lambda: kernels.expert_route(logits.cpu(), 1), "GPU"),
    ]:
        with pytest.raises(LinnetError, match=message):
            call()
