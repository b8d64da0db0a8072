"""The router of a mixture of experts, row by row in f64: scores, choice and weights as
`linnet_amd.torch.kernels.expert_route` defines them. The reference runs a router as framework
ops, so nothing of its text is restated; the pin is a brute-force search over the sets of
experts (tests/test_mxfp4_host.py::test_route_against_a_search)."""

from __future__ import annotations

import math

import numpy as np


def expert_route(logits: np.ndarray, top: int, bias: np.ndarray | None = None, score: str = "softmax", groups: int = 1,
                 group_top: int = 1, group_best: int = 2, renormalize: bool = True,
                 scale: float = 1.0) -> tuple[np.ndarray, np.ndarray]:
    """(experts [rows, top] int64, weights [rows, top] f64)."""
    rows, count = logits.shape
    experts = np.full((rows, top), -1, dtype=np.int64)
    weights = np.zeros((rows, top), dtype=np.float64)
    for r in range(rows):
        l = [float(v) for v in logits[r]]
        if any(math.isnan(v) or (score == "softmax" and v == math.inf) for v in l):
            weights[r] = math.nan
            continue
        if score == "softmax":
            most = max(l)
            p = [math.exp(v - most) if v > -math.inf else 0.0 for v in l]
            total = sum(p)
            s = [v / total if total > 0 else 0.0 for v in p]
        else:
            s = [0.0 if v < -700 else 1 / (1 + math.exp(-v)) for v in l]
        if bias is None:
            c = list(l)
        else:
            c = [s[e] + float(bias[e]) if l[e] > -math.inf else -math.inf for e in range(count)]
            c = [-math.inf if math.isnan(v) else v for v in c]
        if groups > 1:
            size = count // groups
            best = min(group_best, size)
            totals = []
            for g in range(groups):
                order = sorted(range(g * size, (g + 1) * size), key=lambda e: (-c[e], e))[:best]
                if any(c[e] == -math.inf for e in order):
                    totals.append(-math.inf)
                else:
                    totals.append(c[order[0]] if best == 1 else sum((s if bias is None else c)[e] for e in order))
            kept = sorted(range(groups), key=lambda g: (-totals[g], g))[:group_top]
            c = [c[e] if e // size in kept else -math.inf for e in range(count)]
        chosen = [e for e in sorted(range(count), key=lambda e: (-c[e], e)) if c[e] > -math.inf][:top]
        total = sum(s[e] for e in chosen)
        for i, e in enumerate(chosen):
            experts[r, i] = e
            weights[r, i] = (s[e] / total if total > 0 else 0.0) * scale if renormalize else s[e] * scale
    return experts, weights
