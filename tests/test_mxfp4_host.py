"""MXFP4 rounding, the product and the router without a GPU: what the C ABI refuses before it
touches a device, what the wrappers refuse, and the oracle's pins."""

from __future__ import annotations

import ctypes
import itertools
import math

import numpy as np
import pytest
import torch

from linnet_amd import LinnetError, _lib
from linnet_amd.torch import kernels, quantized
from oracle import quant, route

NULL = ctypes.c_void_p(0)
FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(4098)


def _status(name: str, *args: object) -> tuple[int, str]:
    status = getattr(_lib.load(), name)(*args)
    return status, _lib.last_error()


@pytest.mark.parametrize(("name", "args", "message"), [
    ("lnq_mxfp4_quantize", (FAKE, FAKE, FAKE, 4, 40, 0, NULL), "in % 32"),
    ("lnq_mxfp4_quantize", (FAKE, FAKE, FAKE, 4, 64, 7, NULL), "dtype 7"),
    ("lnq_mxfp4_quantize", (FAKE, FAKE, FAKE, -1, 64, 0, NULL), "bad shape"),
    ("lnq_mxfp4_quantize", (ODD, FAKE, FAKE, 4, 64, 0, NULL), "aligned"),
    ("lnq_mxfp4_quantize", (NULL, FAKE, FAKE, 4, 64, 0, NULL), "null"),
    ("lnq_mxfp4_dequantize", (FAKE, FAKE, FAKE, 4, 40, 0, NULL), "in % 32"),
    ("lnq_mxfp4_dequantize", (ODD, FAKE, FAKE, 4, 64, 0, NULL), "aligned"),
    ("lnq_mxfp4_dequantize", (FAKE, NULL, FAKE, 4, 64, 0, NULL), "null"),
    ("lnq_mxfp4_rows", (FAKE, 65, FAKE, FAKE, 4, 64, 0, NULL), "aligned"),
    ("lnq_mxfp4_rows", (FAKE, -64, FAKE, FAKE, 4, 64, 0, NULL), "aligned"),
    ("lnq_mxfp4_rows", (FAKE, 64, FAKE, FAKE, 4, 32 * 2 ** 24, 0, NULL), "too large"),
    ("lnq_mxfp4_scale_tiles", (FAKE, FAKE, 1, 4, 40, NULL), "in % 32"),
    ("lnq_mxfp4_scale_tiles", (FAKE, FAKE, 70000, 4, 64, NULL), "too large"),
    ("lnq_mxfp4_linear", (FAKE, 64, FAKE, FAKE, NULL, FAKE, 4, 8, 64, 2, NULL), "bf16 or f16"),
    ("lnq_mxfp4_linear", (FAKE, 64, FAKE, FAKE, NULL, FAKE, 4, 8, 48, 0, NULL), "in % 32"),
    ("lnq_mxfp4_linear", (FAKE, 32, FAKE, FAKE, NULL, FAKE, 4, 8, 64, 0, NULL), "rows of at least in"),
    ("lnq_mxfp4_linear", (FAKE, 1 << 23, FAKE, FAKE, NULL, FAKE, 4, 8, 64, 0, NULL), "less than 2^23"),
    ("lnq_mxfp4_linear", (FAKE, 131072, FAKE, FAKE, NULL, FAKE, 4, 8, 131072, 0, NULL), "inputs"),
    ("lnq_mxfp4_linear", (FAKE, 64, FAKE, FAKE, NULL, FAKE, 70000, 8, 64, 0, NULL), "65535 rows"),
    ("lnq_mxfp4_linear", (FAKE, 64, ODD, FAKE, NULL, FAKE, 4, 8, 64, 0, NULL), "aligned"),
    ("lnq_mxfp4_mm", (FAKE, FAKE, FAKE, FAKE, NULL, FAKE, 4, 8, 64, 2, NULL), "bf16 or f16"),
    ("lnq_mxfp4_mm", (FAKE, FAKE, FAKE, FAKE, NULL, FAKE, 4, 8, 0, 0, NULL), "in % 32"),
    ("lnq_mxfp4_mm", (FAKE, ODD, FAKE, FAKE, NULL, FAKE, 4, 8, 64, 0, NULL), "aligned"),
    ("lnq_mxfp4_mm", (FAKE, FAKE, FAKE, FAKE, NULL, FAKE, 1 << 28, 8, 64, 0, NULL), "2^27"),
    ("lnq_mxfp4_mm", (FAKE, FAKE, FAKE, FAKE, NULL, FAKE, 1 << 27, 1 << 27, 64, 0, NULL), "too large"),
    ("lnq_mxfp4_experts_workspace", (-1, 4, 4, 64, ctypes.byref(ctypes.c_int64())), "pairs"),
    ("lnq_mxfp4_experts_workspace", (4, 4, 4096, 64, ctypes.byref(ctypes.c_int64())), "experts"),
    ("lnq_mxfp4_experts_mm", (FAKE, 64, *[FAKE] * 4, 4, 2, 4096, 8, 64, 1, 0, FAKE, 1 << 30, NULL), "experts=4096"),
    ("lnq_mxfp4_experts_mm", (FAKE, 64, *[FAKE] * 4, 4, 2, 4, 8, 64, 1, 2, FAKE, 1 << 30, NULL), "bf16 or f16"),
    ("lnq_mxfp4_experts_mm", (FAKE, 64, *[FAKE] * 4, 4, 2, 4, 8, 64, 1, 0, FAKE, 16, NULL), "workspace of 16 bytes"),
    ("lnq_mxfp4_experts_mm", (FAKE, 64, *[FAKE] * 4, 4, 2, 4, 8, 64, 1, 0, NULL, 1 << 30, NULL), "workspace"),
    ("lnq_mxfp4_experts_mm", (FAKE, 60, *[FAKE] * 4, 4, 2, 4, 8, 64, 1, 0, FAKE, 1 << 30, NULL), "aligned"),
    ("lnq_mxfp4_experts_mm", (FAKE, 8192, *[FAKE] * 4, 1 << 20, 2, 4, 8, 8192, 1, 0, FAKE, 1 << 40, NULL), "2 GiB"),
    ("lnq_expert_route", (FAKE, 8, NULL, FAKE, FAKE, 4, 8, 9, 1, 1, 1, 1, 1, 1.0, 0, NULL), "choices a row"),
    ("lnq_expert_route", (FAKE, 8, NULL, FAKE, FAKE, 4, 8, 2, 3, 1, 1, 1, 1, 1.0, 0, NULL), "3 groups"),
    ("lnq_expert_route", (FAKE, 8, NULL, FAKE, FAKE, 4, 2048, 2, 1, 1, 1, 1, 1, 1.0, 0, NULL), "2048 experts"),
    ("lnq_expert_route", (FAKE, 8, NULL, FAKE, FAKE, 4, 8, 2, 1, 1, 1, 1, 1, 1.0, 5, NULL), "dtype 5"),
    ("lnq_expert_route", (NULL, 8, NULL, FAKE, FAKE, 4, 8, 2, 1, 1, 1, 1, 1, 1.0, 0, NULL), "null"),
])
def test_the_abi_refuses(name: str, args: tuple, message: str) -> None:
    status, error = _status(name, *args)
    assert status == _lib.LNQ_ERROR and message in error, error


@pytest.mark.parametrize(("sizes", "strides", "message"), [
    ((4, 2, 8, 64, 65568), (65568, 0), "multiple of 32 up to 65536"), ((4, 2, 8, 64, 8208), (8208, 0), "multiple of 32"),
    ((4, 4096, 8, 64, 8224), (8224, 0), "rows choose up to 2048"), ((4, 2, 65535, 64, 8224), (8224, 0), "65534 experts"),
    ((4, 2, 8, 64, 8224), (8224, 1 << 29), "2.29 elements"), ((4, 2, 8, 64, 8224), (-8224, 0), "not negative")])
def test_wide_experts_refuse(sizes: tuple, strides: tuple, message: str) -> None:
    with pytest.raises(LinnetError, match=message):
        _lib.call("lnq_mxfp4_experts", FAKE, *strides, *[FAKE] * 4, *sizes, _lib.BF16, NULL)


@pytest.mark.parametrize(("rows", "pairs"), [(1, 8), (4, 8), (20, 16), (200, 32)])
def test_wide_experts_take_the_grouped_kernel(rows: int, pairs: int) -> None:
    got = ctypes.c_int32(-1)
    for out, width in ((64, 8224), (4096, 14336), (100000, 65536)):
        _lib.call("lnq_mxfp4_experts_plan", rows, 2, 8, out, width, ctypes.byref(got))
        assert got.value == pairs


def test_empty_calls_succeed_without_a_device() -> None:
    for name, args in [
        ("lnq_mxfp4_quantize", (NULL, NULL, NULL, 0, 64, 0, NULL)),
        ("lnq_mxfp4_dequantize", (NULL, NULL, NULL, 4, 0, 0, NULL)),
        ("lnq_mxfp4_rows", (NULL, 64, NULL, NULL, 0, 64, 0, NULL)),
        ("lnq_mxfp4_scale_tiles", (NULL, NULL, 0, 4, 64, NULL)),
        ("lnq_mxfp4_linear", (NULL, 64, NULL, NULL, NULL, NULL, 0, 8, 64, 0, NULL)),
        ("lnq_mxfp4_mm", (NULL, NULL, NULL, NULL, NULL, NULL, 0, 8, 64, 0, NULL)),
        ("lnq_mxfp4_experts_mm", (NULL, 64, *[NULL] * 4, 0, 2, 4, 8, 64, 1, 0, NULL, 0, NULL)),
        ("lnq_expert_route", (NULL, 8, NULL, NULL, NULL, 0, 8, 2, 1, 1, 1, 1, 1, 1.0, 0, NULL)),
    ]:
        assert _status(name, *args)[0] == _lib.LNQ_OK, name


def test_the_wrappers_refuse_cpu_tensors() -> None:
    u8 = lambda *shape: torch.zeros(*shape, dtype=torch.uint8)  # noqa: E731
    for call in (lambda: kernels.mxfp4_quantize(torch.zeros(2, 32)), lambda: kernels.mxfp4_rows(torch.zeros(2, 32)),
                 lambda: kernels.mxfp4_dequantize(u8(2, 1, 16), u8(2, 1), torch.float32),
                 lambda: kernels.mxfp4_scale_tiles(u8(2, 1), 32),
                 lambda: kernels.mxfp4_w4a16(torch.zeros(2, 32).bfloat16(), u8(2, 1, 16), u8(2, 1)),
                 lambda: kernels.mxfp4_mm(u8(2, 16), u8(1, 1, 64, 8), u8(2, 1, 16), u8(1, 1, 64, 8), torch.bfloat16),
                 lambda: kernels.mxfp4_experts_mm(torch.zeros(2, 32).bfloat16(), u8(3, 2, 1, 16), u8(3, 1, 1, 64, 8),
                                                  torch.zeros(2, 1, dtype=torch.int64)),
                 lambda: kernels.expert_route(torch.zeros(2, 8), 2), lambda: quantized.mxfp4_operands(u8(2, 1, 16), u8(2, 1), 1),
                 lambda: quantized.mxfp4_experts_operands(u8(3, 2, 1, 16), u8(3, 2, 1), 1)):
        with pytest.raises(LinnetError, match="GPU"):
            call()


# ------------------------------------------------------------------ the oracle's pins


def test_mxfp4_rounding_by_search() -> None:
    """Each value against all 16 codes by distance, ties to the even code; the scale against the
    definition's logarithm; blocks at both ends of f32."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 32)) * np.exp2(rng.integers(-30, 30, (40, 1)))
    x[0], x[1, :4], x[2] = 0.0, [5.0, 3.5, -2.5, 7.0], 2.0 ** -149
    x[3] = float(np.finfo(np.float32).max)
    x[4, ::3] = 0.25 * np.abs(x[4]).max()
    x = x.astype(np.float32)
    blocks, scales = quant.quantize_mxfp4(x)
    codes = np.stack([blocks & 15, blocks >> 4], -1).reshape(40, 32)
    for r in range(40):
        top = float(np.abs(x[r]).max())
        exponent = -127 if top == 0 else max(math.floor(math.log2(top)) - 2, -127)
        assert scales[r, 0] == exponent + 127
        for v, code in zip(x[r], codes[r]):
            a = abs(float(v)) / 2.0 ** exponent
            best = min(range(8), key=lambda c: (abs(a - float(quant.FP4_VALUES[c])), c & 1))
            assert code & 7 == best and code >> 3 == int(math.copysign(1, v) < 0)
    x[5, 9] = np.inf
    assert quant.quantize_mxfp4(x)[1][5, 0] == 255


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 2])
def test_route_against_a_search(score: str, groups: int) -> None:
    """Over all sets of experts from all allowed groups: the chosen set's choices are the largest."""
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((20, 6))
    bias = 0.3 * rng.standard_normal(6)
    experts, weights = route.expert_route(logits, 2, bias, score=score, groups=groups, group_top=1, group_best=2, scale=2.0)
    for r in range(20):
        e = np.exp(logits[r])
        s = e / e.sum() if score == "softmax" else e / (1 + e)
        c = s + bias
        runs = [list(range(6))] if groups == 1 else [[0, 1, 2], [3, 4, 5]]
        best = max((pair for run in runs for pair in itertools.permutations(run, 2)), key=lambda p: (c[p[0]] + c[p[1]], c[p[0]]))
        assert tuple(experts[r]) == best
        chosen = s[list(best)]
        assert np.allclose(weights[r], 2.0 * chosen / chosen.sum(), rtol=1e-14)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_of_groups_of_one(score: str, biased: bool) -> None:
    """A group of one expert goes by that expert, whatever `group_best`: the best groups' experts are the best experts."""
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((20, 6))
    bias = 0.3 * rng.standard_normal(6) if biased else None
    want = route.expert_route(logits, 2, bias, score=score)
    for best in (1, 2):
        got = route.expert_route(logits, 2, bias, score=score, groups=6, group_top=3, group_best=best)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize(("rows", "chosen", "count", "out", "depth"), [(16, 4, 8, 64, 64), (1, 1, 1, 64, 32), (4000, 4, 32, 5760, 2880),
                                                                       (9, 3, 2048, 100, 288), (300, 8, 4, 30000, 96)])
def test_experts_workspace_of_one_byte_less_is_refused(rows: int, chosen: int, count: int, out: int, depth: int) -> None:
    need = ctypes.c_int64(0)
    _lib.call("lnq_mxfp4_experts_workspace", rows * chosen, rows, count, depth, ctypes.byref(need))
    assert need.value >= rows * chosen * 4
    for space, size in ((FAKE, need.value - 1), (FAKE, 0), (NULL, need.value)):
        with pytest.raises(LinnetError, match="workspace"):
            _lib.call("lnq_mxfp4_experts_mm", FAKE, depth, *[FAKE] * 4, rows, chosen, count, out, depth, 1, _lib.BF16, space, size, NULL)
