"""MXFP4 made and multiplied on the GPU: rounding to MXFP4 and back bit for bit against the
oracle, the 4-bit x 4-bit product, the linear layer and the experts of a prompt against f64
products of the exact values.

Tolerance of a product: the MFMA's products are exact and its f32 sum of K terms errs by at
most K ulps of the terms' magnitudes whatever its order (2^-23 each, rounded or cut), then one
rounding: |got - want| <= K 2^-23 sum|x w| + half a step of the type (bf16 2^-8, f16 2^-11
relative, f16 2^-25 absolute below its normal range), the latter of a value that the former
has moved."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from linnet_amd import LinnetError, _lib
from linnet_amd.torch import kernels, quantized
from oracle import quant

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _values(rng: np.random.Generator, *shape: int, spread: int = 3) -> np.ndarray:
    """Values whose blocks have scales of their own."""
    v = rng.standard_normal(shape).astype(np.float32)
    return v * np.exp2(rng.integers(-spread, spread + 1, (*shape[:-1], shape[-1] // 32))).astype(np.float32).repeat(32, -1)


def _weight(rng: np.random.Generator, *shape: int) -> tuple[torch.Tensor, torch.Tensor, np.ndarray]:
    """(blocks, scales on the GPU, values) of a random weight [..., Out, In]: every code, scales a few steps apart."""
    *lead, depth = shape
    blocks = rng.integers(0, 256, (*lead, depth // 32, 16)).astype(np.uint8)
    scales = rng.integers(120, 127, (*lead, depth // 32)).astype(np.uint8)
    return torch.from_numpy(blocks).to(DEV), torch.from_numpy(scales).to(DEV), quant.dequantize_mxfp4(blocks, scales)


def _rounded(x: torch.Tensor) -> np.ndarray:
    return quant.dequantize_mxfp4(*quant.quantize_mxfp4(x.float().cpu().numpy())).astype(np.float64)


def _check(got: torch.Tensor, x: np.ndarray, w: np.ndarray, bias: torch.Tensor | None = None) -> None:
    assert got.dtype in HALF
    x, w = x.astype(np.float64), w.astype(np.float64)
    want, terms = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        b = bias.double().cpu().numpy()
        want, terms = want + b, terms + np.abs(b)
    sums = (x.shape[-1] + 1) * 2.0 ** -23 * terms
    half = HALF[got.dtype]
    bound = sums + half * (np.abs(want) + sums) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    g = got.double().cpu().numpy()
    off = np.abs(g - want)
    assert np.isfinite(g).all()
    assert (off <= bound).all(), f"{int((off > bound).sum())} of {off.size} past the bound, worst {float((off / bound).max()):.3g}"


# ------------------------------------------------------------------ rounding


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(32,), (1, 64), (3, 5, 96), (33, 2880), (7, 4096), (0, 64), (4, 0)])
def test_quantize_is_the_oracles(dtype: torch.dtype, shape: tuple[int, ...]) -> None:
    print(f"quantize {shape} {dtype}", flush=True)
    rng = np.random.default_rng(sum(shape))
    x = torch.from_numpy(_values(rng, *shape)).to(dtype)
    blocks, scales = kernels.mxfp4_quantize(x.to(DEV))
    assert blocks.shape == (*shape[:-1], shape[-1] // 32, 16) and scales.shape == (*shape[:-1], shape[-1] // 32)
    if x.numel():
        want_blocks, want_scales = quant.quantize_mxfp4(x.float().numpy())
        assert np.array_equal(scales.cpu().numpy(), want_scales)
        assert np.array_equal(blocks.cpu().numpy(), want_blocks)
    back = kernels.mxfp4_dequantize(blocks, scales, dtype)
    want = quant.dequantize_mxfp4(blocks.cpu().numpy(), scales.cpu().numpy()).reshape(shape)
    assert back.dtype == dtype and torch.equal(back.cpu(), torch.from_numpy(want).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_at_every_border(dtype: torch.dtype) -> None:
    """Midpoints, their neighbours in the type, zeros of both signs, the smallest and largest
    magnitudes, at scales over the type's whole range."""
    print(f"borders {dtype}", flush=True)
    top = torch.finfo(dtype)
    points = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0], dtype=dtype)
    bits = points.view(torch.int32 if dtype == torch.float32 else torch.int16)
    points = torch.cat([points, (bits + 1).view(dtype), (bits - (bits > 0).to(bits.dtype)).view(dtype), points + top.eps])
    points = torch.cat([points, -points]).view(4, 32)
    points[:, 0] = 7.75  # the largest: a scale of 1 before the factor below
    low = {torch.float32: -148, torch.bfloat16: -132, torch.float16: -23}[dtype]
    high = {torch.float32: 125, torch.bfloat16: 125, torch.float16: 13}[dtype]
    rows = [(points.double() * 2.0 ** e).to(dtype) for e in range(low, high + 1)]
    rows += [torch.zeros(1, 32, dtype=dtype), -torch.zeros(1, 32, dtype=dtype),
             torch.full((1, 32), top.max, dtype=dtype), torch.full((1, 32), -top.smallest_normal, dtype=dtype),
             torch.full((1, 32), top.smallest_normal * top.eps, dtype=dtype)]
    x = torch.cat(rows)
    assert torch.isfinite(x).all()
    blocks, scales = kernels.mxfp4_quantize(x.to(DEV))
    want_blocks, want_scales = quant.quantize_mxfp4(x.float().numpy())
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(blocks.cpu().numpy(), want_blocks)


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_that_are_not_finite(dtype: torch.dtype) -> None:
    print(f"not finite {dtype}", flush=True)
    x = torch.from_numpy(_values(np.random.default_rng(1), 4, 128)).to(dtype)
    x[0, 5], x[1, 40], x[2, 127] = float("nan"), float("inf"), float("-inf")
    blocks, scales = kernels.mxfp4_quantize(x.to(DEV))
    want_blocks, want_scales = quant.quantize_mxfp4(x.float().numpy())
    assert np.array_equal(scales.cpu().numpy(), want_scales) and (want_scales == 255).sum() == 3
    assert np.array_equal(blocks.cpu().numpy(), want_blocks)
    back = kernels.mxfp4_dequantize(blocks, scales, dtype).view(4, 4, 32).cpu()
    assert torch.equal(back.isnan().all(-1), torch.from_numpy(want_scales == 255))
    assert torch.equal(back.isnan().any(-1), torch.from_numpy(want_scales == 255))


@pytest.mark.parametrize("dtype", TYPES)
def test_dequantize_every_code_and_scale(dtype: torch.dtype) -> None:
    print(f"dequantize {dtype}", flush=True)
    codes = np.arange(256, dtype=np.uint8)[None].repeat(256, 0).reshape(256, 16, 16)
    scales = np.arange(256, dtype=np.uint8)[:, None].repeat(16, 1)
    got = kernels.mxfp4_dequantize(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), dtype).cpu()
    values = np.stack([quant.FP4_VALUES[codes & 15], quant.FP4_VALUES[codes >> 4]], -1).reshape(256, 512).astype(np.float64)
    want = torch.from_numpy(values * np.exp2(np.arange(256.0) - 127)[:, None]).to(torch.float32).to(dtype)
    assert torch.equal(got[:255], want[:255]) and got[255].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize(("rows", "depth"), [(1, 32), (2, 96), (4, 128), (33, 2880), (64, 544), (131, 512), (3, 4128), (0, 64)])
def test_rows_are_quantize_laid_out(rows: int, depth: int, dtype: torch.dtype) -> None:
    print(f"rows {rows} x {depth} {dtype}", flush=True)
    wide = torch.from_numpy(_values(np.random.default_rng(rows + depth), rows, depth + 32)).to(dtype).to(DEV)
    for x in (wide[:, 32:], wide[:, :depth].contiguous()):  # strided rows, packed ones
        q, row_scales = kernels.mxfp4_rows(x)
        blocks, scales = kernels.mxfp4_quantize(x)
        assert torch.equal(q, blocks.view(rows, depth // 2))
        assert torch.equal(row_scales, kernels.mxfp4_scale_tiles(scales, depth))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("at", [0, 3, 4])
def test_rows_of_one_row_of_an_odd_pitch(at: int, dtype: torch.dtype) -> None:
    x = torch.from_numpy(_values(np.random.default_rng(at), 5, 128)).to(dtype).to(DEV)[:, :101].contiguous()[2:3, at : at + 96]
    q, row_scales = kernels.mxfp4_rows(x)
    blocks, scales = kernels.mxfp4_quantize(x.clone(memory_format=torch.contiguous_format))
    assert torch.equal(q, blocks.view(1, 48)) and torch.equal(row_scales, kernels.mxfp4_scale_tiles(scales, 96))


@pytest.mark.parametrize(("lead", "out", "depth"), [((), 1, 32), ((), 128, 256), ((5,), 70, 288), ((2,), 300, 2880)])
def test_scale_tiles(lead: tuple[int, ...], out: int, depth: int) -> None:
    scales = torch.randint(0, 256, (*lead, out, depth // 32), dtype=torch.uint8, device=DEV)
    tiles = kernels.mxfp4_scale_tiles(scales, depth)
    pairs, blocks = -(-depth // 256), -(-out // 64)
    assert tiles.shape == (*lead, pairs, blocks, 64, 8)
    full = torch.zeros(*lead, blocks * 64, pairs * 8, dtype=torch.uint8, device=DEV)
    full[..., :out, : depth // 32] = scales
    # [block, f, r] x [pair, u, j] -> [pair, block, (j, r), (u, f)]
    full = full.view(-1, blocks, 4, 16, pairs, 2, 4).permute(0, 4, 1, 6, 3, 5, 2)
    assert torch.equal(tiles.view(-1), full.reshape(-1))


# ------------------------------------------------------------------ products

SIZES = [(1, 1, 32), (3, 7, 96), (33, 64, 128), (64, 100, 160), (65, 257, 256), (129, 130, 288), (300, 513, 544),
         (40, 96, 2880), (257, 300, 1056)]
# Of 64, 128 and 256 rows a tile, with fewer tiles than workgroups at a time and with more.
WIDE = [(40, 66000, 64), (70, 20600, 96), (400, 17000, 544), (300, 24701, 288), (1030, 14000, 160), (260, 49500, 32)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize(("rows", "out", "depth"), SIZES + WIDE)
def test_mm(rows: int, out: int, depth: int, dtype: torch.dtype, bias: bool) -> None:
    print(f"mm {rows} x {depth} -> {out} {dtype} bias={bias}", flush=True)
    rng = np.random.default_rng(rows * 7 + out + depth)
    x = torch.from_numpy(_values(rng, rows, depth)).to(dtype).to(DEV)
    blocks, scales, w = _weight(rng, out, depth)
    b = torch.from_numpy(rng.standard_normal(out).astype(np.float32)).to(dtype).to(DEV) if bias else None
    q, row_scales = kernels.mxfp4_rows(x)
    y = kernels.mxfp4_mm(q, row_scales, blocks, kernels.mxfp4_scale_tiles(scales, depth), dtype, b)
    assert y.shape == (rows, out)
    _check(y, _rounded(x), w, b)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize(("rows", "out", "depth"), [(1, 1, 32), (1, 4096, 4096), (2, 100, 96), (4, 300, 2880), (8, 65, 544),
                                                    (16, 1000, 1056), (17, 33, 288), (32, 257, 160), (64, 96, 128)])
def test_w4a16(rows: int, out: int, depth: int, dtype: torch.dtype, bias: bool) -> None:
    print(f"w4a16 {rows} x {depth} -> {out} {dtype} bias={bias}", flush=True)
    rng = np.random.default_rng(rows * 7 + out + depth)
    wide = torch.from_numpy(_values(rng, rows, depth + 32)).to(dtype).to(DEV)
    blocks, scales, w = _weight(rng, out, depth)
    b = torch.from_numpy(rng.standard_normal(out).astype(np.float32)).to(dtype).to(DEV) if bias else None
    for x in (wide[:, :depth], wide[:, 32:].contiguous()):
        _check(kernels.mxfp4_w4a16(x, blocks, scales, b), x.float().cpu().numpy(), w, b)


def test_scales_that_are_nan_reach_every_output_of_theirs() -> None:
    """A row's or an output's block with the scale 255 makes that row's or output's values NaN
    and no others, in both products."""
    rng = np.random.default_rng(5)
    rows, out, depth = 40, 72, 288
    x = torch.from_numpy(_values(rng, rows, depth)).to(torch.bfloat16)
    x[3, 287], x[17, 0] = float("inf"), float("nan")
    blocks, scales, w = _weight(rng, out, depth)
    scales[5, 8] = 255
    scales[70, 0] = 255
    want = torch.zeros(rows, out, dtype=torch.bool)
    want[[3, 17]] = True
    want[:, [5, 70]] = True
    operands = quantized.mxfp4_operands(blocks, scales, 1)
    y = quantized.mxfp4_linear(x.to(DEV), operands, None)
    assert torch.equal(y.isnan().cpu(), want) and y[~want].isfinite().all()
    few = quantized.mxfp4_linear(x[:20].to(DEV), operands, None)
    assert torch.equal(few.isnan().cpu()[:3], want[:3]) and few[:3][~want[:3]].isfinite().all()
    widened = quantized.mxfp4_linear(x[:3].float().to(DEV), operands, None)
    assert torch.equal(widened.isnan().cpu(), want[:3])


@pytest.mark.parametrize("scale", [0, 1, 60, 200])
def test_extreme_scales(scale: int) -> None:
    """Products far from 1: scale bytes at and near the ends, still in bf16's range."""
    rng = np.random.default_rng(scale)
    blocks, _, _ = _weight(rng, 40, 160)
    scales = torch.full((40, 5), scale, dtype=torch.uint8, device=DEV)
    w = quant.dequantize_mxfp4(blocks.cpu().numpy(), scales.cpu().numpy())
    # x such that the products are about 1: its own block scales are at the other end.
    power = min(127 - scale, 120)
    x = (torch.from_numpy(_values(rng, 40, 160, spread=0)).double() * 2.0 ** power).to(torch.bfloat16).to(DEV)
    operands = quantized.mxfp4_operands(blocks, scales, 1)
    _check(quantized.mxfp4_linear(x, operands, None), _rounded(x), w)
    _check(quantized.mxfp4_linear(x[:9], operands, None), x[:9].float().cpu().numpy(), w)


def test_nothing_behind_the_last_row_is_read_into_the_sums_or_written() -> None:
    """q, scales and y inside larger buffers: NaN scales and full codes behind the rows change no
    output, and what lies behind y stays."""
    rng = np.random.default_rng(9)
    for rows, out, depth in [(33, 50, 160), (65, 130, 96), (130, 70, 2880), (300, 260, 288)]:
        x = torch.from_numpy(_values(rng, rows, depth)).to(torch.bfloat16).to(DEV)
        blocks, scales, _ = _weight(rng, out, depth)
        q, row_scales = kernels.mxfp4_rows(x)
        tiles = kernels.mxfp4_scale_tiles(scales, depth)
        want = kernels.mxfp4_mm(q, row_scales, blocks, tiles, torch.bfloat16)

        def behind(t: torch.Tensor) -> torch.Tensor:
            room = torch.full((t.numel() + (1 << 16),), 255, dtype=torch.uint8, device=DEV)
            room[: t.numel()] = t.reshape(-1)
            return room

        # Scales of outputs past the last are NaN too.
        pad = torch.full((-(-out // 64) * 64, depth // 32), 255, dtype=torch.uint8, device=DEV)
        pad[:out] = scales
        tiles = kernels.mxfp4_scale_tiles(pad, depth)
        pad = torch.full((-(-rows // 64) * 64, depth // 32), 255, dtype=torch.uint8, device=DEV)
        pad[:rows] = kernels.mxfp4_quantize(x)[1]
        row_scales = kernels.mxfp4_scale_tiles(pad, depth)
        held = [behind(t) for t in (q, row_scales, blocks, tiles)]
        y = torch.full((rows * out + 4096,), 3.0, dtype=torch.bfloat16, device=DEV)
        _lib.call("lnq_mxfp4_mm", *(t.data_ptr() for t in held), None, y.data_ptr(), rows, out, depth, _lib.BF16,
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(y[: rows * out].view(rows, out), want)
        assert (y[rows * out:] == 3.0).all()


@pytest.mark.parametrize("dtype", list(HALF))
def test_linear_takes_the_documented_product(dtype: torch.dtype) -> None:
    rng = np.random.default_rng(3)
    blocks, scales, w = _weight(rng, 96, 288)
    bias = torch.from_numpy(rng.standard_normal(96).astype(np.float32)).to(dtype).to(DEV)
    for rounded in (0, 1):
        operands = quantized.mxfp4_operands(blocks, scales, rounded)
        for rows in (0, 1, 32, 33, 64, 65, 200):
            print(f"linear rounded={rounded} rows={rows} {dtype}", flush=True)
            x = torch.from_numpy(_values(rng, rows, 288)).to(dtype).to(DEV)
            y = quantized.mxfp4_linear(x, operands, bias)
            assert y.shape == (rows, 96) and y.dtype == dtype
            values = _rounded(x) if rounded and rows > 32 else x.float().cpu().numpy()
            if rows:
                _check(y, values, w, bias)
    x = torch.from_numpy(_values(rng, 2, 3, 288)).to(dtype).to(DEV)
    y = quantized.mxfp4_linear(x, operands, None)
    assert y.shape == (2, 3, 96)
    _check(y.view(6, 96), x.view(6, 288).float().cpu().numpy(), w)
    wide = quantized.mxfp4_linear(x.float(), operands, None)
    assert wide.dtype == torch.float32
    torch.testing.assert_close(wide.cpu().double().view(6, 96), torch.from_numpy(x.view(6, 288).double().cpu().numpy() @ w.T.astype(np.float64)),
                               rtol=288 * 2.0 ** -24, atol=288 * 2.0 ** -23 * float(np.abs(w).max() * x.abs().max().item() * 288))


def test_linear_of_no_inputs_and_no_rows() -> None:
    bias = torch.randn(24, device=DEV).to(torch.bfloat16)
    for rounded in (0, 1):
        none = quantized.mxfp4_operands(torch.empty(24, 0, 16, dtype=torch.uint8, device=DEV),
                                        torch.empty(24, 0, dtype=torch.uint8, device=DEV), rounded)
        some = quantized.mxfp4_operands(torch.zeros(24, 2, 16, dtype=torch.uint8, device=DEV),
                                        torch.zeros(24, 2, dtype=torch.uint8, device=DEV), rounded)
        for lead in ((), (3,), (2, 3), (4, 5, 2)):
            y = quantized.mxfp4_linear(torch.empty(*lead, 0, dtype=torch.bfloat16, device=DEV), none, bias)
            assert y.shape == (*lead, 24) and torch.equal(y, bias.expand(*lead, 24))
        for lead in ((0,), (0, 3), (3, 0), (2, 0, 3)):
            assert quantized.mxfp4_linear(torch.empty(*lead, 64, dtype=torch.bfloat16, device=DEV), some, bias).shape == (*lead, 24)
        with pytest.raises(LinnetError, match="mxfp4_linear: x"):
            quantized.mxfp4_linear(torch.zeros((), dtype=torch.bfloat16, device=DEV), some, None)


@pytest.mark.parametrize(("out", "depth"), [(70, 65536), (70, 65568), (4194304, 32)])
def test_linear_of_the_widest_layers(out: int, depth: int) -> None:
    """x is rounded past a few rows at any width, and unrounded up to those."""
    gen = torch.Generator(DEV).manual_seed(depth)
    blocks = torch.randint(0, 256, (out, depth // 32, 16), dtype=torch.uint8, device=DEV, generator=gen)
    scales = torch.randint(120, 127, (out, depth // 32), dtype=torch.uint8, device=DEV, generator=gen)
    operands = quantized.mxfp4_operands(blocks, scales, 1)
    at = torch.tensor(sorted({0, 1, out // 2, out - 1}), device=DEV)
    w = quant.dequantize_mxfp4(blocks[at].cpu().numpy(), scales[at].cpu().numpy())
    for rows in (1, 32, 33, 65):
        print(f"linear {depth} -> {out} rows={rows}", flush=True)
        x = torch.from_numpy(_values(np.random.default_rng(rows), rows, depth)).to(torch.bfloat16).to(DEV)
        y = quantized.mxfp4_linear(x, operands, None)
        _check(y[:, at], _rounded(x) if rows > 32 else x.double().cpu().numpy(), w)


# ------------------------------------------------------------------ experts


def _experts(rng: np.random.Generator, kind: str, rows: int, chosen: int, count: int) -> np.ndarray:
    if kind == "spread":
        return np.stack([rng.permutation(count)[:chosen] if chosen <= count else rng.integers(0, count, chosen) for _ in range(rows)])
    if kind == "one":
        return np.full((rows, chosen), count - 1)
    if kind == "ends":  # choices that are no expert among the others
        e = rng.integers(-2, count + 2, (rows, chosen))
        e[0, 0], e[-1, -1] = -(2 ** 40), 2 ** 40
        return e
    return np.full((rows, chosen), -1)


@pytest.mark.parametrize("kind", ["spread", "one", "ends", "none"])
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize(("rows", "chosen", "count", "out", "depth"), [
    (1, 1, 1, 1, 32), (33, 4, 8, 70, 96), (40, 2, 5, 128, 288), (70, 1, 3, 33, 160), (257, 4, 4, 64, 128),
    (300, 3, 40, 36, 64), (64, 8, 2, 200, 544), (100, 2, 3, 500, 96), (700, 4, 40, 520, 160), (1400, 4, 40, 1100, 96)])
def test_experts_mm(rows: int, chosen: int, count: int, out: int, depth: int, dtype: torch.dtype, kind: str) -> None:
    print(f"experts {kind} rows={rows} chosen={chosen} E={count} {depth} -> {out} {dtype}", flush=True)
    rng = np.random.default_rng(rows + chosen + count + out)
    blocks, scales, w = _weight(rng, count, out, depth)
    tiles = kernels.mxfp4_scale_tiles(scales, depth)
    experts = _experts(rng, kind, rows, chosen, count).astype(np.int64)
    ids = torch.from_numpy(experts).to(DEV)
    for shared in (True, False):
        x = torch.from_numpy(_values(rng, rows if shared else rows * chosen, depth)).to(dtype).to(DEV)
        y = kernels.mxfp4_experts_mm(x, blocks, tiles, ids)
        assert y.shape == (rows, chosen, out)
        values = _rounded(x)
        for e in range(count):
            r, k = np.nonzero(experts == e)
            if r.size:
                _check(y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)], values[r if shared else r * chosen + k], w[e])
        r, k = np.nonzero((experts < 0) | (experts >= count))
        assert not y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)].any()


# Workgroups that are resident at a time, a CU, by the rows of a tile. (Tiles of 64 rows are taken only where those
# of 128 leave CUs idle, at most 160 of them by the average of an expert's pairs: fewer than 1024 of 64.)
RESIDENT = {32: 3, 128: 2, 256: 1}


@pytest.mark.parametrize("kind", ["spread", "ends"])
@pytest.mark.parametrize(("bm", "bn", "rows", "chosen", "count", "out", "depth"), [
    (32, 128, 40, 4, 16, 13549, 96), (32, 128, 60, 4, 16, 12801, 544), (128, 128, 400, 2, 16, 8301, 288),
    (128, 128, 500, 2, 16, 8197, 512), (256, 256, 600, 2, 8, 17003, 160), (256, 256, 700, 2, 8, 16900, 32)])
def test_experts_mm_of_several_tiles_a_workgroup(bm: int, bn: int, rows: int, chosen: int, count: int, out: int, depth: int,
                                                 kind: str) -> None:
    """More tiles than workgroups at a time, two and more rounds of them: tiles that are looked up, loaded and stored
    while others' steps run, of two k-steps and of more."""
    cus = torch.cuda.get_device_properties(DEV).multi_processor_count
    rng = np.random.default_rng(rows + count)
    experts = _experts(rng, kind, rows, chosen, count).astype(np.int64)
    buckets = np.bincount(np.where((experts < 0) | (experts >= count), count, experts).ravel(), minlength=count + 1)
    tiles = int((-(-buckets // bm)).sum()) * -(-out // bn)
    print(f"experts {kind} {rows} x {chosen} of {count} {depth} -> {out}: {tiles} tiles of {bm} x {bn}", flush=True)
    assert tiles > 2 * RESIDENT[bm] * cus
    dtype = torch.bfloat16 if kind == "spread" else torch.float16
    gen = torch.Generator(DEV).manual_seed(rows)
    blocks = torch.randint(0, 256, (count, out, depth // 32, 16), dtype=torch.uint8, device=DEV, generator=gen)
    scales = torch.randint(120, 127, (count, out, depth // 32), dtype=torch.uint8, device=DEV, generator=gen)
    tiles = kernels.mxfp4_scale_tiles(scales, depth)
    ids = torch.from_numpy(experts).to(DEV)
    for shared in (True, False):
        x = torch.from_numpy(_values(rng, rows if shared else rows * chosen, depth)).to(dtype).to(DEV)
        y = kernels.mxfp4_experts_mm(x, blocks, tiles, ids)
        values = _rounded(x)
        for e in range(count):
            r, k = np.nonzero(experts == e)
            w = quant.dequantize_mxfp4(blocks[e].cpu().numpy(), scales[e].cpu().numpy())
            _check(y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)], values[r if shared else r * chosen + k], w)
        r, k = np.nonzero((experts < 0) | (experts >= count))
        assert not y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)].any()


def test_experts_linear_takes_the_documented_product() -> None:
    rng = np.random.default_rng(11)
    count, out, depth = 6, 96, 160
    blocks, scales, w = _weight(rng, count, out, depth)
    for rounded in (0, 1):
        operands = quantized.mxfp4_experts_operands(blocks, scales, rounded)
        for rows in (1, 32, 33, 100):
            experts = torch.from_numpy(_experts(rng, "spread", rows, 2, count)).to(DEV)
            for shape in ((rows, depth), (rows, 2, depth)):
                print(f"experts_linear rounded={rounded} {shape}", flush=True)
                x = torch.from_numpy(_values(rng, *shape)).to(torch.bfloat16).to(DEV)
                y = quantized.mxfp4_experts_linear(x, operands, experts)
                values = _rounded(x) if rounded and rows > 32 else x.double().cpu().numpy()
                pairs = values if len(shape) == 3 else values[:, None].repeat(2, 1)
                for e in range(count):
                    r, k = np.nonzero(experts.cpu().numpy() == e)
                    if r.size:
                        _check(y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)], pairs[r, k], w[e])


@pytest.mark.parametrize("rounded", [0, 1])
@pytest.mark.parametrize("rows", [1, 32, 33])
@pytest.mark.parametrize(("depth", "out"), [(8192, 40), (8224, 40), (14336, 65), (65536, 70)])
def test_experts_linear_of_wide_layers(depth: int, out: int, rows: int, rounded: int) -> None:
    """A layer's width is taken at one token as over a prompt."""
    print(f"wide experts {depth} -> {out} rows={rows} rounded={rounded}", flush=True)
    rng = np.random.default_rng(rows + depth)
    count, chosen = 3, 2
    blocks, scales, w = _weight(rng, count, out, depth)
    operands = quantized.mxfp4_experts_operands(blocks, scales, rounded)
    experts = _experts(rng, "spread", rows, chosen, count)
    experts[-1, 1] = -1
    for shape in ((rows, depth), (rows, chosen, depth)):
        x = torch.from_numpy(_values(rng, *shape)).to(torch.bfloat16).to(DEV)
        y = quantized.mxfp4_experts_linear(x, operands, torch.from_numpy(experts).to(DEV))
        values = _rounded(x) if rounded and rows > 32 else x.double().cpu().numpy()
        pairs = values if len(shape) == 3 else values[:, None].repeat(chosen, 1)
        for e in range(count):
            r, k = np.nonzero(experts == e)
            if r.size:
                _check(y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)], pairs[r, k], w[e])
        assert not y[-1, 1].any()


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize(("rows", "chosen", "count", "out", "depth"), [
    (1, 1, 2, 8, 8224), (40, 2, 2, 130, 46080), (9, 4, 5, 33, 65536), (300, 2, 3, 72, 16384), (700, 4, 300, 9, 8224)])
def test_wide_experts_at_decode(rows: int, chosen: int, count: int, out: int, depth: int, dtype: torch.dtype) -> None:
    """`mxfp4_experts` past the width a pair's workgroup holds: each number of pairs a pass, and the widest rows' scales."""
    print(f"mxfp4_experts {rows} x {chosen} of {count} {depth} -> {out} {dtype}", flush=True)
    rng = np.random.default_rng(rows + depth)
    blocks, scales, w = _weight(rng, count, out, depth)
    experts = _experts(rng, "ends", rows, chosen, count).astype(np.int64)
    x = torch.from_numpy(_values(rng, rows, depth)).to(dtype).to(DEV)
    y = kernels.mxfp4_experts(x[:, None].expand(rows, chosen, depth), blocks, scales, torch.from_numpy(experts).to(DEV))
    values = x.double().cpu().numpy()
    for e in range(count):
        r, k = np.nonzero(experts == e)
        if r.size:
            _check(y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)], values[r], w[e])
    r, k = np.nonzero((experts < 0) | (experts >= count))
    assert not y[torch.from_numpy(r).to(DEV), torch.from_numpy(k).to(DEV)].any()


def _halves(rng: np.random.Generator, rows: int, shape: tuple[int, ...]) -> tuple:
    """x of -2 .. 2 and weights of scale 1: every product is a multiple of 1/2 and every sum of them exact in f32, in any
    order and with x rounded or not. (x, blocks, scales, weights.)"""
    x = torch.from_numpy(rng.integers(-2, 3, (rows, shape[-1])).astype(np.float32))
    blocks = rng.integers(0, 256, (*shape[:-1], shape[-1] // 32, 16)).astype(np.uint8)
    scales = np.full((*shape[:-1], shape[-1] // 32), 127, dtype=np.uint8)
    w = torch.from_numpy(quant.dequantize_mxfp4(blocks, scales)).double().to(DEV)
    return x.to(DEV), torch.from_numpy(blocks).to(DEV), torch.from_numpy(scales).to(DEV), w


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows", [1, 5, 20, 33, 300])
@pytest.mark.parametrize(("out", "depth"), [(70, 96), (65, 2880), (40, 8192), (130, 8224), (70, 46080), (33, 65536), (33, 65568)])
def test_sums_of_wide_layers_are_exact(out: int, depth: int, rows: int, dtype: torch.dtype) -> None:
    """Where no sum is rounded, only the output is: each of the inputs counts, once."""
    print(f"exact {depth} -> {out} rows={rows} {dtype}", flush=True)
    x, blocks, scales, w = _halves(np.random.default_rng(rows + depth), rows, (3, out, depth))
    experts = torch.from_numpy(np.random.default_rng(rows).integers(0, 3, (rows, 2))).to(DEV)
    want = torch.stack([x.double() @ w[e].T for e in range(3)], 1).float().to(dtype)
    pairs = want.gather(1, experts[..., None].expand(rows, 2, out))
    for rounded in (0, 1):
        assert torch.equal(quantized.mxfp4_linear(x.to(dtype), quantized.mxfp4_operands(blocks[0], scales[0], rounded), None), want[:, 0])
        if depth <= 65536 or (rounded and rows > 32):
            operands = quantized.mxfp4_experts_operands(blocks, scales, rounded)
            assert torch.equal(quantized.mxfp4_experts_linear(x.to(dtype), operands, experts), pairs)


def test_rows_are_rounded_at_any_width() -> None:
    """x of 1.2, which rounds to 1 (4.8 in its block's scale goes to 4), times weights of 1."""
    for depth in (65536, 65568):
        blocks = torch.full((8, depth // 32, 16), 0x22, dtype=torch.uint8, device=DEV)
        scales = torch.full((8, depth // 32), 127, dtype=torch.uint8, device=DEV)
        x = torch.full((33, depth), 1.2, dtype=torch.bfloat16, device=DEV)
        y = quantized.mxfp4_linear(x, quantized.mxfp4_operands(blocks, scales, 1), None)
        assert (y == torch.tensor(depth, dtype=torch.bfloat16, device=DEV)).all()


def test_wide_experts_of_far_rows() -> None:
    """Rows of x 2^28 elements apart: more than a launch's offsets hold."""
    rng = np.random.default_rng(3)
    blocks, scales, w = _weight(rng, 2, 24, 8224)
    far = torch.empty(2 * 2 ** 28 + 8224, dtype=torch.bfloat16, device=DEV)
    x = far.as_strided((3, 1, 8224), (2 ** 28, 8224, 1))
    x.copy_(torch.from_numpy(_values(rng, 3, 1, 8224)))
    y = kernels.mxfp4_experts(x, blocks, scales, torch.tensor([[1], [0], [1]], device=DEV))
    for r, e in enumerate((1, 0, 1)):
        _check(y[r], x[r].double().cpu().numpy(), w[e])


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rounded", [0, 1])
@pytest.mark.parametrize(("rows", "chosen", "depth"), [(1, 2, 96), (2, 3, 8192), (2, 3, 8224), (32, 4, 96), (40, 2, 288)])
def test_choices_of_no_expert_are_zeros_whatever_x_holds(rows: int, chosen: int, depth: int, rounded: int, dtype: torch.dtype) -> None:
    print(f"no expert rows={rows} chosen={chosen} {depth} rounded={rounded} {dtype}", flush=True)
    rng = np.random.default_rng(rows + depth)
    blocks, scales, _ = _weight(rng, 4, 40, depth)
    operands = quantized.mxfp4_experts_operands(blocks, scales, rounded)
    experts = rng.integers(0, 4, (rows, chosen))
    experts[0, 0], experts[-1, -1] = -1, 4
    x = torch.from_numpy(_values(rng, rows, depth)).to(dtype)
    x[0, 5], x[-1, depth - 1] = float("inf"), float("nan")
    y = quantized.mxfp4_experts_linear(x.to(DEV), operands, torch.from_numpy(experts).to(DEV)).cpu()
    none = torch.from_numpy((experts < 0) | (experts > 3))
    assert not y[none].any()
    if rows > 2:
        assert y[1:-1].isfinite().all() and y[-1][~none[-1]].isnan().all()


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rounded", [0, 1])
@pytest.mark.parametrize(("rows", "chosen", "depth"), [(1, 1, 288), (2, 3, 2112), (20, 2, 288), (32, 4, 96), (40, 2, 288), (600, 4, 96)])
def test_experts_scales_that_are_nan(rows: int, chosen: int, depth: int, rounded: int, dtype: torch.dtype) -> None:
    """A block with the scale 255 (as `mxfp4_quantize` marks one that is not finite, its codes 0) makes its output of
    its expert NaN, and no other value, whichever kernel takes the rows."""
    print(f"experts nan rows={rows} chosen={chosen} {depth} rounded={rounded} {dtype}", flush=True)
    rng = np.random.default_rng(rows)
    count, out = 4, 72
    blocks, scales, _ = _weight(rng, count, out, depth)
    for e, o, g in ((0, 0, 0), (1, 5, depth // 32 - 1), (3, 71, depth // 64)):
        scales[e, o, g] = 255
        blocks[e, o, g] = 0
    experts = rng.integers(-1, count, (rows, chosen))
    experts[0, 0] = 1
    want = torch.zeros(rows, chosen, out, dtype=torch.bool)
    for e, o in ((0, 0), (1, 5), (3, 71)):
        want[..., o] |= torch.from_numpy(experts == e)
    operands = quantized.mxfp4_experts_operands(blocks, scales, rounded)
    x = torch.from_numpy(_values(rng, rows, depth)).to(dtype).to(DEV)
    y = quantized.mxfp4_experts_linear(x, operands, torch.from_numpy(experts).to(DEV)).cpu()
    assert torch.equal(y.isnan(), want) and y[~want].isfinite().all()


# ------------------------------------------------------------------ refusals, streams, graphs


@pytest.mark.parametrize(("rows", "out", "depth"), [(70001, 40000, 32), (140000, 64, 32768), (40, 140000, 65536)])
def test_offsets_past_32_bits(rows: int, out: int, depth: int) -> None:
    """More than 2^31 outputs, codes of x and of the weight: rows and outputs of both ends and between."""
    print(f"mm {rows} x {depth} -> {out}", flush=True)
    gen = torch.Generator(DEV).manual_seed(rows)
    code = [torch.randint(0, 256, (n, depth // 32, 16), dtype=torch.uint8, device=DEV, generator=gen) for n in (rows, out)]
    scale = [torch.randint(120, 127, (n, depth // 32), dtype=torch.uint8, device=DEV, generator=gen) for n in (rows, out)]
    y = kernels.mxfp4_mm(code[0].view(rows, -1), kernels.mxfp4_scale_tiles(scale[0], depth), code[1],
                         kernels.mxfp4_scale_tiles(scale[1], depth), torch.bfloat16)
    at = [torch.tensor(sorted({0, 1, n // 3, n // 2, n - 2, n - 1}), device=DEV) for n in (rows, out)]
    values = [quant.dequantize_mxfp4(c[i].cpu().numpy(), s[i].cpu().numpy()) for c, s, i in zip(code, scale, at)]
    _check(y[at[0]][:, at[1]], *values)


def test_experts_past_32_bits() -> None:
    """Expert weights of more than 2^32 bytes, the last expert's among those read."""
    rows, chosen, count, out, depth = 40, 2, 65, 8192, 16384
    gen = torch.Generator(DEV).manual_seed(1)
    blocks = torch.randint(0, 256, (count, out, depth // 32, 16), dtype=torch.uint8, device=DEV, generator=gen)
    scales = torch.randint(120, 127, (count, out, depth // 32), dtype=torch.uint8, device=DEV, generator=gen)
    x = torch.randn(rows, depth, device=DEV, generator=gen).to(torch.bfloat16)
    experts = torch.randint(0, count, (rows, chosen), device=DEV, generator=gen)
    experts[0], experts[-1] = count - 1, torch.tensor([0, count - 1], device=DEV)
    y = kernels.mxfp4_experts_mm(x, blocks, kernels.mxfp4_scale_tiles(scales, depth), experts)
    at = torch.tensor([0, 1, out // 2, out - 1], device=DEV)
    values = _rounded(x)
    for r, k in ((0, 0), (0, 1), (7, 1), (rows - 1, 0), (rows - 1, 1)):
        e = int(experts[r, k])
        w = quant.dequantize_mxfp4(blocks[e, at].cpu().numpy(), scales[e, at].cpu().numpy())
        _check(y[r, k, at][None], values[r : r + 1], w)


@pytest.mark.parametrize(("rows", "chosen"), [(1, 1), (1, 3), (3, 1), (6, 2)])
@pytest.mark.parametrize(("pitch", "at"), [(101, 0), (101, 3), (96, 0), (96, 4), (104, 0)])
def test_experts_at_decode_of_views(rows: int, chosen: int, pitch: int, at: int) -> None:
    """x of an odd pitch, of one row or one choice too, and packed but off 16 bytes; blocks off 16 bytes: as packed ones."""
    print(f"mxfp4_experts of a view {rows} x {chosen} pitch={pitch} at={at}", flush=True)
    rng = np.random.default_rng(rows)
    blocks, scales, _ = _weight(rng, 5, 72, 96)
    ids = torch.from_numpy(rng.integers(0, 5, (rows, chosen))).to(DEV)
    room = torch.from_numpy(_values(rng, 1, 4096)[0]).to(torch.bfloat16).to(DEV)
    x = room[at : at + rows * chosen * pitch].view(rows, chosen, pitch)[..., :96]
    want = kernels.mxfp4_experts(x.clone(memory_format=torch.contiguous_format), blocks, scales, ids)
    assert torch.equal(kernels.mxfp4_experts(x, blocks, scales, ids), want)
    off = torch.empty(blocks.numel() + 8, dtype=torch.uint8, device=DEV)[8:].view(blocks.shape).copy_(blocks)
    assert torch.equal(kernels.mxfp4_experts(x, off, scales, ids), want)
    if chosen == 1:
        operands = quantized.mxfp4_experts_operands(blocks, scales, 1)
        assert torch.equal(quantized.mxfp4_experts_linear(x[:, 0], operands, ids), want)


@pytest.mark.parametrize("rows", [20, 45])
def test_experts_of_views(rows: int) -> None:
    """x with gaps between its rows, transposed and expanded, experts in 32 bits and of a view: as packed ones."""
    rng = np.random.default_rng(rows)
    blocks, scales, _ = _weight(rng, 5, 72, 96)
    operands = quantized.mxfp4_experts_operands(blocks, scales, 1)
    wide = torch.from_numpy(_values(rng, rows, 160)).to(torch.bfloat16).to(DEV)
    ids = torch.from_numpy(rng.integers(0, 5, (rows, 6))).to(DEV)
    for x in (wide[:, 32:128], wide[:, 4:100], wide[:, :96].t().contiguous().t(), wide[:1, :96].expand(rows, 96)):
        want = quantized.mxfp4_experts_linear(x.contiguous(), operands, ids[:, ::2].contiguous())
        assert torch.equal(quantized.mxfp4_experts_linear(x, operands, ids[:, ::2]), want)
        assert torch.equal(quantized.mxfp4_experts_linear(x, operands, ids[:, ::2].to(torch.int32)), want)
        each = x[:, None, :].expand(rows, 3, 96)
        assert torch.equal(quantized.mxfp4_experts_linear(each, operands, ids[:, ::2]), want)
    plain = quantized.mxfp4_operands(blocks[0], scales[0], 1)
    for x in (wide[:, 32:128], wide[:, 4:100], wide[:, :96].t().contiguous().t(), wide[:1, :96].expand(rows, 96)):
        assert torch.equal(quantized.mxfp4_linear(x, plain, None), quantized.mxfp4_linear(x.contiguous(), plain, None))


def test_refusals() -> None:
    u8 = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=DEV)  # noqa: E731
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    for call, message in [
        (lambda: kernels.mxfp4_quantize(torch.zeros(4, 40, device=DEV)), "In % 32"),
        (lambda: kernels.mxfp4_quantize(torch.zeros(4, 64, dtype=torch.float64, device=DEV)), "dtype"),
        (lambda: kernels.mxfp4_dequantize(u8(4, 2, 15), u8(4, 2), torch.float32), "16"),
        (lambda: kernels.mxfp4_dequantize(u8(4, 2, 16), u8(4, 3), torch.float32), "scales"),
        (lambda: kernels.mxfp4_rows(torch.zeros(4, 2, 64, device=DEV)), "rows, In"),
        (lambda: kernels.mxfp4_scale_tiles(u8(4, 2), 96), "scales are"),
        (lambda: kernels.mxfp4_w4a16(x, u8(8, 3, 16), u8(8, 3)), "against"),
        (lambda: kernels.mxfp4_w4a16(x.float(), u8(8, 2, 16), u8(8, 2)), "dtype"),
        (lambda: kernels.mxfp4_w4a16(x, u8(8, 2, 16), u8(8, 2), torch.zeros(8, device=DEV)), "bias"),
        (lambda: kernels.mxfp4_mm(u8(4, 32), u8(1, 1, 64, 8), u8(8, 3, 16), u8(1, 1, 64, 8), torch.bfloat16), "against"),
        (lambda: kernels.mxfp4_mm(u8(4, 32), u8(1, 2, 64, 8), u8(8, 2, 16), u8(1, 1, 64, 8), torch.bfloat16), "scale tiles"),
        (lambda: kernels.mxfp4_mm(u8(4, 32), u8(1, 1, 64, 8), u8(8, 2, 16), u8(2, 1, 64, 8), torch.bfloat16), "scale tiles"),
        (lambda: kernels.mxfp4_mm(u8(4, 32), u8(1, 1, 64, 8), u8(8, 2, 16), u8(1, 1, 64, 8), torch.float32), "dtype"),
        (lambda: kernels.mxfp4_experts_mm(x[:3], u8(2, 8, 2, 16), u8(2, 1, 1, 64, 8),
                                          torch.zeros(4, 2, dtype=torch.int64, device=DEV)), "against"),
        (lambda: kernels.mxfp4_experts_mm(x, u8(2, 8, 2, 16), u8(2, 1, 1, 64, 8), torch.zeros(4, 2, device=DEV)), "integers"),
        (lambda: kernels.mxfp4_experts_mm(x.float(), u8(2, 8, 2, 16), u8(2, 1, 1, 64, 8),
                                          torch.zeros(4, 2, dtype=torch.int64, device=DEV)), "dtype"),
        (lambda: quantized.mxfp4_operands(u8(2, 8, 2, 16), u8(2, 8, 2), 1), "blocks"),
        (lambda: quantized.mxfp4_experts_operands(u8(8, 2, 16), u8(8, 2), 1), "blocks"),
        (lambda: quantized.mxfp4_experts_linear(x, quantized.mxfp4_experts_operands(u8(2, 8, 2, 16), u8(2, 8, 2), 1),
                                                torch.zeros(5, 2, dtype=torch.int64, device=DEV)), "experts"),
    ]:
        with pytest.raises(LinnetError, match=message):
            call()


def test_workspace_is_checked() -> None:
    need = ctypes.c_int64(0)
    _lib.call("lnq_mxfp4_experts_workspace", 64, 16, 8, 64, ctypes.byref(need))
    with pytest.raises(LinnetError, match="workspace"):
        _lib.call("lnq_mxfp4_experts_mm", 4096, 64, *[4096] * 4, 16, 4, 8, 64, 64, 1, _lib.BF16, 4096, need.value - 1, None)


def _mixture(x: torch.Tensor, router: torch.Tensor, gate_up: tuple, down: tuple) -> torch.Tensor:
    """A mixture's layer as a program strings the calls together."""
    experts, weights = kernels.expert_route(x @ router, 2)
    h = quantized.mxfp4_experts_linear(x, gate_up, experts)
    g, u = h.chunk(2, dim=-1)
    h = (torch.nn.functional.silu(g.float()) * u.float()).to(x.dtype)
    y = quantized.mxfp4_experts_linear(h, down, experts)
    return (y.float() * weights[..., None]).sum(1).to(x.dtype)


def _mixture_case(rows: int):
    rng = np.random.default_rng(rows)
    hidden, inner, count = 96, 64, 6
    gate_up = _weight(rng, count, 2 * inner, hidden)
    down = _weight(rng, count, hidden, inner)
    x = torch.from_numpy(rng.standard_normal((rows, hidden)).astype(np.float32)).to(torch.bfloat16).to(DEV)
    router = torch.from_numpy(rng.standard_normal((hidden, count)).astype(np.float32)).to(torch.bfloat16).to(DEV)
    return x, router, gate_up, down


@pytest.mark.parametrize("rows", [1, 70])
def test_a_mixture_layer_end_to_end(rows: int) -> None:
    """Router, gate | up experts, SiLU, down experts and the weighted sum, against the same in f64
    from each stage's own inputs (so that a stage's rounding is not another's error)."""
    print(f"mixture rows={rows}", flush=True)
    x, router, gate_up, down = _mixture_case(rows)
    up_ops = quantized.mxfp4_experts_operands(*gate_up[:2], 1)
    down_ops = quantized.mxfp4_experts_operands(*down[:2], 1)
    got = _mixture(x, router, up_ops, down_ops)
    experts, weights = kernels.expert_route(x @ router, 2)
    logits = (x @ router).double()
    assert torch.equal(experts, torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :2])
    torch.testing.assert_close(weights.double(), torch.softmax(logits.gather(1, experts), -1), rtol=2e-7, atol=0)
    h = quantized.mxfp4_experts_linear(x, up_ops, experts)
    g, u = h.chunk(2, dim=-1)
    h = (torch.nn.functional.silu(g.float()) * u.float()).to(x.dtype)
    v = _rounded(h) if rows > 32 else h.double().cpu().numpy()
    ids = experts.cpu().numpy()
    pair = np.einsum("rki,rkoi->rko", v, down[2].astype(np.float64)[ids])
    terms = np.einsum("rki,rkoi->rko", np.abs(v), np.abs(down[2]).astype(np.float64)[ids])
    wk = weights.double().cpu().numpy()[..., None]
    want = (pair * wk).sum(1)
    # Each pair's product is rounded to bf16 (half a step of it and of its sum's error), the sum once more.
    bound = (wk * (2.0 ** -8 * np.abs(pair) + 64 * 2.0 ** -23 * terms)).sum(1) * 1.02 + 2.0 ** -8 * np.abs(want) * 1.02
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


def test_captured_and_replayed() -> None:
    """The layer's calls in a graph, replayed on new inputs with eager work between, against the
    eager calls; two graphs side by side keep their own workspaces."""
    graphs = []
    for rows in (70, 40):
        x, router, gate_up, down = _mixture_case(rows)
        ops = [quantized.mxfp4_experts_operands(*w[:2], 1) for w in (gate_up, down)]
        linear = quantized.mxfp4_operands(gate_up[0][0], gate_up[1][0], 1)

        def layer(x=x, router=router, ops=ops, linear=linear):
            return _mixture(x, router, *ops), quantized.mxfp4_linear(x, linear, None)

        layer()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer()
        graphs.append((graph, x, layer, out))
    for i in range(3):
        for graph, x, layer, out in graphs:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, layer, out in graphs:
            for got, want in zip(out, layer()):
                assert torch.equal(got, want)


def test_two_streams_at_once() -> None:
    cases = [_mixture_case(rows) for rows in (90, 50)]
    layers = [(c[0], c[1], *(quantized.mxfp4_experts_operands(*w[:2], 1) for w in c[2:])) for c in cases]
    want = [_mixture(*layer) for layer in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got: list[list[torch.Tensor]] = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(_mixture(*layers[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])
