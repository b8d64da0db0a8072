// Rounding to MXFP4 (OCP microscaling: 32 values share an E8M0 scale, E2M1 elements) and
// back, and the scale layout of the MXFP4 x MXFP4 product (mxfp4_mm.hip).
//
// A block of 32 values with largest magnitude m: the scale byte is s = floor(log2 m) - 2 +
// 127 (E2M1's largest exponent is 2), at least 0, and each value is x / 2^(s - 127) rounded
// to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, ties to the even code,
// past 6 to 6. floor(log2 m) is m's f32 exponent field; the division by a power of two is
// exact in f32, so the one rounding is the conversion's (v_cvt_scalef32_pk_fp4_f32 with a
// scale of 1). A block that holds an infinity or a NaN gets s = 255, E8M0's NaN, and codes
// of 0: every reader of it gives NaN.
//
// Bound by HBM: 2 or 4 bytes a value read, 17/32 written (back: the reverse). Four lanes
// take a block, 8 values each: a wave's loads are whole kilobytes. 8192 x 14336 bf16: 50 us each
// way, 5.9 TB/s; as rows of the product, 4096 x 8192: 16.6 us, 5.1 TB/s (half
// a line of codes a workgroup and a row, the other half written from another XCD: 24.7).
#include "mx4_round.hpp"

namespace lnq {

// Blocks one after another, as a checkpoint stores them: thread i of the grid takes values
// 8 i .. 8 i + 7 of all.
template <int DT>
__global__ __launch_bounds__(mxr::THREADS) void mxfp4_quantize_kernel(const typename Elem<DT>::storage* __restrict__ x,
                                                                      uint32_t* __restrict__ codes,
                                                                      uint8_t* __restrict__ scales, int64_t eights) {
  using namespace mxr;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  if (i >= eights) return;  // eights % 4 == 0: whole quads
  float v[8];
  widen8<DT>(load8<DT>(x + i * 8), v);
  uint32_t byte;
  codes[i] = round8(v, byte);
  if ((threadIdx.x & 3) == 0) scales[i >> 2] = static_cast<uint8_t>(byte);
}

// Rows for the product, ROWS by SPAN inputs a workgroup, those of a row together.
template <int DT>
__global__ __launch_bounds__(mxr::THREADS) void mxfp4_rows_kernel(const typename Elem<DT>::storage* __restrict__ x,
                                                                  int64_t x_stride, uint32_t* __restrict__ codes,
                                                                  uint32_t* __restrict__ scales, int rows, int K, int spans) {
  __shared__ uint32_t unit[2 * mxr::ROWS];
  mxr::round_rows<DT>(x, x_stride, codes, scales, rows, K, unit, threadIdx.x, blockIdx.x / spans, blockIdx.x % spans, true);
}

template <int DT>
__global__ __launch_bounds__(mxr::THREADS) void mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                                        const uint8_t* __restrict__ scales,
                                                                        typename Elem<DT>::storage* __restrict__ out,
                                                                        int64_t eights) {
  using namespace mxr;
  using E = Elem<DT>;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  if (i >= eights) return;
  const uint32_t w = codes[i];
  const float s = scale_of(scales[i >> 2]);
  const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3)};
  if constexpr (DT == LNQ_F32) {
    *reinterpret_cast<f32x4*>(out + i * 8) = f32x4{p[0][0] * s, p[0][1] * s, p[1][0] * s, p[1][1] * s};
    *reinterpret_cast<f32x4*>(out + i * 8 + 4) = f32x4{p[2][0] * s, p[2][1] * s, p[3][0] * s, p[3][1] * s};
  } else {
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = static_cast<uint32_t>(E::from_f32(p[e][0] * s)) | (static_cast<uint32_t>(E::from_f32(p[e][1] * s)) << 16);
    *reinterpret_cast<u32x4*>(out + i * 8) = o;
  }
}

// Scales as stored, [count, N, groups], as scale tiles (mx4.hpp), a workgroup two tiles.
__global__ __launch_bounds__(mxr::THREADS) void mxfp4_scale_tiles_kernel(const uint8_t* __restrict__ scales,
                                                                         uint32_t* __restrict__ tiles, int N, int groups) {
  const int block = blockIdx.x * 2 + (threadIdx.x >> 7), blocks = mx4::blocks_of(N);
  if (block >= blocks) return;
  const int lane = (threadIdx.x >> 1) & 63, u = threadIdx.x & 1;
  const int g = (2 * blockIdx.y + u) * 4 + (lane >> 4);
  uint32_t word = 0;
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    const int n = block * 64 + 16 * f + (lane & 15);
    if (n < N && g < groups)
      word |= static_cast<uint32_t>(scales[(static_cast<int64_t>(blockIdx.z) * N + n) * groups + g]) << (8 * f);
  }
  const int64_t tile = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * blocks + block;
  tiles[tile * (mx4::TILE_BYTES / 4) + (threadIdx.x & 127)] = word;
}

}  // namespace lnq

using namespace lnq;

namespace {

LnqStatus check_rounding(const char* what, int64_t rows, int64_t in_features, int32_t dtype) {
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16 || dtype == LNQ_F32, "%s: dtype %d is not bf16, f16 or f32", what, dtype);
  LNQ_REQUIRE(rows >= 0 && in_features >= 0 && in_features % 32 == 0, "%s: bad shape rows=%lld in=%lld (in %% 32 == 0)", what,
              static_cast<long long>(rows), static_cast<long long>(in_features));
  LNQ_REQUIRE(in_features <= INT32_MAX && rows <= INT32_MAX - 128, "%s: sizes exceed 2^31", what);
  return LNQ_OK;
}

}  // namespace

extern "C" {

LNQ_API LnqStatus lnq_mxfp4_quantize(const void* x, uint8_t* blocks, uint8_t* scales, int64_t rows, int64_t in_features,
                                     int32_t dtype, void* stream) {
  if (const LnqStatus st = check_rounding("lnq_mxfp4_quantize", rows, in_features, dtype)) return st;
  if (rows == 0 || in_features == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(x && blocks && scales, "lnq_mxfp4_quantize: null pointer");
  LNQ_REQUIRE(aligned(x, 16) && aligned(blocks, 16), "lnq_mxfp4_quantize: x and blocks must be 16-byte aligned");
  const int64_t eights = rows * (in_features / 8), grid = (eights + mxr::THREADS - 1) / mxr::THREADS;
  LNQ_REQUIRE(grid <= INT32_MAX, "lnq_mxfp4_quantize: too large");
#define LNQ_MXQ(DT)                                                                                          \
  hipLaunchKernelGGL((mxfp4_quantize_kernel<DT>), dim3(static_cast<unsigned>(grid)), dim3(mxr::THREADS), 0,  \
                     static_cast<hipStream_t>(stream), static_cast<const typename Elem<DT>::storage*>(x),    \
                     reinterpret_cast<uint32_t*>(blocks), scales, eights)
  if (dtype == LNQ_BF16) LNQ_MXQ(LNQ_BF16);
  else if (dtype == LNQ_F16) LNQ_MXQ(LNQ_F16);
  else LNQ_MXQ(LNQ_F32);
#undef LNQ_MXQ
  return launched("mxfp4_quantize");
}

LNQ_API LnqStatus lnq_mxfp4_dequantize(const uint8_t* blocks, const uint8_t* scales, void* out, int64_t rows,
                                       int64_t in_features, int32_t dtype, void* stream) {
  if (const LnqStatus st = check_rounding("lnq_mxfp4_dequantize", rows, in_features, dtype)) return st;
  if (rows == 0 || in_features == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(blocks && scales && out, "lnq_mxfp4_dequantize: null pointer");
  LNQ_REQUIRE(aligned(blocks, 16) && aligned(out, 16), "lnq_mxfp4_dequantize: blocks and out must be 16-byte aligned");
  const int64_t eights = rows * (in_features / 8), grid = (eights + mxr::THREADS - 1) / mxr::THREADS;
  LNQ_REQUIRE(grid <= INT32_MAX, "lnq_mxfp4_dequantize: too large");
#define LNQ_MXD(DT)                                                                                           \
  hipLaunchKernelGGL((mxfp4_dequantize_kernel<DT>), dim3(static_cast<unsigned>(grid)), dim3(mxr::THREADS), 0, \
                     static_cast<hipStream_t>(stream), reinterpret_cast<const uint32_t*>(blocks), scales,     \
                     static_cast<typename Elem<DT>::storage*>(out), eights)
  if (dtype == LNQ_BF16) LNQ_MXD(LNQ_BF16);
  else if (dtype == LNQ_F16) LNQ_MXD(LNQ_F16);
  else LNQ_MXD(LNQ_F32);
#undef LNQ_MXD
  return launched("mxfp4_dequantize");
}

LNQ_API LnqStatus lnq_mxfp4_rows(const void* x, int64_t x_stride, uint8_t* q, uint8_t* scales, int64_t rows,
                                 int64_t in_features, int32_t dtype, void* stream) {
  if (const LnqStatus st = check_rounding("lnq_mxfp4_rows", rows, in_features, dtype)) return st;
  if (rows == 0 || in_features == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(x && q && scales, "lnq_mxfp4_rows: null pointer");
  LNQ_REQUIRE(x_stride >= 0 && x_stride % 8 == 0 && aligned(x, 16) && aligned(q, 16) && aligned(scales, 16),
              "lnq_mxfp4_rows: x (with its row stride), q and scales must be 16-byte aligned");
  const int spans = mxr::spans_of(in_features);
  const int64_t grid = (rows + mxr::ROWS - 1) / mxr::ROWS * spans;
  LNQ_REQUIRE(in_features <= (1 << 22) && grid <= INT32_MAX, "lnq_mxfp4_rows: too large (in past 2^22)");
  const int R = static_cast<int>(rows), K = static_cast<int>(in_features);
#define LNQ_MXW(DT)                                                                                                         \
  hipLaunchKernelGGL((mxfp4_rows_kernel<DT>), dim3(static_cast<unsigned>(grid)), dim3(mxr::THREADS), 0,                    \
                     static_cast<hipStream_t>(stream), static_cast<const typename Elem<DT>::storage*>(x), x_stride,        \
                     reinterpret_cast<uint32_t*>(q), reinterpret_cast<uint32_t*>(scales), R, K, spans)
  if (dtype == LNQ_BF16) LNQ_MXW(LNQ_BF16);
  else if (dtype == LNQ_F16) LNQ_MXW(LNQ_F16);
  else LNQ_MXW(LNQ_F32);
#undef LNQ_MXW
  return launched("mxfp4_rows");
}

LNQ_API LnqStatus lnq_mxfp4_scale_tiles(const uint8_t* scales, uint8_t* tiles, int64_t count, int64_t out_features,
                                        int64_t in_features, void* stream) {
  LNQ_REQUIRE(count >= 0 && out_features >= 0 && in_features >= 0 && in_features % 32 == 0,
              "lnq_mxfp4_scale_tiles: bad shape count=%lld out=%lld in=%lld (in %% 32 == 0)", static_cast<long long>(count),
              static_cast<long long>(out_features), static_cast<long long>(in_features));
  if (count == 0 || out_features == 0 || in_features == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(scales && tiles, "lnq_mxfp4_scale_tiles: null pointer");
  LNQ_REQUIRE(aligned(tiles, 16), "lnq_mxfp4_scale_tiles: tiles must be 16-byte aligned");
  LNQ_REQUIRE(count <= 65535 && in_features <= 256 * 65535 && out_features <= INT32_MAX - 128, "lnq_mxfp4_scale_tiles: too large");
  const int N = static_cast<int>(out_features), K = static_cast<int>(in_features);
  const dim3 grid(static_cast<unsigned>((mx4::blocks_of(N) + 1) / 2), static_cast<unsigned>(mx4::pairs_of(K)),
                  static_cast<unsigned>(count));
  hipLaunchKernelGGL(mxfp4_scale_tiles_kernel, grid, dim3(mxr::THREADS), 0, static_cast<hipStream_t>(stream), scales,
                     reinterpret_cast<uint32_t*>(tiles), N, K / 32);
  return launched("mxfp4_scale_tiles");
}

}  // extern "C"
