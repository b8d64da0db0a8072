// The MXFP4 linear layer at few rows, y = x W^T (+ bias) with x in 16 bits: the streaming
// product (stream.hpp) over codes and E8M0 scales as a checkpoint stores them. 16 rows, 4096 ->
// 14336: 13.0 us, 2.4 TB/s.
#include "stream.hpp"

using namespace lnq;

extern "C" {

LNQ_API LnqStatus lnq_mxfp4_linear(const void* x, int64_t x_stride, const uint8_t* blocks, const uint8_t* scales,
                                   const void* bias, void* y, int64_t rows, int64_t out_features, int64_t in_features,
                                   int32_t dtype, void* stream) {
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16, "lnq_mxfp4_linear: x is bf16 or f16, not dtype %d", dtype);
  LNQ_REQUIRE(rows >= 0 && out_features >= 0 && in_features > 0 && in_features % 32 == 0,
              "lnq_mxfp4_linear: bad shape rows=%lld out=%lld in=%lld (in %% 32 == 0)", static_cast<long long>(rows),
              static_cast<long long>(out_features), static_cast<long long>(in_features));
  LNQ_REQUIRE(in_features <= stream::MAX_K && out_features <= stream::MAX_N && rows <= 65535,
              "lnq_mxfp4_linear: rows=%lld out=%lld in=%lld past 65535 rows, %d outputs or %d inputs",
              static_cast<long long>(rows), static_cast<long long>(out_features), static_cast<long long>(in_features),
              stream::MAX_N, stream::MAX_K);
  if (rows == 0 || out_features == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(x && blocks && scales && y, "lnq_mxfp4_linear: null pointer");
  LNQ_REQUIRE(x_stride % 8 == 0 && x_stride >= in_features && x_stride < (int64_t{1} << 23) && aligned(x, 16) && aligned(blocks, 16),
              "lnq_mxfp4_linear: x (rows of at least in and less than 2^23 elements) and blocks must be 16-byte aligned");
  stream::Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.w = blocks;
  a.scale = scales;
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.x_stride = static_cast<int>(x_stride);
  a.y_stride = static_cast<int>(out_features);
  a.row_bytes = static_cast<int>(in_features / 2);
  a.M = static_cast<int>(rows);
  a.N = static_cast<int>(out_features);
  a.K = static_cast<int>(in_features);
  a.span = 1;
  a.cols = static_cast<int>(in_features / 32);
  a.row_block = 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == LNQ_BF16) stream::launch<LNQ_BF16, stream::FP4, 4>(a, s);
  else stream::launch<LNQ_F16, stream::FP4, 4>(a, s);
  return launched("mxfp4_linear");
}

}  // extern "C"
