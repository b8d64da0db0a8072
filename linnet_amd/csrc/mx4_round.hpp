// Rounding to MXFP4: a lane's values of a block, and rows of x laid out for the MXFP4 x MXFP4
// product (mx4.hpp), as mxfp4_round.hip and mxfp4_mm.hip share them.
#pragma once

#include "mx4.hpp"

namespace lnq {

namespace mxr {
constexpr int THREADS = 256;
constexpr int SPAN = 256;  // inputs of a block of threads that rounds rows: a line of codes

// 8 values as loaded.
template <int DT>
struct Raw {
  u32x4 v;
};
template <>
struct Raw<LNQ_F32> {
  f32x4 a, b;
};

template <int DT>
__device__ inline Raw<DT> load8(const typename Elem<DT>::storage* p) {
  Raw<DT> r;
  if constexpr (DT == LNQ_F32) {
    r.a = *reinterpret_cast<const f32x4*>(p);
    r.b = *reinterpret_cast<const f32x4*>(p + 4);
  } else {
    r.v = *reinterpret_cast<const u32x4*>(p);
  }
  return r;
}

template <int DT>
__device__ inline void widen8(const Raw<DT>& r, float (&v)[8]) {
  if constexpr (DT == LNQ_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = r.a[e], v[4 + e] = r.b[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t d = r.v[e];
      v[2 * e] = Elem<DT>::to_f32(static_cast<uint16_t>(d & 0xffffu));
      v[2 * e + 1] = Elem<DT>::to_f32(static_cast<uint16_t>(d >> 16));
    }
  }
}

// This lane's 8 values of a block whose other values the lanes of its quad (l & ~3 .. l | 3)
// hold: the scale byte (the same in all four) and the 8 codes, element 0 lowest.
__device__ inline uint32_t round8(const float (&v)[8], uint32_t& byte) {
  uint32_t top = 0;  // magnitudes order as their bits
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu);
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1, 64)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2, 64)));
  const uint32_t exponent = top >> 23;
  if (exponent == 255) {
    byte = 255;
    return 0;
  }
  byte = max(exponent, 2u) - 2u;
  const float inverse = __builtin_bit_cast(float, (254u - byte) << 23);  // 2^(127 - byte), byte <= 252
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0] * inverse, v[1] * inverse, 1.0f, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2] * inverse, v[3] * inverse, 1.0f, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4] * inverse, v[5] * inverse, 1.0f, 2);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6] * inverse, v[7] * inverse, 1.0f, 3);
  return word;
}

// 2^(byte - 127); 255 is NaN.
__device__ inline float scale_of(uint32_t byte) {
  const uint32_t bits = byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : byte << 23;
  return __builtin_bit_cast(float, bits);
}

// Rows for the product: codes [rows, K / 2], blocks in a row, and scale tiles. 256 threads (tid)
// take ROWS rows (from `bx` times that) by SPAN inputs (from `by` times that), 32 lanes a row, all of
// their loads before the first conversion; then their scales, one byte of each dword of a tile. (64 rows
// and whole dwords: 8192 x 8192 30.9 us against 28.6, level at 2048 rows.) `unit`: 2 ROWS dwords of LDS.
// Every thread of the workgroup calls it (one barrier), without `live` for nothing.
constexpr int PASSES = 2, ROWS = THREADS / 32 * PASSES;

template <int DT>
__device__ __attribute__((always_inline)) inline void round_rows(const typename Elem<DT>::storage* x, int64_t x_stride, uint32_t* codes,
                                                                 uint32_t* scales, int rows, int K, uint32_t* unit, int tid, int bx,
                                                                 int by, bool live) {
  constexpr int A_PASS = THREADS / 32;
  static_assert(ROWS == 16, "a byte of the scales' dwords");
  const int lane = tid & 63;
  const int r0 = bx * ROWS, k = by * SPAN + (tid & 31) * 8;
  const bool in = live && k < K;
  Raw<DT> raw[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = min(r0 + i * A_PASS + (tid >> 5), rows - 1);
    raw[i] = load8<DT>(x + r * x_stride + (in ? k : 0));
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = i * A_PASS + (tid >> 5);
    float v[8];
    widen8<DT>(raw[i], v);
    uint32_t byte;
    const uint32_t word = round8(v, byte);
    if (r0 + r < rows && in) codes[(static_cast<int64_t>(r0 + r) * K + k) >> 3] = word;
    // The four blocks of a unit, 16 lanes: block b's byte at bits 8 b.
    uint32_t four = in ? byte << (8 * ((lane >> 2) & 3)) : 0u;
    four |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(four), 4, 64));
    four |= static_cast<uint32_t>(__shfl_xor(static_cast<int>(four), 8, 64));
    if ((lane & 15) == 0) unit[2 * r + (lane >> 4 & 1)] = r0 + r < rows ? four : 0u;
  }
  __syncthreads();
  if (!live || tid >= 128) return;
  // Dword `tid` of the scale tile: place tid / 2 (row % 16, block of the unit), unit tid % 2.
  const int row = tid >> 1 & 15, u = tid & 1, shift = 8 * (tid >> 5);
  uint32_t* const at = scales + (static_cast<int64_t>(by) * mx4::blocks_of(rows) + r0 / 64) * (mx4::TILE_BYTES / 4) + tid;
  const int f = r0 % 64 / 16, last = r0 + ROWS >= rows ? 4 : f + 1;  // the last rows' threads write the tile's rest
  for (int i = f; i < last; ++i) reinterpret_cast<uint8_t*>(at)[i] = static_cast<uint8_t>(i == f ? unit[2 * row + u] >> shift : 0u);
}

inline int spans_of(int64_t K) { return static_cast<int>((K + SPAN - 1) / SPAN); }
}  // namespace mxr

}  // namespace lnq
