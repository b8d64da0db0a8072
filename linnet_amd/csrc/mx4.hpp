// The MXFP4 x MXFP4 product's operands (mxfp4_mm.hip), which mxfp4_round.hip lays out, its
// arguments and loads.
#pragma once

#include <utility>

#include "eight_bit.hpp"

namespace lnq {
namespace mx4 {

constexpr int BKB = 128;                   // bytes of a row a step
constexpr int BK = 2 * BKB;                // inputs a step
constexpr uint32_t NOWHERE = 0x80000000u;  // an offset past every buffer (each below 2 GiB): reads zeros
constexpr int MAX_EXPERTS = 2048;          // of the pair lists' LDS

// The MFMA (v_mfma_scale_f32_16x16x128_f8f6f4): lane l holds row l % 16, inputs 32 (l / 16) .. +
// 31 of 128 (a unit) in 16 bytes, and their scale in a byte, which the instruction selects, of a
// register. Scales lie so that the registers come as they are ("scale tiles"), x's by its rows and a
// weight's by its outputs: [pairs of units][blocks of 64 rows][64 lanes][2 units] dwords, lane l's for
// a unit holding the bytes of rows 16 f + l % 16 (f = 0 .. 3) of the block at block l / 16 of the
// unit: four MFMAs' scales. Rows and inputs past the last have 0.
__host__ __device__ inline int pairs_of(int K) { return (K + 255) / 256; }
__host__ __device__ inline int blocks_of(int N) { return (N + 63) / 64; }
constexpr int TILE_BYTES = 512;  // of a scale tile: 64 rows by 256 inputs

struct Args {
  const uint8_t* q;      // x's codes [rows, K / 2]
  const uint8_t* xs;     // and scale tiles, of the rows or of the experts' tiles' rows
  const uint8_t* w;      // codes [N, K / 2], of each expert
  const uint8_t* ws;     // scale tiles, of each expert
  const uint16_t* bias;
  uint16_t* y;
  int M, N, K;
  int x_blocks;          // of 64 rows, of x's scale tiles
  // Experts: the pairs by the places of their tiles, and the tiles: (expert, first place, pairs + 512 *
  // tiles of the expert, the expert's first tile); used[0]: the tiles there are.
  const int* order;
  const i32x4* table;
  const int* used;
  int tiles, count, chosen;  // tiles at most; pairs that share a row of x, 1 for none
  int64_t w_step, ws_step;   // from an expert's weight / scales to the next one's
};

// 16 bytes a lane from `at` of a buffer to LDS, lane l's at to + 16 l. (Called in a
// kernel template with arguments of known types the builtin makes the host's pass drop the
// kernel's stub without a word.)
__device__ inline void load16(__amdgpu_buffer_rsrc_t r, uint8_t* to, uint32_t at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)to, 16, at, 0, 0, 0);
}

// The MFMA of 32 codes a lane of a weight (a, scale byte F of sa) and of x (b, byte G of sb).
template <int F, int G>
__device__ inline f32x4 mma(i32x4 a, i32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 x = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 y = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, F, static_cast<int>(sa), G, static_cast<int>(sb));
}

// f(constant 0), .. f(constant N - 1).
template <class F, int... I>
__device__ __attribute__((always_inline)) inline void each_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// The b-th of `total` tiles as the XCDs take them (workgroups go to the 8 in turn): each a run
// of neighbours, or -1 past its run.
__device__ inline int xcd_tile(int b, int total) {
  const int xcd = b % mm8::XCDS, at = b / mm8::XCDS;
  const int each = total / mm8::XCDS, more = total % mm8::XCDS;
  if (at >= each + (xcd < more ? 1 : 0)) return -1;
  return xcd * each + min(xcd, more) + at;
}

}  // namespace mx4
}  // namespace lnq
