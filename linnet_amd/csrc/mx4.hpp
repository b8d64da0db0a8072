// What the MXFP4 x MXFP4 product's kernels share (mxfp4_mm.hip: small tiles; mxfp4_large.hip:
// the persistent 256 x 256 form): arguments, the experts' tiles and the loads into LDS.
#pragma once

#include "eight_bit.hpp"

namespace lnq {
namespace mx4 {

constexpr int BKB = 128;                   // bytes of a row a step
constexpr int BK = 2 * BKB;                // inputs a step
constexpr uint32_t NOWHERE = 0x80000000u;  // an offset past every buffer (each below 2 GiB): reads zeros
constexpr int MAX_EXPERTS = 2048;          // of the pair lists' LDS

// Scale tiles: a dword holds a row's four scale bytes of a unit (128 inputs); [units][rows
// rounded up to 128], the rows of each 128 dealt so that the 4 rows 32 apart that a lane of the
// large tiles meets (l, l + 32, l + 64, l + 96) are 16 bytes together.
__host__ __device__ inline int padded_rows(int rows) { return (rows + 127) / 128 * 128; }
__host__ __device__ inline int scale_place(int row) { return (row & ~127) + (row & 31) * 4 + ((row >> 5) & 3); }

struct Args {
  const uint8_t* q;      // x's codes [rows, K / 2]
  const uint32_t* xs;    // and scale tiles [units][xp]
  const uint8_t* w;      // codes [N, K / 2], of each expert
  const uint32_t* ws;    // scale tiles [units][wp], of each expert
  const uint16_t* bias;
  uint16_t* y;
  int M, N, K, xp, wp;
  // Experts: the pairs by expert, and tiles of them: (expert, first place in `order`, pairs + 512 *
  // tiles of the expert, the expert's first tile); used[0]: the tiles there are.
  const int* order;
  const i32x4* table;
  const int* used;
  int tiles, count, chosen;  // tiles at most; pairs that share a row of x, 1 for none
  int64_t w_step, ws_step;   // from an expert's weight / scales to the next one's
};

// 16 or 4 bytes a lane from `at` of a buffer to LDS, lane l's at to + 16 l (4 l). (Called in a
// kernel template with arguments of known types the builtin makes the host's pass drop the
// kernel's stub without a word.)
__device__ inline void load16(__amdgpu_buffer_rsrc_t r, uint8_t* to, uint32_t at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)to, 16, at, 0, 0, 0);
}

__device__ inline void load4(__amdgpu_buffer_rsrc_t r, uint8_t* to, uint32_t at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)to, 4, at, 0, 0, 0);
}

// The MFMA of two operands of 32 codes a lane; `odd`: their scales are byte 2 of sa and sb, byte 0
// otherwise.
__device__ inline f32x16 mma(bool odd, i32x4 a, i32x4 b, f32x16 c, int sa, int sb) {
  const i32x8 x = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 y = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return odd ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, 2, sa, 2, sb)
             : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, 4, 4, 0, sa, 0, sb);
}

// The b-th of `total` tiles as the XCDs take them (workgroups go to the 8 in turn): each a run
// of neighbours, or -1 past its run.
__device__ inline int xcd_tile(int b, int total) {
  const int xcd = b % mm8::XCDS, at = b / mm8::XCDS;
  const int each = total / mm8::XCDS, more = total % mm8::XCDS;
  if (at >= each + (xcd < more ? 1 : 0)) return -1;
  return xcd * each + min(xcd, more) + at;
}

// mxfp4_large.hip. `experts`: the launch's tiles are of 256 pairs.
LnqStatus launch_large(const Args& a, bool experts, int dtype, hipStream_t s);

}  // namespace mx4
}  // namespace lnq
