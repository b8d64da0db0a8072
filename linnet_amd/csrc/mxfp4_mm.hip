// The MXFP4 x MXFP4 product on gfx950's block-scaled MFMA, y = x W^T (+ bias), and the same
// for the experts of a mixture: the (row, choice) pairs of each expert against its weight.
//
// Operands: codes [rows, K / 2] bytes, two E2M1 values each, a row's 32-value blocks in a
// row; scales as scale tiles (mx4.hpp; mxfp4_round.hip writes both so). The MFMA
// (v_mfma_scale_f32_32x32x64_f8f6f4, 131072 operations in 32 cycles) takes a lane's 32 codes and
// their scale byte and adds the exact products of 64 inputs in f32; the sum is rounded once,
// after the bias.
//
// A workgroup owns BM rows by BN columns, its waves WM x WN of them in 32 x 32 MFMA tiles.
// 256 inputs (128 bytes a row) a step: codes and scales move to LDS by buffer_load ... lds,
// S - 1 steps ahead, one barrier a step. The codes' 16-byte columns are XOR-swizzled by bits
// 1..3 of the row. A lane's scale dword of a row holds the unit's 4 bytes; shifted by 8 (lane
// / 32) once, bytes 0 and 2 are those of its halves of the unit's two MFMAs, named by the
// instruction's operand selects.
#include <algorithm>
#include <cstdlib>

#include "mx4.hpp"

namespace lnq {

namespace mx4 {
constexpr int LIST_THREADS = 1024;
}

template <int DT, int BM, int BN, int WM, int WN, int S, bool EXPERTS>
__global__ __launch_bounds__(64 * WM * WN, 1) void mx4_kernel(mx4::Args a) {
  using namespace mx4;
  using E = Elem<DT>;
  constexpr int NW = WM * WN, FA = BM / 32 / WM, FB = BN / 32 / WN;
  constexpr int CODES = (BM + BN) * BKB, STAGE = CODES + (BM + BN) * 8;
  constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;      // loads of a wave a step: 8 rows of codes each
  constexpr int LS = ((BM + BN) / 32 + NW - 1) / NW;     // and of 64 scale dwords each
  constexpr int LOADS = LA + LB + LS;
  static_assert(LA * 8 * NW == BM && LB * 8 * NW == BN && BM % 32 == 0 && BN % 32 == 0, "whole loads");
  static_assert(S >= 2 && S <= 4, "stages");
  // A stage array each (the compiler tracks loads into LDS by variable).
  __shared__ __attribute__((aligned(16))) uint8_t S0[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t S1[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t S2[S > 2 ? STAGE : 16];
  __shared__ __attribute__((aligned(16))) uint8_t S3[S > 3 ? STAGE : 16];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_n = (a.N + BN - 1) / BN;
  int m0 = 0, tn, live, first = 0;
  const uint8_t* w = a.w;
  const uint32_t* ws = a.ws;
  if constexpr (EXPERTS) {
    // Expert by expert, its tiles of rows together for each run of columns.
    const int at = xcd_tile(blockIdx.x, a.used[0] * tiles_n);
    if (at < 0) return;
    const i32x4 any = a.table[at / tiles_n];
    const int many = __builtin_amdgcn_readfirstlane(any.z) >> 9, tile0 = __builtin_amdgcn_readfirstlane(any.w);
    tn = (at - tile0 * tiles_n) / many;
    const i32x4 entry = a.table[tile0 + (at - tile0 * tiles_n) % many];
    const int e = __builtin_amdgcn_readfirstlane(entry.x);
    first = __builtin_amdgcn_readfirstlane(entry.y);
    live = __builtin_amdgcn_readfirstlane(entry.z) & 511;
    const int n0 = tn * BN;
    if (e >= a.count) {  // pairs whose choice is no expert: zeros
      const int width = min(BN, a.N - n0);
      for (int i = threadIdx.x; i < live * width; i += 64 * NW)
        a.y[static_cast<int64_t>(a.order[first + i / width]) * a.N + n0 + i % width] = 0;
      return;
    }
    w += e * a.w_step;
    ws += e * a.ws_step;
  } else {
    const int tiles_m = (a.M + BM - 1) / BM;
    int tm;
    mm8_tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    if (tm >= tiles_m || tn >= tiles_n) return;
    m0 = tm * BM;
    live = min(BM, a.M - m0);
  }
  const int n0 = tn * BN;
  const int steps = (a.K + BK - 1) / BK;
  const uint32_t row_bytes = static_cast<uint32_t>(a.K) >> 1;
  const int units = (a.K + 127) / 128;

  // Rows of x by place in the tile: the row, or -1 past the last.
  auto x_row = [&](int r) -> int {
    if (r >= live) return -1;
    if constexpr (EXPERTS) return a.order[first + r] / a.chosen;
    else return m0 + r;
  };
  // Load i of this wave: rows 8 (wave + NW i) .. + 7 of the tile, lane l row l / 8, stored
  // column l % 8 holding source column (l % 8) ^ key(row), key = bits 1..3 of the row (the
  // same for every i: NW is even).
  static_assert(NW % 2 == 0, "one key a wave");
  const int lrow8 = 8 * wave + (lane >> 3);
  const uint32_t lcol = static_cast<uint32_t>((lane & 7) ^ ((lrow8 >> 1) & 7)) * 16u;
  uint32_t aoff_g[LA], boff_g[LB], soff_g[LS];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int r = x_row(lrow8 + 8 * NW * i);
    aoff_g[i] = r < 0 ? NOWHERE : static_cast<uint32_t>(r - m0) * row_bytes + lcol;
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int n = lrow8 + 8 * NW * i;
    boff_g[i] = n0 + n < a.N ? static_cast<uint32_t>(n) * row_bytes + lcol : NOWHERE;
  }
  // Scale dword d of a stage: rows of x at the step's first unit, its second, columns of W
  // at the first, the second. Loads past the last repeat it.
  constexpr int XC = BM / 32, SC = (BM + BN) / 32;  // loads of x's scales, of all
#pragma unroll
  for (int i = 0; i < LS; ++i) {
    const int c = min(wave + NW * i, SC - 1);
    const bool is_x = c < XC;
    const int d = is_x ? c * 64 + lane : (c - XC) * 64 + lane;
    const int rows = is_x ? BM : BN, p = is_x ? a.xp : a.wp;
    const int unit = d / rows, r = d % rows;
    const int row = is_x ? x_row(r) : (n0 + r < a.N ? n0 + r : -1);
    soff_g[i] = row < 0 ? NOWHERE : (static_cast<uint32_t>(unit) * p + scale_place(row)) * 4u;
  }
  const uint8_t* const qb = EXPERTS ? a.q : a.q + static_cast<int64_t>(m0) * row_bytes;
  const uint32_t q_bytes = EXPERTS ? static_cast<uint32_t>(a.M) * row_bytes : static_cast<uint32_t>(live) * row_bytes;
  const uint8_t* const wb = w + static_cast<int64_t>(n0) * row_bytes;
  const uint32_t w_bytes = static_cast<uint32_t>(min(BN, a.N - n0)) * row_bytes;

  // Everything of step ks into stage st; a step past the end through descriptors of no
  // bytes. Columns past K in the last step, and its second unit where there is none, lie
  // nowhere.
  auto load = [&](int ks, uint8_t* st) {
    const bool in = ks < steps, last = ks == steps - 1;
    const uint32_t k0 = in ? static_cast<uint32_t>(ks) * BKB : 0u;
    const __amdgpu_buffer_rsrc_t ra = buffer_rsrc(qb + k0, in ? q_bytes - k0 : 0u);
    const __amdgpu_buffer_rsrc_t rb = buffer_rsrc(wb + k0, in ? w_bytes - k0 : 0u);
    const uint32_t past = last && k0 + lcol >= row_bytes ? NOWHERE : 0u;
#pragma unroll
    for (int i = 0; i < LA; ++i)
      load16(ra, st + (wave + NW * i) * 1024, aoff_g[i] | past);
#pragma unroll
    for (int i = 0; i < LB; ++i)
      load16(rb, st + BM * BKB + (wave + NW * i) * 1024, boff_g[i] | past);
    const uint32_t u0 = in ? static_cast<uint32_t>(ks) * 2u : 0u, left = in ? static_cast<uint32_t>(units) - u0 : 0u;
#pragma unroll
    for (int i = 0; i < LS; ++i) {
      const int c = min(wave + NW * i, SC - 1);
      const bool is_x = c < XC;
      const uint32_t p = static_cast<uint32_t>(is_x ? a.xp : a.wp);
      const uint32_t* const from = (is_x ? a.xs : ws) + static_cast<int64_t>(u0) * p;
      load4(buffer_rsrc(from, min(left, 2u) * p * 4u), st + CODES + c * 256, soff_g[i]);
    }
  };

  f32x16 acc[FA][FB];
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  const int lrow = lane & 31, lk = lane >> 5;
  uint32_t aoff[4], boff[4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const uint32_t col = static_cast<uint32_t>(((2 * kk + lk) ^ ((lrow >> 1) & 7)) << 4);
    aoff[kk] = static_cast<uint32_t>((wm * FA * 32 + lrow) * BKB) + col;
    boff[kk] = static_cast<uint32_t>(BM * BKB + (wn * FB * 32 + lrow) * BKB) + col;
  }
  const uint32_t sa_at = static_cast<uint32_t>(CODES + (wm * FA * 32 + lrow) * 4);
  const uint32_t sb_at = static_cast<uint32_t>(CODES + BM * 8 + (wn * FB * 32 + lrow) * 4);

  auto step = [&](int ks, const uint8_t* st, uint8_t* next) {
    // This wave's loads of step ks have landed (those of the S - 2 steps after it may be in
    // flight); past the barrier every wave's have, and every wave is done with step
    // ks - 1's stage, which step ks + S - 1 fills.
    wait_vm<(S - 2) * LOADS>();
    __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    load(ks + S - 1, next);
    __builtin_amdgcn_sched_barrier(0);
    int sa[FA][2], sb[FB][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < FA; ++i)
        sa[i][u] = static_cast<int>(*reinterpret_cast<const uint32_t*>(st + sa_at + u * BM * 4 + i * 128) >> (8 * lk));
#pragma unroll
      for (int j = 0; j < FB; ++j)
        sb[j][u] = static_cast<int>(*reinterpret_cast<const uint32_t*>(st + sb_at + u * BN * 4 + j * 128) >> (8 * lk));
    }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      i32x4 af[FA], bf[FB];
      auto fetch = [&](i32x4& o, uint32_t at) { o = *reinterpret_cast<const i32x4*>(st + at); };
#pragma unroll
      for (int i = 0; i < FA; ++i) fetch(af[i], aoff[kk] + i * 32 * BKB);
#pragma unroll
      for (int j = 0; j < FB; ++j) fetch(bf[j], boff[kk] + j * 32 * BKB);
#pragma unroll
      for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
          // The weight is the MFMA's A operand: a lane then holds 4 outputs of a row together.
          acc[i][j] = mma(kk & 1, bf[j], af[i], acc[i][j], sb[j][kk >> 1], sa[i][kk >> 1]);
    }
  };

  uint8_t* const st[4] = {S0, S1, S2, S3};
#pragma unroll
  for (int j = 0; j < S - 1; ++j) {
    load(j, st[j]);
    __builtin_amdgcn_sched_barrier(0);
  }
  for (int ks = 0; ks < steps; ks += S) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      if (ks + j >= steps) break;
      step(ks + j, st[j], st[(j + S - 1) % S]);
    }
  }
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // Lane l, register r of a tile: row m = l % 32, output feature 8 (r / 4) + 4 (l / 32) +
  // r % 4.
  const bool vec_out = (a.N & 3) == 0;
#pragma unroll
  for (int i = 0; i < FA; ++i) {
    const int m = (wm * FA + i) * 32 + lrow;
    if (m >= live) continue;
    int64_t row;
    if constexpr (EXPERTS) row = a.order[first + m];
    else row = m0 + m;
    uint16_t* const yrow = a.y + row * a.N;
#pragma unroll
    for (int j = 0; j < FB; ++j) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int n = n0 + (wn * FB + j) * 32 + 8 * q4 + 4 * lk;
        uint16_t out[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v = acc[i][j][4 * q4 + r];
          if (!EXPERTS && a.bias != nullptr) v += n + r < a.N ? E::to_f32(a.bias[n + r]) : 0.f;
          out[r] = E::from_f32(v);
        }
        if (vec_out && n + 3 < a.N) {
          *reinterpret_cast<u32x2*>(yrow + n) =
              u32x2{static_cast<uint32_t>(out[0]) | (static_cast<uint32_t>(out[1]) << 16),
                    static_cast<uint32_t>(out[2]) | (static_cast<uint32_t>(out[3]) << 16)};
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < a.N) yrow[n + r] = out[r];
        }
      }
    }
  }
}

// The pairs of each expert, in order: workgroup e counts every expert's pairs, which tells it
// where its own begin in `order` and in the tile table, then lists them. Workgroup `count`
// lists the pairs whose choice is no expert and writes how many tiles there are.
__global__ __launch_bounds__(mx4::LIST_THREADS) void expert_lists_kernel(const int64_t* __restrict__ experts, int pairs,
                                                                         int count, int bm,
                                                                         int* __restrict__ order, i32x4* __restrict__ table,
                                                                         int* __restrict__ used) {
  using namespace mx4;
  constexpr int WAVES = LIST_THREADS / 64;
  __shared__ int number[MAX_EXPERTS + 1];
  __shared__ int part[3][WAVES];
  __shared__ int found[WAVES];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto bucket = [&](int p) -> int {
    const int64_t id = experts[p];
    return id >= 0 && id < count ? static_cast<int>(id) : count;
  };
  for (int i = tid; i <= count; i += LIST_THREADS) number[i] = 0;
  __syncthreads();
  for (int p = tid; p < pairs; p += LIST_THREADS) atomicAdd(&number[bucket(p)], 1);
  __syncthreads();
  // Pairs and tiles of the experts before this one, and tiles of all.
  int sums[3] = {0, 0, 0};
  for (int i = tid; i <= count; i += LIST_THREADS) {
    const int n = number[i], t = (n + bm - 1) / bm;
    if (i < e) sums[0] += n, sums[1] += t;
    sums[2] += t;
  }
#pragma unroll
  for (int s = 0; s < 3; ++s) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sums[s] += __shfl_xor(sums[s], off, 64);
    if (lane == 0) part[s][wave] = sums[s];
  }
  __syncthreads();
  int first = 0, tile = 0, all = 0;
#pragma unroll
  for (int v = 0; v < WAVES; ++v) first += part[0][v], tile += part[1][v], all += part[2][v];
  const int mine = number[e];
  for (int i = tid; i * bm < mine; i += LIST_THREADS) 
    table[tile + i] = i32x4{e, first + i * bm, min(bm, mine - i * bm) + 512 * ((mine + bm - 1) / bm), tile};
  if (e == count && tid == 0) used[0] = all;
  if (mine == 0) return;
  int at = first;
  for (int p0 = 0; p0 < pairs; p0 += LIST_THREADS) {
    const int p = p0 + tid;
    const bool here = p < pairs && bucket(p) == e;
    const uint64_t mask = __ballot(here);
    if (lane == 0) found[wave] = __popcll(mask);
    __syncthreads();
    int to = at;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
      if (v < wave) to += found[v];
      at += found[v];
    }
    if (here) order[to + __popcll(mask & ((uint64_t{1} << lane) - 1))] = p;
    __syncthreads();
  }
}

namespace mx4 {

template <int DT, int BM, int BN, int WM, int WN, int S, bool EXPERTS>
static void launch_one(const Args& a, hipStream_t s) {
  const int64_t tiles_n = (a.N + BN - 1) / BN;
  const int64_t grid = tiles_n * (EXPERTS ? a.tiles : (a.M + BM - 1) / BM);
  hipLaunchKernelGGL((mx4_kernel<DT, BM, BN, WM, WN, S, EXPERTS>), dim3(static_cast<unsigned>(grid)), dim3(64 * WM * WN), 0, s, a);
}

// Rows of a tile.
static int tile_rows(double rows) { return rows > 64 ? 128 : rows > 32 ? 64 : 32; }

template <int DT, bool EXPERTS>
static void launch(const Args& a, int bm, hipStream_t s) {
  if (bm == 32) launch_one<DT, 32, 64, 1, 2, 4, EXPERTS>(a, s);
  else if (bm == 64) launch_one<DT, 64, 64, 2, 2, 4, EXPERTS>(a, s);
  else launch_one<DT, 128, 128, 2, 2, 2, EXPERTS>(a, s);
}

struct Plan {
  int bm, tiles;
  int64_t order_bytes, bytes;
};

// Tiles of the pairs at most: a partial one for each expert that is named.
static Plan experts_plan(int64_t pairs, int64_t count) {
  Plan p{};
  p.bm = tile_rows(static_cast<double>(pairs) / static_cast<double>(count));
  p.tiles = static_cast<int>(pairs / p.bm + std::min(pairs, count + 1));
  p.order_bytes = (pairs * 4 + 15) / 16 * 16;
  p.bytes = p.order_bytes + static_cast<int64_t>(p.tiles) * 16 + 16;
  return p;
}

}  // namespace mx4

}  // namespace lnq

using namespace lnq;

extern "C" {

LNQ_API LnqStatus lnq_mxfp4_mm(const uint8_t* q, const uint8_t* x_scale, const uint8_t* blocks, const uint8_t* tiles,
                               const void* bias, void* y, int64_t rows, int64_t out_features, int64_t in_features,
                               int32_t dtype, void* stream) {
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16, "lnq_mxfp4_mm: output is bf16 or f16, not dtype %d", dtype);
  LNQ_REQUIRE(rows >= 0 && out_features >= 0 && in_features > 0 && in_features % 32 == 0,
              "lnq_mxfp4_mm: bad shape rows=%lld out=%lld in=%lld (in %% 32 == 0)", static_cast<long long>(rows),
              static_cast<long long>(out_features), static_cast<long long>(in_features));
  LNQ_REQUIRE(rows <= (1 << 27) && out_features <= (1 << 27) && in_features <= (1 << 22),
              "lnq_mxfp4_mm: past 2^27 rows or outputs, or 2^22 inputs");
  if (rows == 0 || out_features == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(q && x_scale && blocks && tiles && y, "lnq_mxfp4_mm: null pointer");
  LNQ_REQUIRE(aligned(q, 16) && aligned(x_scale, 16) && aligned(blocks, 16) && aligned(tiles, 16) && aligned(y, 8),
              "lnq_mxfp4_mm: operands must be 16-byte aligned, y 8-byte");
  mx4::Args a{};
  a.q = q;
  a.xs = reinterpret_cast<const uint32_t*>(x_scale);
  a.w = blocks;
  a.ws = reinterpret_cast<const uint32_t*>(tiles);
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.M = static_cast<int>(rows);
  a.N = static_cast<int>(out_features);
  a.K = static_cast<int>(in_features);
  a.xp = mx4::padded_rows(a.M);
  a.wp = mx4::padded_rows(a.N);
  LNQ_REQUIRE((rows + 31) / 32 * ((out_features + 63) / 64) <= INT32_MAX, "lnq_mxfp4_mm: too large");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (getenv("MXL")) return mx4::launch_large(a, false, dtype, s);
  const int bm = mx4::tile_rows(static_cast<double>(rows));
  if (dtype == LNQ_BF16) mx4::launch<LNQ_BF16, false>(a, bm, s);
  else mx4::launch<LNQ_F16, false>(a, bm, s);
  return launched("mxfp4_mm");
}

LNQ_API LnqStatus lnq_mxfp4_experts_workspace(int64_t pairs, int64_t num_experts, int64_t* bytes) {
  LNQ_REQUIRE(bytes != nullptr, "lnq_mxfp4_experts_workspace: null pointer");
  LNQ_REQUIRE(pairs >= 0 && pairs <= (1 << 26) && num_experts > 0 && num_experts <= mx4::MAX_EXPERTS,
              "lnq_mxfp4_experts_workspace: %lld pairs of %lld experts (1 to %d)", static_cast<long long>(pairs),
              static_cast<long long>(num_experts), mx4::MAX_EXPERTS);
  *bytes = pairs == 0 ? 0 : mx4::experts_plan(pairs, num_experts).bytes;
  clear_error();
  return LNQ_OK;
}

LNQ_API LnqStatus lnq_mxfp4_experts_mm(const uint8_t* q, const uint8_t* x_scale, const uint8_t* blocks, const uint8_t* tiles,
                                       const int64_t* experts, void* y, int64_t rows, int64_t chosen, int64_t num_experts,
                                       int64_t out_features, int64_t in_features, int32_t shared, int32_t dtype,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16, "lnq_mxfp4_experts_mm: output is bf16 or f16, not dtype %d", dtype);
  LNQ_REQUIRE(rows >= 0 && chosen >= 0 && num_experts > 0 && num_experts <= mx4::MAX_EXPERTS && out_features >= 0 &&
                  in_features > 0 && in_features % 32 == 0,
              "lnq_mxfp4_experts_mm: bad shape rows=%lld chosen=%lld experts=%lld (1 to %d) out=%lld in=%lld (in %% 32 == 0)",
              static_cast<long long>(rows), static_cast<long long>(chosen), static_cast<long long>(num_experts),
              mx4::MAX_EXPERTS, static_cast<long long>(out_features), static_cast<long long>(in_features));
  LNQ_REQUIRE(rows <= (1 << 27) && chosen <= (1 << 27) && rows * chosen <= (1 << 26) && out_features <= (1 << 27) &&
                  in_features <= (1 << 22),
              "lnq_mxfp4_experts_mm: past 2^26 pairs, 2^27 outputs or 2^22 inputs");
  if (rows == 0 || chosen == 0 || out_features == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(q && x_scale && blocks && tiles && experts && y, "lnq_mxfp4_experts_mm: null pointer");
  LNQ_REQUIRE(aligned(q, 16) && aligned(x_scale, 16) && aligned(blocks, 16) && aligned(tiles, 16) && aligned(y, 8) &&
                  aligned(workspace, 16),
              "lnq_mxfp4_experts_mm: operands and workspace must be 16-byte aligned, y 8-byte");
  const int64_t pairs = rows * chosen, x_rows = shared ? rows : pairs;
  LNQ_REQUIRE(x_rows * (in_features / 2) < (int64_t{1} << 31), "lnq_mxfp4_experts_mm: x's codes past 2 GiB");
  const mx4::Plan plan = mx4::experts_plan(pairs, num_experts);
  LNQ_REQUIRE(workspace && workspace_bytes >= plan.bytes, "lnq_mxfp4_experts_mm: workspace of %lld bytes, %lld needed",
              static_cast<long long>(workspace_bytes), static_cast<long long>(plan.bytes));
  mx4::Args a{};
  a.q = q;
  a.xs = reinterpret_cast<const uint32_t*>(x_scale);
  a.w = blocks;
  a.ws = reinterpret_cast<const uint32_t*>(tiles);
  a.y = static_cast<uint16_t*>(y);
  a.M = static_cast<int>(x_rows);
  a.N = static_cast<int>(out_features);
  a.K = static_cast<int>(in_features);
  a.xp = mx4::padded_rows(a.M);
  a.wp = mx4::padded_rows(a.N);
  LNQ_REQUIRE(static_cast<int64_t>(plan.tiles) * ((out_features + 63) / 64) <= INT32_MAX,
              "lnq_mxfp4_experts_mm: too large");
  a.order = static_cast<const int*>(workspace);
  a.table = reinterpret_cast<const i32x4*>(static_cast<const uint8_t*>(workspace) + plan.order_bytes);
  a.used = reinterpret_cast<const int*>(a.table + plan.tiles);
  a.tiles = plan.tiles;
  a.count = static_cast<int>(num_experts);
  a.chosen = shared ? static_cast<int>(chosen) : 1;
  a.w_step = out_features * (in_features / 2);
  a.ws_step = (in_features + 127) / 128 * a.wp;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(expert_lists_kernel, dim3(a.count + 1), dim3(mx4::LIST_THREADS), 0, s, experts, static_cast<int>(pairs),
                     a.count, plan.bm, const_cast<int*>(a.order), const_cast<i32x4*>(a.table), const_cast<int*>(a.used));
  if (const LnqStatus st = launched("expert_lists")) return st;
  if (dtype == LNQ_BF16) mx4::launch<LNQ_BF16, true>(a, plan.bm, s);
  else mx4::launch<LNQ_F16, true>(a, plan.bm, s);
  return launched("mxfp4_experts_mm");
}

}  // extern "C"
