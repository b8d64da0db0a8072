// The MXFP4 x MXFP4 product in persistent 256 x 256 tiles (layouts: mxfp4_mm.hip).
//
// One workgroup a CU walks its tiles, and the k-steps of all of them form one stream: the
// loads of step g + 2, the next tile's near a tile's end, are issued while step g multiplies.
// 4 waves, one a SIMD, each 128 x 128 outputs (4 x 4 MFMA 32x32 tiles, 256 accumulator
// registers): per MFMA a wave reads half an operand. 256 inputs (128 bytes a row) a step in two
// stages of 68 KB, codes and scales; 16-byte columns XOR-swizzled by bits 1..3 of the row. Per
// step, a region per kk (64 inputs): 16 MFMAs on kk's operands while kk + 1's are read. One
// barrier, before the last kk: past it every wave's loads of step g + 1 have landed and no wave
// reads step g's stage again, so the last region reads step g + 1's first operands and scales
// and issues step g + 2's loads into step g's stage. A tile has an even number of steps (one
// past K loads nothing and adds zeros), so a step's stage is known at compile time.
#include "mx4.hpp"

namespace lnq {

namespace mx4l {
constexpr int BM = 256, BN = 256, NW = 4, THREADS = 64 * NW;
constexpr int FA = 4, FB = 4;
constexpr int CODES = (BM + BN) * mx4::BKB, STAGE = CODES + (BM + BN) * 8;
constexpr int LPW = (BM + BN) / 8 / NW;  // code loads of a wave a step, 8 rows each
}  // namespace mx4l

template <int DT>
__global__ __launch_bounds__(mx4l::THREADS, 1) void mx4_large_kernel(mx4::Args a) {
  using namespace mx4;
  using namespace mx4l;
  using E = Elem<DT>;
  // One array per stage: the compiler then waits, before reading a stage, for that stage's
  // loads only.
  __shared__ __attribute__((aligned(16))) uint8_t L0[STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t L1[STAGE];
  LNQ_MFMA_IN_AGPRS();

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN;
  const int total = tiles_m * tiles_n;
  const int G = gridDim.x;
  const int b0 = blockIdx.x;
  if (b0 >= total) return;
  const int mine = (total - 1 - b0) / G + 1;  // tiles b0, b0 + G, ..
  const int steps = (a.K + 2 * BK - 1) / (2 * BK) * 2;
  const int nsteps = mine * steps;
  const uint32_t row_bytes = static_cast<uint32_t>(a.K) >> 1;
  const int units = (a.K + 127) / 128;

  // Load i (0..15) of wave w fills stage rows 8 (4 i + w) .. + 7 (i < 8: A rows 32 i + 8 w +
  // l / 8 of the tile; else B rows 32 (i - 8) + 8 w + l / 8): lane l at byte 16 l of the 1 KB,
  // stored column l % 8 holding source column (l % 8) ^ key(row), key = (row >> 1) & 7, the
  // same for every i. Rows past the last lie past the buffer.
  const int lr = 8 * wave + (lane >> 3);
  const uint32_t lcol = 16u * ((lane & 7) ^ ((lr >> 1) & 7));
  uint32_t voff[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) voff[i] = static_cast<uint32_t>(lr + 32 * i) * row_bytes + lcol;

  // The tile whose steps are being loaded.
  const uint8_t *qb, *wb;
  uint32_t q_bytes, w_bytes;
  const uint32_t* sb0;  // this wave's scales: x's (waves 0, 1) or the weight's, unit wave % 2 of a step
  uint32_t s_bytes;
  const uint32_t sp = static_cast<uint32_t>(wave < 2 ? a.xp : a.wp);
  auto load_tile = [&](int r) {
    int tm, tn;
    mm8_tile_of(min(b0 + r * G, total - 1), tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    qb = a.q + static_cast<int64_t>(m0) * row_bytes;
    wb = a.w + static_cast<int64_t>(n0) * row_bytes;
    q_bytes = static_cast<uint32_t>(min(BM, a.M - m0)) * row_bytes;
    w_bytes = static_cast<uint32_t>(min(BN, a.N - n0)) * row_bytes;
    const int s0 = wave < 2 ? m0 : n0;
    sb0 = (wave < 2 ? a.xs : a.ws) + s0;
    s_bytes = (min(static_cast<uint32_t>(s0 + 256), sp) - static_cast<uint32_t>(s0)) * 4u;
  };
  // Load i of k-step ks into stage st (16: the scales). Steps past the stream, and columns and
  // units past K, read through 0-byte descriptors or past the buffer.
  auto load_one = [&](uint8_t* st, bool in, int ks, int i) __attribute__((always_inline)) {
    if (i < LPW) {
      const uint32_t k0 = static_cast<uint32_t>(ks) * BKB;
      const bool x = i < 8;
      const uint32_t bytes = x ? q_bytes : w_bytes;
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc((x ? qb : wb) + k0, in && k0 < row_bytes ? bytes - k0 : 0u);
      load16(r, st + (4 * i + wave) * 1024, voff[i & 7] | (k0 + lcol >= row_bytes ? NOWHERE : 0u));
    } else {
      const int u = 2 * ks + (wave & 1);
      const __amdgpu_buffer_rsrc_t r = buffer_rsrc(sb0 + static_cast<int64_t>(u) * sp, in && u < units ? s_bytes : 0u);
      load16(r, st + CODES + wave * 1024, lane * 16u);
    }
  };

  // Each tile's first step starts its accumulators with C = 0.
  f32x16 acc[FA][FB];

  const int lrow = lane & 31, lk = lane >> 5;
  uint32_t aoff[4], boff[4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    aoff[kk] = static_cast<uint32_t>(swz8(wm * 128 + lrow, 2 * kk + lk));
    boff[kk] = static_cast<uint32_t>(swz8(BM + wn * 128 + lrow, 2 * kk + lk));
  }
  // A lane's scale dwords of its 4 fragments lie together.
  const uint32_t sa_at = static_cast<uint32_t>(CODES + wm * 512 + lrow * 16);
  const uint32_t sb_at = static_cast<uint32_t>(CODES + 2048 + wn * 512 + lrow * 16);

  // Operand registers: set 0 holds even kk, set 1 odd kk. Scales of a unit as read, then shifted
  // for this lane's half of the unit's MFMAs.
  i32x4 af[2][FA], bf[2][FB];
  u32x4 sa[2], sb[2];
  // In the order that the next kk's MFMAs need them.
  auto read_one = [&](int set, const uint8_t* st, int kk, int r) __attribute__((always_inline)) {
    constexpr int ORDER[8] = {4, 0, 5, 6, 7, 1, 2, 3};
    const int f = ORDER[r];
    const i32x4 o = *reinterpret_cast<const i32x4*>(st + (f < FA ? aoff[kk] + f * 4096 : boff[kk] + (f - FA) * 4096));
    if (f < FA) af[set][f] = o;
    else bf[set][f - FA] = o;
  };
  auto read_scales = [&](const uint8_t* st, int u) __attribute__((always_inline)) {
    sa[u] = *reinterpret_cast<const u32x4*>(st + sa_at + u * 1024);
    sb[u] = *reinterpret_cast<const u32x4*>(st + sb_at + u * 1024);
  };
  auto take_scales = [&](int u) __attribute__((always_inline)) {
    sa[u] >>= 8 * lk;
    sb[u] >>= 8 * lk;
  };

  // One kk of step g on stage `cur`: 16 MFMA slots, the first 8 reading kk + 1's operands from
  // `cur`, or, in the last kk, step g + 1's first operands from `nxt`; there every slot
  // issues one of step g + 2's loads (k-step ks2, `ld2` whether inside the stream) into `cur`. A
  // unit's scales are read a kk before their use.
  auto region = [&](int kk, auto first_tag, const uint8_t* cur, const uint8_t* nxt, bool ld2,
                    int ks2) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first_tag)::value;  // a tile's first step
    const int set = kk & 1, u = kk >> 1;
    const bool last = kk == 3;
    if (!(kk & 1)) take_scales(u);
#pragma unroll
    for (int s = 0; s < 16; ++s) {
      const int i = s / FB, j = s % FB;
      const f32x16 c = FIRST && kk == 0 ? f32x16{} : acc[i][j];
      // The weight is the MFMA's A operand: a lane then holds 4 outputs of a row together.
      acc[i][j] = mma(kk & 1, bf[set][j], af[set][i], c, static_cast<int>(sb[u][j]), static_cast<int>(sa[u][i]));
      if (s < 8) read_one(set ^ 1, last ? nxt : cur, last ? 0 : kk + 1, s);
      if (s == 8 && kk == 1) read_scales(cur, 1);
      if (s == 8 && kk == 3) read_scales(nxt, 0);
      if (last) {
        load_one(const_cast<uint8_t*>(cur), ld2, ks2, s);
        if (s == 15) load_one(const_cast<uint8_t*>(cur), ld2, ks2, 16);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto step = [&](auto first_tag, const uint8_t* cur, const uint8_t* nxt, bool ld2, int ks2) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < 3; ++kk) region(kk, first_tag, cur, nxt, false, 0);
    wait_vm<0>();
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    region(3, first_tag, cur, nxt, ld2, ks2);
  };

  // Lane l, register r of fragment (i, j): row 128 wm + 32 i + l % 32 of the tile, column 128 wn +
  // 32 j + 8 (r / 4) + 4 (l / 32) + r % 4.
  const bool vec_out = (a.N & 3) == 0;
  auto epilogue = [&](int m0, int n0) {
#pragma unroll
    for (int j = 0; j < FB; ++j) {
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int n = n0 + wn * 128 + j * 32 + 8 * q4 + 4 * lk;
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.bias != nullptr) {
#pragma unroll
          for (int r = 0; r < 4; ++r) b[r] = n + r < a.N ? E::to_f32(a.bias[n + r]) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < FA; ++i) {
          const int m = m0 + wm * 128 + i * 32 + lrow;
          uint32_t o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = E::from_f32(acc[i][j][4 * q4 + r] + b[r]);
          if (m >= a.M) continue;
          uint16_t* const to = a.y + static_cast<int64_t>(m) * a.N + n;
          if (vec_out) {
            if (n < a.N) *reinterpret_cast<u32x2*>(to) = u32x2{o[0] | (o[1] << 16), o[2] | (o[3] << 16)};
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n + r < a.N) to[r] = static_cast<uint16_t>(o[r]);
          }
        }
      }
      // One column fragment at a time: the next tile's operands are live here.
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // Prologue: steps 0 and 1 requested; step 0 landed (this wave's, then every wave's); its
  // first operands and scales read.
  load_tile(0);
#pragma unroll
  for (int i = 0; i <= LPW; ++i) load_one(L0, true, 0, i);
#pragma unroll
  for (int i = 0; i <= LPW; ++i) load_one(L1, true, 1, i);
  wait_vm<LPW + 1>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int r = 0; r < FA + FB; ++r) read_one(0, L0, 0, r);
  read_scales(L0, 0);

  // Pairs of steps g, g + 1 of tile r at k-step ks on stages L0, L1: they issue steps g + 2, g +
  // 3, the next pair's (tile r, or r + 1 after a tile's last pair), with no branch inside.
  using T = std::integral_constant<bool, true>;
  using F = std::integral_constant<bool, false>;
  auto pair = [&](int g, int r, int ks, auto first_tag) __attribute__((always_inline)) {
    const bool ends = ks + 2 == steps;
    const int ks_n = ends ? 0 : ks + 2;
    if (ends) load_tile(r + 1);
    step(first_tag, L0, L1, g + 2 < nsteps, ks_n);
    step(F{}, L1, L0, g + 3 < nsteps, ks_n + 1);
  };
  int g = 0;
  for (int r = 0; r < mine; ++r) {
    pair(g, r, 0, T{});
    g += 2;
    for (int ks = 2; ks < steps; ks += 2, g += 2) pair(g, r, ks, F{});
    int tm, tn;
    mm8_tile_of(b0 + r * G, tiles_m, tiles_n, tm, tn);
    epilogue(tm * BM, tn * BN);
  }
  // Loads of the steps past the stream (0-byte reads) may be in flight.
  wait_vm<0>();
}

LnqStatus mx4::launch_large(const Args& a, bool, int dtype, hipStream_t s) {
  const int64_t total = static_cast<int64_t>((a.M + mx4l::BM - 1) / mx4l::BM) * ((a.N + mx4l::BN - 1) / mx4l::BN);
  const int cus = compute_units();
  const dim3 grid(static_cast<unsigned>(total < cus ? total : cus));
  if (dtype == LNQ_BF16) hipLaunchKernelGGL((mx4_large_kernel<LNQ_BF16>), grid, dim3(mx4l::THREADS), 0, s, a);
  else hipLaunchKernelGGL((mx4_large_kernel<LNQ_F16>), grid, dim3(mx4l::THREADS), 0, s, a);
  return launched("mxfp4_mm");
}

}  // namespace lnq
