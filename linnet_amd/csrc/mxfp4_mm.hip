// The MXFP4 x MXFP4 product on gfx950's block-scaled MFMA, y = x W^T (+ bias), and the same
// for the experts of a mixture: the (row, choice) pairs of each expert against its weight.
//
// Operands: codes [rows, K / 2] bytes, two E2M1 values each, a row's 32-value blocks in a row;
// scales laid out for the MFMA (mx4.hpp; mxfp4_round.hip writes both so), which adds the exact
// products of 128 inputs in f32 (65536 operations in 16 cycles). The sum is rounded once, after
// the bias. (The 32x32x64 form does as much a cycle, but at the clock that the power allows
// random codes run at 7.6 PFLOP/s on this one and 5.6 on that, registers alone: it reads and
// writes half the accumulators.)
//
// A workgroup owns BM rows by BN columns of y, its waves WM x WN of them, FA x FB MFMA tiles
// each, and walks its tiles of the launch; the k-steps of all of them form one stream. 256 inputs
// (128 bytes a row) a step: codes and scales move to LDS by buffer_load ... lds, the codes' 16-byte
// columns XOR-swizzled by bits 1..3 of the row, into two stages. Per step, a region a unit (128
// inputs): FA x FB MFMAs on the unit's operands while the next ones are read. One barrier, inside
// the second: past it every wave's loads of step g + 1 have landed and no wave reads step g's stage
// again, so the rest reads step g + 1's first operands and issues step g + 2's loads, the next
// tile's near a tile's end, into step g's stage.
//
// Bound by the power that MFMAs, LDS and loads share (a 4096 x 8192 -> 28672 call: 425 to 455 us by
// the card and its warmth, 4.2 to 4.5 PFLOP/s at 1.75 GHz; its MFMAs alone 213, its loads alone 218, all but
// the stores 390), with few tiles by a step's latency (0.4 us of 64-row tiles, 0.6 of 128), with few
// rows by HBM (32 experts of 2880 -> 5760: 59 us, 4.7 TB/s).
//
// Experts: tiles of BM pairs of one expert, expert by expert with its tiles of rows together for
// each run of columns; where the next tiles lie is looked up a tile ahead a lookup.
#include <algorithm>
#include <cmath>

#include "mx4_round.hpp"

namespace lnq {

namespace mx4 {
constexpr int LIST_THREADS = 1024;

template <int WM, int WN, int FA_, int FB_>
struct Form {
  static constexpr int FA = FA_, FB = FB_, BLOCKS = FA_ * WM / 4 > 0 ? FA_ * WM / 4 : 1;  // blocks of 64 rows
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int BM = 16 * FA * WM, BN = 16 * FB * WN;
  static constexpr int CODES = (BM + BN) * BKB;
  static constexpr int XC = (BLOCKS + 1) / 2, ALL = XC + (BN + 127) / 128;  // loads of a step's scales: x's, all
  static constexpr int STAGE = CODES + ALL * 1024;         // the codes, x's scales of the 2 units, the weight's
  static constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;  // loads of a wave a step: 8 rows of codes each
  static constexpr int LOADS = LA + LB + 1;                // and of scales
  static constexpr int GROUPS = 160 * 1024 / (2 * STAGE);  // workgroups that a CU's LDS holds
  static constexpr int PER_CU = GROUPS < 4 ? GROUPS : 4;
  static constexpr int WAVES_A_SIMD = NW * PER_CU / 4 > 0 ? NW * PER_CU / 4 : 1;
  static_assert(LA * 8 * NW == BM && LB * 8 * NW == BN && NW % 2 == 0, "whole loads, one key a wave");
  static_assert((FB == 2 || FB == 4) && BN % 64 == 0 && (FA == 2 || FA == 4 || FA == 8) && ALL <= NW, "scales a lane");
};
}  // namespace mx4

template <int DT, class FORM, bool EXPERTS>
__global__ __launch_bounds__(FORM::THREADS, FORM::WAVES_A_SIMD) void mx4_kernel(mx4::Args a) {
  using namespace mx4;
  using E = Elem<DT>;
  constexpr int FA = FORM::FA, FB = FORM::FB, NW = FORM::NW, BM = FORM::BM, BN = FORM::BN, CODES = FORM::CODES;
  constexpr int LA = FORM::LA, LB = FORM::LB, LOADS = FORM::LOADS, XC = FORM::XC, BLOCKS = FORM::BLOCKS;
  constexpr int WN = BN / 16 / FB;
  // One array per stage: the compiler then waits, before reading a stage, for that stage's
  // loads only.
  __shared__ __attribute__((aligned(16))) uint8_t L0[FORM::STAGE];
  __shared__ __attribute__((aligned(16))) uint8_t L1[FORM::STAGE];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN;
  const int total = EXPERTS ? a.used[0] * tiles_n : tiles_m * tiles_n;
  const int G = gridDim.x, b0 = blockIdx.x;
  // Tiles b0, b0 + G, .. of the XCDs' order.
  int mine = 0;
  if constexpr (EXPERTS) {
    // G is a multiple of the XCDs: a run of an XCD in turn.
    const int xcd = b0 % mm8::XCDS, run = total / mm8::XCDS + (xcd < total % mm8::XCDS ? 1 : 0);
    const int at = b0 / mm8::XCDS, every = G / mm8::XCDS;
    mine = at < run ? (run - 1 - at) / every + 1 : 0;
  } else {
    mine = b0 < total ? (total - 1 - b0) / G + 1 : 0;
  }
  if (mine == 0) return;
  const int steps = (a.K + 2 * BK - 1) / (2 * BK) * 2;  // a step past K adds zeros
  const int nsteps = mine * steps;
  const uint32_t row_bytes = static_cast<uint32_t>(a.K) >> 1;

  // Load i of wave w fills stage rows 8 (NW i + w) .. + 7 (i < LA: rows of x; then columns): lane l
  // row l / 8 at byte 16 l of the 1 KB, stored column l % 8 holding source column (l % 8) ^
  // key(row), key = (row >> 1) & 7, the same for every i. Rows past the last lie nowhere.
  const int lr = 8 * wave + (lane >> 3);
  const uint32_t lcol = 16u * ((lane & 7) ^ ((lr >> 1) & 7));
  // This wave's load of scales, a kilobyte: two tiles of x's rows or of columns (waves past the last
  // load what others do). soff: nowhere past what a step has.
  const int chunk = wave % FORM::ALL;
  const bool x_chunk = chunk < XC;
  const uint32_t scale_at = static_cast<uint32_t>(x_chunk ? chunk : chunk - XC) * 1024 + lane * 16;
  const uint32_t soff = scale_at < static_cast<uint32_t>((x_chunk ? BLOCKS : BN / 64) * TILE_BYTES) ? scale_at : NOWHERE;
  const uint32_t s_step = static_cast<uint32_t>(x_chunk ? a.x_blocks : blocks_of(a.N)) * TILE_BYTES;

  // A tile of this launch: columns from n0; rows from m0, or an expert's pairs from `first` (their
  // scales as rows from m0).
  struct Tile {
    int n0, m0, live, first, e;
  };
  auto plain_tile = [&](int r) -> Tile {
    int tm, tn;
    mm8_tile_of(b0 + r * G, tiles_m, tiles_n, tm, tn);
    return Tile{tn * BN, tm * BM, min(BM, a.M - tm * BM), 0, 0};
  };
  // The experts' tile r in two lookups: the entry of some tile of its expert, then its own.
  auto place_of = [&](int r) -> int { return max(xcd_tile(b0 + min(r, mine - 1) * G, total), 0); };
  auto expert_of = [&](int r) -> i32x4 { return a.table[place_of(r) / tiles_n]; };
  auto entry_of = [&](int r, i32x4 any, int& n0, int& m0) -> i32x4 {
    const int many = __builtin_amdgcn_readfirstlane(any.z) >> 9, tile0 = __builtin_amdgcn_readfirstlane(any.w);
    const int j = place_of(r) - tile0 * tiles_n;
    n0 = j / many * BN;
    m0 = (tile0 + j % many) * (BLOCKS * 64);
    return a.table[tile0 + j % many];
  };
  auto expert_tile = [&](i32x4 entry, int n0, int m0) -> Tile {
    return Tile{n0, m0, __builtin_amdgcn_readfirstlane(entry.z) & 511, __builtin_amdgcn_readfirstlane(entry.y),
                __builtin_amdgcn_readfirstlane(entry.x)};
  };
  // The pairs whose rows of x this thread loads of an experts' tile.
  int pairs[EXPERTS ? LA : 1];
  auto take_pairs = [&](const Tile& t) {
    if constexpr (EXPERTS) {
#pragma unroll
      for (int i = 0; i < LA; ++i) pairs[i] = a.order[t.first + min(lr + 8 * NW * i, t.live - 1)];
    }
  };

  // The tile whose steps are being loaded: where this wave's rows lie from the bases, and the bytes
  // from there. (Chosen here: a choice in the steps would be a branch, and the compiler then moves the
  // MFMAs across the blocks it splits the step into.)
  const uint8_t *qb, *wb, *sb;
  uint32_t q_bytes, w_bytes, s_bytes, xoff[LA], woff[LB];
  auto load_tile = [&](const Tile& t) {
    const int e = EXPERTS ? min(t.e, a.count - 1) : 0;  // a tile of no expert multiplies the last one's weight, for nothing
    qb = a.q + (EXPERTS ? 0 : static_cast<int64_t>(t.m0) * row_bytes);
    q_bytes = static_cast<uint32_t>(EXPERTS ? a.M : t.live) * row_bytes;
    wb = a.w + e * a.w_step + static_cast<int64_t>(t.n0) * row_bytes;
    const int outs = min(BN, a.N - t.n0);
    w_bytes = static_cast<uint32_t>(outs) * row_bytes;
    const uint32_t from = static_cast<uint32_t>(x_chunk ? t.m0 : t.n0) / 64 * TILE_BYTES;
    sb = (x_chunk ? a.xs : a.ws + e * a.ws_step) + from;
    s_bytes = s_step - from;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int r = lr + 8 * NW * i;
      xoff[i] = r < t.live ? static_cast<uint32_t>(EXPERTS ? pairs[EXPERTS ? i : 0] / a.chosen : r) * row_bytes + lcol : NOWHERE;
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const int r = lr + 8 * NW * i;
      woff[i] = r < outs ? static_cast<uint32_t>(r) * row_bytes + lcol : NOWHERE;
    }
  };
  // The sources of a k-step's loads; steps past the stream or past K read through 0-byte ones. The
  // last step of a row may end inside a line: x's bytes past it are left out, the weight's then
  // multiply zeros (every code is finite, and scales past K are 0).
  struct Source {
    __amdgpu_buffer_rsrc_t q, w, s;
    uint32_t past;
  };
  auto source_of = [&](bool in, int ks) __attribute__((always_inline)) -> Source {
    const uint32_t k0 = static_cast<uint32_t>(ks) * BKB;
    const bool live = in && k0 < row_bytes;
    return Source{buffer_rsrc(qb + k0, live ? q_bytes - k0 : 0u), buffer_rsrc(wb + k0, live ? w_bytes - k0 : 0u),
                  buffer_rsrc(sb + static_cast<uint64_t>(static_cast<uint32_t>(ks)) * s_step, live ? s_bytes : 0u),
                  k0 + lcol >= row_bytes ? NOWHERE : 0u};
  };
  auto load_one = [&](uint8_t* st, const Source& from, int i) __attribute__((always_inline)) {
    if (i < LA) load16(from.q, st + (NW * i + wave) * 1024, xoff[i < LA ? i : 0] | from.past);
    else if (i < LA + LB) load16(from.w, st + (NW * i + wave) * 1024, woff[i >= LA && i < LA + LB ? i - LA : 0]);
    else load16(from.s, st + CODES + chunk * 1024, soff);
  };

  f32x4 acc[FA][FB];

  const int lrow = lane & 15, lk = lane >> 4;
  uint32_t aoff[2], boff[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    aoff[u] = static_cast<uint32_t>(swz8(wm * FA * 16 + lrow, 4 * u + lk));
    boff[u] = static_cast<uint32_t>(swz8(BM + wn * FB * 16 + lrow, 4 * u + lk));
  }
  // Scales of this wave's rows and columns, a dword a unit for 4 fragments (for 2: the half of a
  // dword from these bits on).
  constexpr int SA = FA == 8 ? 2 : 1;
  const uint32_t sa_at = static_cast<uint32_t>(CODES + wm * FA / 4 * TILE_BYTES + lane * 8);
  const uint32_t sw_at = static_cast<uint32_t>(CODES + XC * 1024 + wn * FB / 4 * TILE_BYTES + lane * 8);
  const int a_bits = 8 * (wm * FA % 4), w_bits = 8 * (wn * FB % 4);

  // Operands: the columns' of a unit, a set a unit; the rows' in a ring of 4, read three rows of
  // MFMAs ahead (a wave of two rows: a set a unit too); both's scales, a set a unit.
  constexpr bool RING = FA >= 4;
  i32x4 af[4], bf[2][FB];
  uint32_t sa[2][SA], sw[2];
  auto read_a = [&](int u, const uint8_t* st, int f) __attribute__((always_inline)) {
    af[(RING ? 0 : 2 * u) + (f & 3)] = *reinterpret_cast<const i32x4*>(st + aoff[u] + f * 16 * BKB);
  };
  auto read_b = [&](int u, const uint8_t* st, int f) __attribute__((always_inline)) {
    bf[u][f] = *reinterpret_cast<const i32x4*>(st + boff[u] + f * 16 * BKB);
  };
  auto read_scales = [&](int u, const uint8_t* st) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < SA; ++h) sa[u][h] = *reinterpret_cast<const uint32_t*>(st + sa_at + h * TILE_BYTES + u * 4);
    sw[u] = *reinterpret_cast<const uint32_t*>(st + sw_at + u * 4);
  };

  // Unit u of a step on stage `cur`, a slot an MFMA: a row's first slot reads the rows ahead, others
  // the next unit's columns and scales. In the second unit, from row TURN on, those are the next
  // step's, from `nxt`, and the slots issue step g + 2's loads into `cur`: ahead of that row this
  // wave's loads of step g + 1 have landed and its reads of `cur`, all of whose operands it has read,
  // are done; past the barrier every wave's.
  constexpr int SLOTS = FA * FB, TURN = RING ? FA - 3 : 0;
  auto region = [&](auto unit_tag, const uint8_t* cur, const uint8_t* nxt, const Source& from) __attribute__((always_inline)) {
    constexpr int U = decltype(unit_tag)::value;
    constexpr int AT = RING ? 0 : 2 * U, FROM = U == 1 ? TURN * FB : 0;
    if constexpr (FA == 2) sa[U][0] >>= a_bits;
    if constexpr (FB == 2) sw[U] >>= w_bits;
    each_of([&](auto slot) __attribute__((always_inline)) {
      constexpr int s = decltype(slot)::value, i = s / FB, j = s % FB;
      if constexpr (U == 1 && s == FROM) {
        wait_vm<0>();
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
      // The weight is the MFMA's A operand: a lane then holds 4 outputs of a row together.
      acc[i][j] = mma<j & 3, i & 3>(bf[U][j], af[AT + (i & 3)], acc[i][j], sw[U], sa[U][i / 4]);
      if constexpr (j == 0) {
        if constexpr (!RING) read_a(U ^ 1, nxt, i);
        else if constexpr (i + 3 < FA) read_a(U, cur, i + 3);
        else read_a(U ^ 1, nxt, i + 3 - FA);
      }
      if constexpr (s > FROM && (s - FROM - 1) % 2 == 0 && (s - FROM - 1) / 2 < FB) read_b(U ^ 1, nxt, (s - FROM - 1) / 2);
      if constexpr (s == FROM + 2) read_scales(U ^ 1, nxt);
      if constexpr (U == 1 && s >= FROM) {
#pragma unroll
        for (int q = 0; q < LOADS; ++q)
          if (FROM + q * (SLOTS - FROM) / LOADS == s) load_one(const_cast<uint8_t*>(cur), from, q);
      }
      __builtin_amdgcn_sched_barrier(0);
    }, std::make_integer_sequence<int, SLOTS>{});
  };
  // Lane l, register r of fragment (i, j): row 16 i + l % 16 of the wave's, column 16 j + 4 (l / 16)
  // + r. Two fragments' trade between the lanes of a row (v_permlane16_swap) gives each lane 8
  // columns together, and with four fragments the lanes of rows r and r + 8 trade (row_ror:8), so
  // that a store writes 8 rows of 128 bytes: whole lines (8 bytes a lane as they come, 32 together,
  // took a quarter of a 4096 x 8192 -> 28672 call's time, as the next step's wait for its loads waits
  // for the stores too).
  typedef u32x4 __attribute__((aligned(2))) loose_u32x4;  // rows of an odd width begin anywhere
  constexpr int STORES = FB == 2 ? 1 : 2;                // of a row of fragments
  auto store_tile = [&](const Tile& t, auto whole_tag) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole_tag)::value;  // all columns are there
    const int n0 = t.n0 + wn * FB * 16;
    // This lane's row of store i, of the tile: first + 16 / STORES i; its columns, from n0.
    const int first = wm * FA * 16 + (FB == 2 ? lrow : lrow & 7);
    const int col = 16 * (lk & 1) + 8 * (lk >> 1) + (FB == 2 ? 0 : 32 * (lrow >> 3));
    int to_row[EXPERTS ? STORES * FA : 1];
    if constexpr (EXPERTS) {
#pragma unroll
      for (int i = 0; i < STORES * FA; ++i) to_row[i] = a.order[t.first + min(first + (16 / STORES) * i, t.live - 1)];
    }
    // The rows are here before the first store: a wait for them between stores would wait for the
    // stores too, each in turn.
    if constexpr (EXPERTS) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __builtin_amdgcn_sched_barrier(0);
    // The next store's row, or with experts the columns of any.
    uint16_t* to = EXPERTS ? a.y + n0 + col : a.y + static_cast<int64_t>(t.m0 + first) * a.N + n0 + col;
    const int64_t step = static_cast<int64_t>(16 / STORES) * a.N;
    auto store = [&](int i, u32x4 v) __attribute__((always_inline)) {
      if (first + (16 / STORES) * i >= t.live) return;
      uint16_t* const at = EXPERTS ? to + static_cast<int64_t>(to_row[EXPERTS ? i : 0]) * a.N : to;
      if (WHOLE || n0 + col + 8 <= a.N) {
        // Past the L2's usual order: what y would push out there, the operands, is read again.
        __builtin_nontemporal_store(v, reinterpret_cast<loose_u32x4*>(at));
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (n0 + col + r < a.N) at[r] = static_cast<uint16_t>(v[r >> 1] >> (16 * (r & 1)));
      }
    };
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      uint32_t o[FB][2];
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float lo = acc[i][j][2 * h], hi = acc[i][j][2 * h + 1];
          o[j][h] = DT == LNQ_BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
        }
      // Lane quarter k of fragments 2 p, 2 p + 1 then holds columns 8 (k / 2) .. + 7 of fragment 2 p + k % 2.
#pragma unroll
      for (int j = 0; j < FB; j += 2)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const auto r = __builtin_amdgcn_permlane16_swap(o[j][h], o[j + 1][h], false, false);
          o[j][h] = r[0], o[j + 1][h] = r[1];
        }
      if constexpr (FB == 2) {
        store(i, u32x4{o[0][0], o[0][1], o[1][0], o[1][1]});
        if (!EXPERTS) to += step;
      } else {
        u32x4 p, q;
        const uint32_t pv[4] = {o[0][0], o[0][1], o[1][0], o[1][1]}, qv[4] = {o[2][0], o[2][1], o[3][0], o[3][1]};
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          // Rows 0 .. 7: the first half of the columns from their own lanes, the second in the lanes of
          // rows 8 .. 15; then the same of those rows.
          p[d] = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(pv[d]), static_cast<int>(qv[d]), 0x128, 0xf, 0xc, false));
          q[d] = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(qv[d]), static_cast<int>(pv[d]), 0x128, 0xf, 0x3, false));
        }
        store(2 * i, p);
        if (!EXPERTS) to += step;
        store(2 * i + 1, q);
        if (!EXPERTS) to += step;
      }
      // One row of fragments at a time: the next tile's operands are live here.
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto epilogue = [&](const Tile& t) __attribute__((always_inline)) {
    if (EXPERTS && t.e >= a.count) {  // pairs whose choice is no expert: zeros
#pragma unroll
      for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (!EXPERTS && a.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < FB; ++j) {
        f32x4 bias;
#pragma unroll
        for (int r = 0; r < 4; ++r) bias[r] = E::to_f32(a.bias[min(t.n0 + (wn * FB + j) * 16 + 4 * lk + r, a.N - 1)]);
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] += bias[r];
      }
    }
    if (t.n0 + BN <= a.N) store_tile(t, std::true_type{});
    else store_tile(t, std::false_type{});
  };

  // `now` multiplies, `loading` is the tile of the loads (the same, or the next one: a tile has two
  // steps or more), tile `ready` comes after it. Experts: its rows' pairs are asked for, the entry of
  // the one after and the expert of the one after that, a tile before they are used.
  Tile now, loading, next;
  i32x4 ahead = {0, 0, 0, 0}, ahead2 = {0, 0, 0, 0};
  int ahead_n0 = 0, ahead_m0 = 0, ready = 1;
  auto prepare = [&]() {
    if constexpr (EXPERTS) {
      next = expert_tile(ahead, ahead_n0, ahead_m0);
      ahead = entry_of(ready + 1, ahead2, ahead_n0, ahead_m0);
      ahead2 = expert_of(ready + 2);
      take_pairs(next);
    } else {
      next = plain_tile(min(ready, mine - 1));
    }
  };
  if constexpr (EXPERTS) {
    int n0, m0;
    const i32x4 entry = entry_of(0, expert_of(0), n0, m0);
    now = expert_tile(entry, n0, m0);
    ahead = entry_of(1, expert_of(1), ahead_n0, ahead_m0);
    ahead2 = expert_of(2);
  } else {
    now = plain_tile(0);
  }
  take_pairs(now);
  loading = now;
  load_tile(loading);
  // Steps 0 and 1 requested; step 0 landed (this wave's, then every wave's); its first operands and
  // scales read.
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const Source from = source_of(true, j);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_one(j ? L1 : L0, from, i);
  }
  wait_vm<LOADS>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int i = 0; i < FB; ++i) read_b(0, L0, i);
#pragma unroll
  for (int i = 0; i < (RING ? 3 : 2); ++i) read_a(0, L0, i);
  read_scales(0, L0);
  prepare();

  int ks = 2;  // k-step of the next load
  // Step g on stage `cur`, no branch inside.
  auto step = [&](uint8_t* cur, uint8_t* nxt, bool in) __attribute__((always_inline)) {
    const Source from = source_of(in, ks);
    region(std::integral_constant<int, 0>{}, cur, cur, from);
    region(std::integral_constant<int, 1>{}, cur, nxt, from);
    ++ks;
  };
  for (int g = 0; g < nsteps;) {
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (const int end = g + steps; g < end; g += 2) {
      if (ks == steps) {
        ks = 0;
        loading = next;
        load_tile(loading);
        ++ready;
        prepare();
      }
      step(L0, L1, g + 2 < nsteps);
      step(L1, L0, g + 3 < nsteps);
    }
    epilogue(now);
    now = loading;
  }
  // Loads of the steps past the stream (0-byte reads) may be in flight.
  wait_vm<0>();
}

// The pairs of each expert, in order, by the places of its tiles: workgroup e counts every expert's
// pairs, which tells it where its own tiles begin, then lists them, each wave those of its own run
// of the pairs; places past them name pair 0. Workgroup `count` lists the pairs whose choice is no
// expert and writes how many tiles there are.
__device__ __attribute__((always_inline)) inline void list_pairs(int e, const int64_t* experts, int pairs, int count, int bm, int* order, i32x4* table, int* used) {
  using namespace mx4;
  constexpr int WAVES = LIST_THREADS / 64, DEEP = 8;  // loads in flight
  __shared__ int number[MAX_EXPERTS + 1];
  __shared__ int part[2][WAVES], found[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (pairs + 64 * WAVES - 1) / (64 * WAVES) * 64;  // pairs of a wave
  const int from = wave * run, to = min(pairs, from + run);
  // Calls f(pair, its bucket) for this wave's pairs, a lane each; past the last, a bucket of -1.
  auto each = [&](auto f) {
    for (int p0 = from; p0 < to; p0 += 64 * DEEP) {
      int64_t id[DEEP];
#pragma unroll
      for (int d = 0; d < DEEP; ++d) id[d] = experts[min(p0 + 64 * d + lane, pairs - 1)];
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        const int p = p0 + 64 * d + lane;
        f(p, p >= to ? -1 : id[d] >= 0 && id[d] < count ? static_cast<int>(id[d]) : count);
      }
    }
  };
  for (int i = tid; i <= count; i += LIST_THREADS) number[i] = 0;
  __syncthreads();
  int here = 0;
  each([&](int, int bucket) {
    if (bucket >= 0) atomicAdd(&number[bucket], 1);
    here += __popcll(__ballot(bucket == e));
  });
  if (lane == 0) found[wave] = here;
  __syncthreads();
  // Tiles of the experts before this one, and of all.
  int sums[2] = {0, 0};
  for (int i = tid; i <= count; i += LIST_THREADS) {
    const int t = (number[i] + bm - 1) / bm;
    if (i < e) sums[0] += t;
    sums[1] += t;
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sums[s] += __shfl_xor(sums[s], off, 64);
    if (lane == 0) part[s][wave] = sums[s];
  }
  __syncthreads();
  int tile = 0, all = 0, at = 0;
#pragma unroll 4
  for (int v = 0; v < WAVES; ++v) {
    tile += part[0][v], all += part[1][v];
    if (v < wave) at += found[v];
  }
  const int mine = number[e], tiles = (mine + bm - 1) / bm;
  for (int i = tid; i < tiles; i += LIST_THREADS) table[tile + i] = i32x4{e, (tile + i) * bm, min(bm, mine - i * bm) + 512 * tiles, tile};
  if (e == count && tid == 0) used[0] = all;
  if (mine == 0) return;
  at += tile * bm;
  if (mine + tid < tiles * bm) order[tile * bm + mine + tid] = 0;
  each([&](int p, int bucket) {
    const uint64_t mask = __ballot(bucket == e);
    if (bucket == e) order[at + __popcll(mask & ((uint64_t{1} << lane) - 1))] = p;
    at += __popcll(mask);
  });
}

// What the product of the experts needs: workgroups 0 .. count list the pairs, and the others round
// x's rows, four blocks of mxr::THREADS threads each (`spans` of them to a run of rows, `blocks` in
// all). Neither waits for the other: in one launch the shorter costs nothing (4 to 10 us).
template <int DT>
__global__ __launch_bounds__(mx4::LIST_THREADS, 8) void expert_prepare_kernel(const int64_t* __restrict__ experts, int pairs,
                                                                           int count, int bm, int* __restrict__ order,
                                                                           i32x4* __restrict__ table, int* __restrict__ used,
                                                                           const uint16_t* __restrict__ x, int64_t x_stride,
                                                                           uint32_t* __restrict__ codes,
                                                                           uint32_t* __restrict__ scales, int rows, int K,
                                                                           int spans, int blocks) {
  if (static_cast<int>(blockIdx.x) <= count) {
    list_pairs(blockIdx.x, experts, pairs, count, bm, order, table, used);
  } else {
    constexpr int EACH = mx4::LIST_THREADS / mxr::THREADS;
    __shared__ uint32_t unit[EACH][2 * mxr::ROWS];
    const int part = __builtin_amdgcn_readfirstlane(threadIdx.x / mxr::THREADS);
    const int b = (blockIdx.x - count - 1) * EACH + part, block = min(b, blocks - 1);
    mxr::round_rows<DT>(x, x_stride, codes, scales, rows, K, unit[part], threadIdx.x % mxr::THREADS, block / spans,
                                block % spans, b < blocks);
  }
}

// x's scales by the tiles' rows, as scale tiles: `each` blocks of 64 rows a tile of bm.
__global__ __launch_bounds__(256) void expert_scales_kernel(const uint8_t* __restrict__ from, uint32_t* __restrict__ to,
                                                            const int* __restrict__ order, const int* __restrict__ used,
                                                            int from_blocks, int blocks, int each, int bm, int chosen) {
  const int i = blockIdx.x * 256 + threadIdx.x, block = i >> 7;
  if (block >= blocks) return;
  const int t = block / each, r0 = (block - t * each) * 64 + (i >> 1 & 15);  // of the tile
  const int64_t pair = blockIdx.y;
  const uint32_t at = (i >> 5 & 3) * 128 + (i & 1) * 4;  // block of the unit, unit
  const int tiles = used[0];
  int place[4];  // beside the load above, and used only if the tile is there
#pragma unroll
  for (int f = 0; f < 4; ++f) place[f] = order[t * bm + min(r0 + 16 * f, bm - 1)];
  if (t >= tiles) return;
  uint32_t word = 0;
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    const int row = place[f] / chosen;
    const uint8_t byte = from[(pair * from_blocks + (row >> 6)) * mx4::TILE_BYTES + at + (row & 15) * 8 + (row >> 4 & 3)];
    word |= static_cast<uint32_t>(byte) << (8 * f);
  }
  to[pair * blocks * 128 + i] = word;
}

namespace mx4 {

template <int DT, class FORM, bool EXPERTS>
static void launch_form(const Args& a, hipStream_t s) {
  const int64_t tiles_n = (a.N + FORM::BN - 1) / FORM::BN;
  const int64_t tiles = EXPERTS ? (a.tiles * tiles_n + mm8::XCDS - 1) / mm8::XCDS * mm8::XCDS
                                : (a.M + FORM::BM - 1) / FORM::BM * tiles_n;
  const int64_t most = compute_units() / mm8::XCDS * mm8::XCDS * FORM::PER_CU;
  hipLaunchKernelGGL((mx4_kernel<DT, FORM, EXPERTS>), dim3(static_cast<unsigned>(tiles < most ? tiles : most)),
                     dim3(FORM::THREADS), 0, s, a);
}

using Form256 = Form<2, 4, 8, 4>;
using Form128 = Form<2, 2, 4, 4>;
using Form64 = Form<2, 2, 2, 2>;
using Form32 = Form<1, 2, 2, 4>;  // (of 64 columns, 100 rows' experts 72.1 us against 68.5)

// Rows of a tile, for `count` matrices of N outputs that multiply `rows` rows each (experts: on
// average). A larger tile reads each operand less often (a wave of 128 x 64 outputs, 24 KB of LDS for
// 64 MFMAs; of 64 x 64, 32 KB; of 32 x 32, 64 KB), a smaller one leaves fewer CUs idle and fewer rows
// empty. Measured on both sides of each bound (256 CUs; us of the smaller | the larger tile):
// 256 rows from 0.7 of a tile a CU: 2048 x 4096 -> 4096, 128 tiles: 21.6 | 28.7; 2048 x 2880 -> 5760,
// 184: 27.4 | 26.7; 1024 x 4096 -> 14336, 224: 37.2 | 32.4; 4096 x 8192 -> 8192, 512: 132 | 116. 128
// rows from 5/8: 128 x 4096 -> 14336, 112 tiles: 11.2 | 13.5; 512 x 2880 -> 5760, 180: 13.6 | 11.2;
// 1024 x 4096 -> 4096, 256: 18.5 | 14.1.
// Of an expert's rows: 256 past 128 (32 experts, 2880 -> 5760: at 75 rows 77 | 89, 188: 129 | 105; 128
// experts, 2048 -> 1536: at 125 63 | 65, 188: 81 | 72; worst, 8 experts, 4096 -> 14336 at 250, whose
// tiles then fill a third round: 85 | 109); 128 past 20 (32 experts, 2880 -> 5760, 32 rows a tile | 128:
// at 12 62 | 66, 25: 65 | 68, 38: 82 | 70; 2880 -> 2880: at 12 35 | 38, 25: 43 | 39; 64 rows are the best
// by 7 percent at most between them, and taken where 128 leave CUs idle).
static int tile_rows(double rows, int64_t count, int64_t N, bool experts) {
  const auto tiles = [&](int bm, int bn) {
    return static_cast<double>(count) * std::ceil(rows / bm) * static_cast<double>((N + bn - 1) / bn);
  };
  const int many = experts ? 20 : 64;
  if (rows > 128 && tiles(256, 256) >= 0.7 * compute_units()) return 256;
  if (rows > many && tiles(128, 128) >= 0.625 * compute_units()) return 128;
  return rows > many || !experts ? 64 : 32;
}

template <int DT, bool EXPERTS>
static void launch(const Args& a, int bm, hipStream_t s) {
  if constexpr (EXPERTS) {
    if (bm == 32) return launch_form<DT, Form32, EXPERTS>(a, s);
  }
  if (bm == 64) launch_form<DT, Form64, EXPERTS>(a, s);
  else if (bm == 128) launch_form<DT, Form128, EXPERTS>(a, s);
  else launch_form<DT, Form256, EXPERTS>(a, s);
}

// The workspace of a call with tiles of `bm` pairs (tiles at most: a partial one for each expert that
// is named): x's codes and scale tiles, the pairs by the tiles' places, the tile table with how many there are, x's
// scales by the tiles' rows.
struct Plan {
  int tiles, each;  // blocks of 64 rows a tile
  int64_t blocks, scales, order, table, sorted, bytes;  // of 64 rows in all; where each begins
};

static Plan experts_plan(int bm, int64_t pairs, int64_t x_rows, int64_t count, int64_t in_features) {
  const auto whole = [](int64_t bytes) { return (bytes + 127) / 128 * 128; };
  const int64_t spans = (in_features + 255) / 256;
  Plan p{};
  p.tiles = static_cast<int>(pairs / bm + std::min(pairs, count + 1));
  p.each = (bm + 63) / 64;
  p.blocks = static_cast<int64_t>(p.tiles) * p.each;
  p.scales = whole(x_rows * (in_features / 2));
  p.order = p.scales + spans * ((x_rows + 63) / 64) * TILE_BYTES;
  p.table = p.order + whole(static_cast<int64_t>(p.tiles) * bm * 4);
  p.sorted = p.table + whole(static_cast<int64_t>(p.tiles) * 16 + 16);
  p.bytes = p.sorted + spans * p.blocks * TILE_BYTES;
  return p;
}

// Of any outputs: whichever tiles they take.
static int64_t workspace_of(int64_t pairs, int64_t x_rows, int64_t count, int64_t in_features) {
  int64_t bytes = 0;
  for (const int bm : {32, 64, 128, 256}) bytes = std::max(bytes, experts_plan(bm, pairs, x_rows, count, in_features).bytes);
  return bytes;
}

template <int DT>
static void prepare(const Args& a, const int64_t* experts, int pairs, int bm, const void* x, int64_t x_stride, uint8_t* scales,
                    hipStream_t s) {
  const int spans = mxr::spans_of(a.K), blocks = (a.M + mxr::ROWS - 1) / mxr::ROWS * spans, each = LIST_THREADS / mxr::THREADS;
  const dim3 grid(static_cast<unsigned>(a.count + 1 + (blocks + each - 1) / each));
  hipLaunchKernelGGL((expert_prepare_kernel<DT>), grid, dim3(LIST_THREADS), 0, s, experts, pairs, a.count, bm,
                     const_cast<int*>(a.order), const_cast<i32x4*>(a.table), const_cast<int*>(a.used), static_cast<const uint16_t*>(x),
                     x_stride, reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(a.q)), reinterpret_cast<uint32_t*>(scales), a.M, a.K,
                     spans, blocks);
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
  LNQ_REQUIRE(aligned(q, 16) && aligned(x_scale, 16) && aligned(blocks, 16) && aligned(tiles, 16) && aligned(y, 2),
              "lnq_mxfp4_mm: operands must be 16-byte aligned");
  mx4::Args a{};
  a.q = q;
  a.xs = x_scale;
  a.w = blocks;
  a.ws = tiles;
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.M = static_cast<int>(rows);
  a.x_blocks = mx4::blocks_of(a.M);
  a.N = static_cast<int>(out_features);
  a.K = static_cast<int>(in_features);
  LNQ_REQUIRE((rows + 31) / 32 * ((out_features + 63) / 64) <= INT32_MAX, "lnq_mxfp4_mm: too large");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int bm = mx4::tile_rows(static_cast<double>(rows), 1, out_features, false);
  if (dtype == LNQ_BF16) mx4::launch<LNQ_BF16, false>(a, bm, s);
  else mx4::launch<LNQ_F16, false>(a, bm, s);
  return launched("mxfp4_mm");
}

LNQ_API LnqStatus lnq_mxfp4_experts_workspace(int64_t pairs, int64_t x_rows, int64_t num_experts, int64_t in_features,
                                              int64_t* bytes) {
  LNQ_REQUIRE(bytes != nullptr, "lnq_mxfp4_experts_workspace: null pointer");
  LNQ_REQUIRE(pairs >= 0 && pairs <= (1 << 26) && x_rows >= 0 && x_rows <= (1 << 27) && num_experts > 0 &&
                  num_experts <= mx4::MAX_EXPERTS && in_features > 0 && in_features <= (1 << 22),
              "lnq_mxfp4_experts_workspace: %lld pairs and %lld rows of %lld experts (1 to %d) of %lld inputs",
              static_cast<long long>(pairs), static_cast<long long>(x_rows), static_cast<long long>(num_experts),
              mx4::MAX_EXPERTS, static_cast<long long>(in_features));
  *bytes = pairs == 0 ? 0 : mx4::workspace_of(pairs, x_rows, num_experts, in_features);
  clear_error();
  return LNQ_OK;
}

LNQ_API LnqStatus lnq_mxfp4_experts_mm(const void* x, int64_t x_stride, const uint8_t* blocks, const uint8_t* tiles,
                                       const int64_t* experts, void* y, int64_t rows, int64_t chosen, int64_t num_experts,
                                       int64_t out_features, int64_t in_features, int32_t shared, int32_t dtype,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16, "lnq_mxfp4_experts_mm: x and y are bf16 or f16, not dtype %d", dtype);
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
  LNQ_REQUIRE(x && blocks && tiles && experts && y, "lnq_mxfp4_experts_mm: null pointer");
  LNQ_REQUIRE(x_stride >= 0 && x_stride % 8 == 0 && aligned(x, 16) && aligned(blocks, 16) && aligned(tiles, 16) &&
                  aligned(y, 2) && aligned(workspace, 16),
              "lnq_mxfp4_experts_mm: x (with its row stride), the weight and the workspace must be 16-byte aligned");
  const int64_t pairs = rows * chosen, x_rows = shared ? rows : pairs;
  LNQ_REQUIRE(x_rows * (in_features / 2) < (int64_t{1} << 31), "lnq_mxfp4_experts_mm: x's codes past 2 GiB");
  const int bm = mx4::tile_rows(static_cast<double>(pairs) / static_cast<double>(num_experts), num_experts, out_features, true);
  const mx4::Plan plan = mx4::experts_plan(bm, pairs, x_rows, num_experts, in_features);
  LNQ_REQUIRE(plan.blocks <= (1 << 21) && static_cast<int64_t>(plan.tiles) * ((out_features + 63) / 64) <= INT32_MAX,
              "lnq_mxfp4_experts_mm: too large");
  const int64_t need = mx4::workspace_of(pairs, x_rows, num_experts, in_features);
  LNQ_REQUIRE(workspace && workspace_bytes >= need, "lnq_mxfp4_experts_mm: workspace of %lld bytes, %lld needed",
              static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  auto* const space = static_cast<uint8_t*>(workspace);
  uint8_t *const scales = space + plan.scales, *const sorted = space + plan.sorted;
  mx4::Args a{};
  a.q = space;
  a.xs = sorted;
  a.w = blocks;
  a.ws = tiles;
  a.y = static_cast<uint16_t*>(y);
  a.M = static_cast<int>(x_rows);
  a.x_blocks = static_cast<int>(plan.blocks);
  a.N = static_cast<int>(out_features);
  a.K = static_cast<int>(in_features);
  a.order = reinterpret_cast<const int*>(space + plan.order);
  a.table = reinterpret_cast<const i32x4*>(space + plan.table);
  a.used = reinterpret_cast<const int*>(a.table + plan.tiles);
  a.tiles = plan.tiles;
  a.count = static_cast<int>(num_experts);
  a.chosen = shared ? static_cast<int>(chosen) : 1;
  a.w_step = out_features * (in_features / 2);
  a.ws_step = static_cast<int64_t>(mx4::pairs_of(a.K)) * mx4::blocks_of(a.N) * mx4::TILE_BYTES;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == LNQ_BF16) mx4::prepare<LNQ_BF16>(a, experts, static_cast<int>(pairs), bm, x, x_stride, scales, s);
  else mx4::prepare<LNQ_F16>(a, experts, static_cast<int>(pairs), bm, x, x_stride, scales, s);
  if (const LnqStatus st = launched("expert_prepare")) return st;
  hipLaunchKernelGGL(expert_scales_kernel, dim3(static_cast<unsigned>((plan.blocks + 1) / 2), static_cast<unsigned>(mx4::pairs_of(a.K))),
                     dim3(256), 0, s, scales, reinterpret_cast<uint32_t*>(sorted), a.order, a.used, mx4::blocks_of(a.M), a.x_blocks,
                     plan.each, bm, a.chosen);
  if (const LnqStatus st = launched("expert_scales")) return st;
  if (dtype == LNQ_BF16) mx4::launch<LNQ_BF16, true>(a, bm, s);
  else mx4::launch<LNQ_F16, true>(a, bm, s);
  return launched("mxfp4_experts_mm");
}

}  // extern "C"
