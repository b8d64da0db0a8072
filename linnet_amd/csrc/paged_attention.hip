// Attention over a KV cache in pages, for a batch of sequences with any number of new tokens each:
//
//   out = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m)),  s_j = scale q . k_j,
//
// over the entries j that a row sees: those up to its own (within its window), or, of a drafted
// tree, the entries before the draft and the nodes on the path to its own. One pass over K and V with a running
// maximum and sum; sums and outputs in f32, the weights e^(s_j - m) rounded to 16 bits for their
// product with V (a rounding of the size of V's own, its errors as likely up as down).
//
// A wave takes 32 rows: the query heads that share a KV head, of one token after the other. Its products are
// S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMAs, both with a row to a column. A lane then has 16 of
// a row's 32 scores (lane + 32 the others), so that a row's maximum and sum are the lane's own and
// one exchange; and with the entries of an MFMA's rows in the order of `entry_of_row`, a lane's
// scores are, in its own registers, the operand of the second product: no weight goes through LDS.
//
// Two ways. `few`: sequences of up to 32 rows (decode steps, small drafts). Bound by memory: 4
// waves of a workgroup take steps of 32 entries in turn, K and V straight from the pages to registers,
// a step ahead, and add up through LDS. `many`: tiles of 128 rows, 32 a wave, which share tiles of
// 64 entries in LDS, loaded a tile ahead. Where the rows are few for the chip, the entries are split over
// workgroups too, and a last kernel adds the parts in order. Which sequence is which is on the device:
// a call that may have both runs both in one launch.
//
// Measured: 64 sequences of 230000 entries together, 32 heads over 8 of 128 (942 MB), 172 to 181 us: 5.2 to 5.5 TB/s. One of 131000 entries
// at head_dim 64, 8 KV heads, 57 to 60 us. Prompts of 8191 tokens (203 GFLOP) 225 us: 0.90 PFLOP/s, bound by the MFMAs (busy
// 46% of the time), the softmax's vector instructions, of which they hide about half, and a clock that falls to 2.0
// GHz under both (a step of 64 entries takes a wave 32 MFMAs and 126 vector instructions, 32 of them
// exponentials). 16 trees of 46 to 67 nodes over 70000 entries 130 us; one token over 1024 entries 9.4.
#include <math.h>

#include <type_traits>

#include "paged.hpp"

namespace lnq {
namespace paged {

constexpr int FEW = 32;          // rows of a sequence that the few-row kernel takes (in tiles of 16 or 32) at most
constexpr int MANY = 128;        // rows of the other's
constexpr int FEW_STEP = 128;    // entries a workgroup of the few-row kernel takes at a time
constexpr int MANY_STEP = 64;
constexpr int NODES = 256;       // of a drafted tree
constexpr int MAX_SPLITS = 256;
// Of a workspace, 1 GiB. Parts are as many as the tables could fill, for every sequence: without a bound, 512 sequences with
// a chunk among them under tables of 131072 entries (32 heads of 128, parts of four tokens each) take 4.4 GB and at
// 1800 to 5400 entries 2584 us, with it 1809 (2669 and 1904 where one sequence has 131000); the largest batches 140 GB.
constexpr int64_t MOST_FLOATS = int64_t{1} << 28;

// f16 weights are kept times 2^7: with the maximum's slack of 2^8 they stay below 2^15 (f16 ends at 2^16), and what
// rounds to 0 is below 2^-32 of the largest, not 2^-25, of which the tail of a long cache can hold a sizable sum.
template <int DT>
constexpr float LIFT = DT == LNQ_F16 ? 7.f : 0.f;

// The maximum of a row's scores in the stored form: times log2 e, less the lift, so that weights are 2^(score - it).
template <int DT>
__device__ inline float stored_max(float m, float c) { return m == -INFINITY ? m : fmaf(m, c, -LIFT<DT>); }

// The sums of tiles whose entries are split, for each of the splits and rows: the outputs so far, [splits][rows]
// [head_dim], and stored_max and sum, [splits][rows][2].
struct Parts {
  float *sums, *stats;
  int64_t rows;
  int splits;  // at most
};

struct AttendArgs {
  const uint16_t *q, *k_cache, *v_cache;
  uint16_t* out;
  int64_t q_stride, out_stride;
  const float* sinks;      // [heads] or nullptr
  const int32_t* parents;  // [tokens]: a node's parent among its sequence's new tokens; nullptr: no tree
  Parts small, large;      // of few rows' sequences and of the others
  Batch batch;
  int heads, kv_heads, group, window;
  int few_tokens;          // few: new tokens of a sequence that may be split
  int few, few_tile;       // rows of a sequence that `few` takes, and of a tile of it
  float scale2;            // scale * log2 e
  bool every;              // few: sequences of any number of rows
  bool fill;               // few: rows past the last sequence become zeros
};

// The MFMAs of 32 x 32 (16 summed) and of 16 x 16 (32 summed): TILE rows or columns in lane l % TILE, the
// lanes' GROUPS = 64 / TILE groups holding eight of the summed indices each; of the result, column l % TILE and
// rows 4 GROUPS (r / 4) + 4 (l / TILE) + r % 4 in registers r < REGS.
template <int TILE>
struct Shape {
  static constexpr int GROUPS = 64 / TILE, REGS = TILE * TILE / 64, SUMMED = 8 * GROUPS;
  typedef float acc __attribute__((ext_vector_type(REGS)));
};

template <int DT, int TILE>
__device__ inline typename Shape<TILE>::acc mma(u32x4 a, u32x4 b, typename Shape<TILE>::acc c) {
  if constexpr (TILE == 16) return mfma16x16x32<DT>(a, b, c);
  else if constexpr (DT == LNQ_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT>
__device__ inline uint32_t pack2(float a, float b) {
  return DT == LNQ_BF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b);
}

// acc + the two values of a dword (as they are after rounding), one instruction.
template <int DT>
__device__ inline float add2(uint32_t pair, float acc) {
  if constexpr (DT == LNQ_BF16) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, Elem<DT>::ONE2), acc, false);
  else return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), __builtin_bit_cast(f16x2, Elem<DT>::ONE2), acc, false);
}

// The entry (of 32) at row m of the first product's n-th tile: a lane's results are then, in the order
// of its registers, runs of the eight entries 8 (GROUPS s + group) .. + 7, the second product's summed indices.
template <int TILE>
__device__ inline int entry_of(int n, int m) {
  if constexpr (TILE == 16) return 8 * (m >> 2) + 4 * n + (m & 3);
  const int b = m >> 3, h = m >> 2 & 1, e = m & 3;
  return 16 * (b >> 1) + 8 * h + 4 * (b & 1) + e;
}

// A value of each of the lanes that share a column (l, l ^ 32; with 16 columns l ^ 16 and l ^ 48 too), joined.
template <int TILE, class F>
__device__ inline float across(float v, F join) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  v = join(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
  if constexpr (TILE == 16) {
    u = __builtin_bit_cast(uint32_t, v);
    const auto q = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = join(__builtin_bit_cast(float, static_cast<uint32_t>(q[0])), __builtin_bit_cast(float, static_cast<uint32_t>(q[1])));
  }
  return v;
}

template <int TILE>
__device__ inline float max_across(float v) {
  return across<TILE>(v, [](float a, float b) { return fmaxf(a, b); });
}

template <int TILE>
__device__ inline float sum_across(float v) {
  return across<TILE>(v, [](float a, float b) { return a + b; });
}

// The entries that the tokens i0 .. i1 of a sequence see among them, [lo, hi), and their division.
struct Range {
  int lo, hi, chunk, used;
};

__device__ inline Range range_of(const AttendArgs& a, const Sequence& q, int i0, int i1, int splits, int step) {
  Range r;
  const bool tree = a.parents != nullptr;
  r.hi = a.batch.pages == 0 ? 0 : min(tree ? q.length : q.base + i1 + 1, capacity(a.batch));
  r.lo = a.window > 0 ? max(0, q.base + (tree ? 0 : i0) - a.window + 1) & -step : 0;
  const int many = max(0, r.hi - r.lo);
  r.chunk = max(((many + splits - 1) / splits + step - 1) / step, 1) * step;
  r.used = max((many + r.chunk - 1) / r.chunk, 1);
  return r;
}

// What a row sees: entries low .. last, and of a tree the nodes `path` (bits, NODES of them in LDS).
struct Row {
  int low, last;
  const uint32_t* path;
};

template <bool TREE>
__device__ inline Row row_of(const AttendArgs& a, const Sequence& q, int i, const uint32_t* paths, const int* depth) {
  Row r;
  r.path = nullptr;
  if constexpr (TREE) {
    const bool node = i < NODES;
    r.path = paths + (node ? i : 0) * (NODES / 32);
    r.last = node ? q.base - 1 : -1;
    r.low = !node ? 0x7fffffff : a.window > 0 ? q.base + depth[node ? i : 0] - a.window + 1 : 0;
    if (!node) r.path = nullptr;
  } else {
    r.last = q.base + i;
    r.low = a.window > 0 ? r.last - a.window + 1 : 0;
  }
  return r;
}

// A tree's parent of this thread's node. (A parent that is no earlier node is the entry before the draft.)
__device__ inline int parent_of(const AttendArgs& a, const Sequence& q) {
  const int i = threadIdx.x;
  if (i >= min(q.n, NODES)) return -1;
  const int p = a.parents[q.first + i];
  return p >= 0 && p < i ? p : -1;
}

// The paths from each node to the draft's root, bit j for node j, within the window, a thread a node (NODES
// threads, all of which take part).
__device__ inline void paths_of(const AttendArgs& a, const Sequence& q, int parent, uint32_t* paths, int* depth, int* up) {
  const int n = min(q.n, NODES), i = threadIdx.x;
  up[i] = parent;
  lds_barrier();
  if (i < n) {
    const int most = a.window > 0 ? a.window : NODES;
    uint32_t* const path = paths + i * (NODES / 32);
#pragma unroll
    for (int w = 0; w < NODES / 32; ++w) path[w] = 0;
    int many = 0, word = i >> 5;
    uint32_t bits = 0;
    for (int j = i; j >= 0; ++many) {
      if (j >> 5 != word) path[word] = bits, bits = 0, word = j >> 5;
      if (many < most) bits |= 1u << (j & 31);
      j = up[j];
    }
    path[word] = bits;
    depth[i] = many - 1;
  }
  lds_barrier();
}

// Of the 32 entries from t, those the row sees, as bits in the order of this lane's registers.
// valid: the entries that are there.
template <bool TREE, int TILE>
__device__ inline uint32_t seen_of(const Row& row, int t, uint32_t valid, int base, int group) {
  constexpr int GROUPS = Shape<TILE>::GROUPS;
  uint32_t bits = 0;
#pragma unroll
  for (int s = 0; s < 4 / GROUPS; ++s) {
    const int at = 8 * (GROUPS * s + group), first = t + at;
    const int from = row.low - first, to = row.last - first;
    uint32_t m = from <= 0 ? 0xffu : from > 7 ? 0u : 0xffu << from & 0xffu;
    m &= to >= 7 ? 0xffu : to < 0 ? 0u : (2u << to) - 1u;
    if constexpr (TREE) {
      const int x = first - base;  // the node at the first of the eight entries
      if (row.path != nullptr && x > -8 && x < NODES) {
        const int w = x >> 5;
        const uint64_t two = (static_cast<uint64_t>(w + 1 < NODES / 32 ? row.path[w + 1] : 0u) << 32) | (w >= 0 ? row.path[w] : 0u);
        m |= static_cast<uint32_t>(two >> (x & 31)) & 0xffu;
      }
    }
    bits |= (m & valid >> at) << (8 * s);
  }
  return bits;
}

// All ones where bit i of `bits` is set, else 0.
__device__ inline uint32_t whole(uint32_t bits, int i) {
  return static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), static_cast<uint32_t>(i), 1u));
}

// Eight 16-bit masks from eight bits.
__device__ inline u32x4 masks_of(uint32_t bits) {
  u32x4 v;
#pragma unroll
  for (int d = 0; d < 4; ++d) v[d] = (whole(bits, 2 * d) & 0xffffu) | (whole(bits, 2 * d + 1) & 0xffff0000u);
  return v;
}

__device__ inline u32x4 and_of(u32x4 a, u32x4 b) { return u32x4{a[0] & b[0], a[1] & b[1], a[2] & b[2], a[3] & b[3]}; }

// Infinities and NaNs in pairs of 16-bit values, by sums that carry into a half's top bit: all
// exponent bits set, and of those a mantissa that is not 0.
template <int DT>
struct Odd {
  static constexpr int BITS = DT == LNQ_BF16 ? 7 : 10;  // of the mantissa
  static constexpr uint32_t MANTISSA = (1u << BITS) - 1, EXPONENT = 0x7fffu & ~MANTISSA, TOP = 0x80008000u;
  __device__ static uint32_t twice(uint32_t v) { return v | v << 16; }
  __device__ static uint32_t odd(uint32_t x) { return ((x & twice(EXPONENT)) + twice(MANTISSA + 1)) & TOP; }
  __device__ static uint32_t nan(uint32_t x) { return odd(x) & ((x & twice(MANTISSA)) + twice(MANTISSA)) << (15 - BITS); }
  __device__ static uint32_t spread(uint32_t tops) { return (tops - (tops >> 15)) | tops; }  // top bits to whole halves
  // 1 where the value is +inf (kind 0), -inf (1) or NaN (2), else 0.
  __device__ static uint32_t is(uint32_t x, int kind) {
    const uint32_t n = nan(x);
    return spread(kind == 2 ? n : odd(x) & ~n & (kind == 1 ? x : ~x)) & Elem<DT>::ONE2;
  }
};

template <int DT>
__device__ inline uint32_t any_odd(u32x4 v) {
  return Odd<DT>::odd(v[0]) | Odd<DT>::odd(v[1]) | Odd<DT>::odd(v[2]) | Odd<DT>::odd(v[3]);
}

// v with its infinities and NaNs as 0.
template <int DT>
__device__ inline u32x4 finite_of(u32x4 v) {
#pragma unroll
  for (int d = 0; d < 4; ++d) v[d] &= ~Odd<DT>::spread(Odd<DT>::odd(v[d]));
  return v;
}

template <int DT>
__device__ inline u32x4 odd_of(u32x4 v, int kind) {
#pragma unroll
  for (int d = 0; d < 4; ++d) v[d] = Odd<DT>::is(opaque(v[d]), kind);  // (opaque: not kept for every kind)
  return v;
}

// 1 for each of eight entries whose bit is set.
template <int DT>
__device__ inline u32x4 ones_of(uint32_t bits) {
  return and_of(masks_of(bits), u32x4{Elem<DT>::ONE2, Elem<DT>::ONE2, Elem<DT>::ONE2, Elem<DT>::ONE2});
}

// A wave's TILE rows: outputs so far (unnormalised), maximum and sum.
template <int DT, int HD, int TILE>
struct Rows {
  using S = Shape<TILE>;
  static constexpr int QK = HD / S::SUMMED;   // operands of a row's head_dim
  static constexpr int NT = 32 / TILE;        // tiles of scores of 32 entries
  static constexpr int NK = 32 / S::SUMMED;   // operands of their weights
  static constexpr int DV = HD / TILE;        // tiles of outputs
  typename S::acc o[DV];
  float m, l;

  __device__ inline void clear() {
#pragma unroll
    for (int d = 0; d < DV; ++d)
#pragma unroll
      for (int r = 0; r < S::REGS; ++r) o[d][r] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }

  // Entries whose bit in `seen` (a lane's, of each 32) is off count nothing, whatever their score.
  template <int N>
  __device__ static inline void hide(typename S::acc (&s)[N * NT], const uint32_t (&seen)[N]) {
#pragma unroll
    for (int n = 0; n < N * NT; ++n)
#pragma unroll
      for (int r = 0; r < S::REGS; ++r) {
        const uint32_t on = whole(seen[n / NT], n % NT * S::REGS + r);
        const float score = s[n][r];  // (a bit cast of a vector's element takes element 0 of it)
        s[n][r] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, score) & on) | (0xff800000u & ~on));
      }
  }

  // 32 N entries: their scores as the first product leaves them to their weights, as operands of the
  // second; the maximum, the sum and the outputs so far go along. The maximum follows only where it has grown
  // by 2^8 (weights of up to 256 are as exact as any), so the outputs are seldom multiplied.
  template <int N>
  __device__ inline void weigh(typename S::acc (&s)[N * NT], u32x4 (&p)[N * NK], float c, float slack) {
    float top = -INFINITY;
#pragma unroll
    for (int n = 0; n < N * NT; ++n)
#pragma unroll
      for (int r = 0; r < S::REGS; ++r) top = fmaxf(top, s[n][r]);
    top = max_across<TILE>(top);
    if (__ballot(top > m + slack) != 0) {
      const float now = fmaxf(m, top);
      // (At the first entries outputs and sum are 0, or what add_odd has put there.)
      const float by = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - now) * c);
      l *= by;
#pragma unroll
      for (int d = 0; d < DV; ++d)
#pragma unroll
        for (int r = 0; r < S::REGS; ++r) o[d][r] *= by;
      m = now;
    }
    const float at = m == -INFINITY ? 0.f : stored_max<DT>(m, c);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < N * NT; ++n)
#pragma unroll
      for (int r = 0; r < S::REGS; ++r) {
        s[n][r] = __builtin_amdgcn_exp2f(fmaf(s[n][r], c, -at));
      }
    // Value i of a lane's 8 NK N, in the order of its registers.
    auto at_of = [&](int i) __attribute__((always_inline)) -> float { return s[i / S::REGS][i % S::REGS]; };
#pragma unroll
    for (int k = 0; k < N * NK; ++k)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        p[k][d] = pack2<DT>(at_of(8 * k + 2 * d), at_of(8 * k + 2 * d + 1));
        sum = add2<DT>(p[k][d], sum);
      }
    l += sum;
  }

  // Adds the infinities and NaNs of V to the rows that see them (and to no other, as 0 times them in
  // the product would): counted by products with ones. v(k, d): the operand of summed entries k, tile d.
  template <int N, class V>
  __device__ inline void add_odd(const uint32_t (&seen)[N], V v) {
#pragma unroll 1
    for (int kind = 0; kind < 3; ++kind) {
      const float what = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
      __asm__ volatile("" ::: "memory");  // V's operands are read again for each
#pragma unroll
      for (int d = 0; d < DV; ++d) {
        typename S::acc count;
#pragma unroll
        for (int r = 0; r < S::REGS; ++r) count[r] = 0.f;
#pragma unroll
        for (int k = 0; k < N * NK; ++k) count = mma<DT, TILE>(odd_of<DT>(v(k, d), kind), ones_of<DT>(seen[k / NK] >> (8 * (k % NK))), count);
#pragma unroll
        for (int r = 0; r < S::REGS; ++r) o[d][r] += count[r] > 0.f ? what : 0.f;
        __builtin_amdgcn_sched_barrier(0);  // few registers are free here: one after the other
      }
    }
  }
};

// Every load of this wave has landed, those into LDS too. (The builtin, which the compiler counts: after an
// asm statement it would wait for the queries again in each step, and with them for the loads after.)
__device__ inline void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// The factor that normalises a row of stored maximum m and sum l.
__device__ inline float norm_of(float m, float l, const float* sinks, int head) {
  if (l == 0.f) return 0.f;  // the row sees nothing
  if (sinks == nullptr) return 1.f / l;
  const float sink = sinks[head] * 1.44269504088896341f;
  const float top = fmaxf(m, sink);
  const float by = __builtin_amdgcn_exp2f(m - top);
  return by / (l * by + __builtin_amdgcn_exp2f(sink - top));
}

__device__ inline int64_t part_row(const AttendArgs& a, bool few, int s, const Sequence& q, int i, int head) {
  return few ? (static_cast<int64_t>(s) * a.few_tokens + i) * a.heads + head : static_cast<int64_t>(q.first + i) * a.heads + head;
}

// LDS of the few-row way: each wave's outputs for the others, and maxima and sums.
template <int HD, int TILE>
struct FewLds {
  static constexpr int OWN = HD * TILE / 64 / 4;  // a wave's share of a lane's outputs
  f32x4 others[4][3][OWN / 4][64];
  float stat[4][TILE][2];
};

// A tree's paths, depths and parents (nothing without a tree).
template <bool TREE>
struct TreeLds {
  uint32_t paths[TREE ? NODES * (NODES / 32) : 1];
  int depth[TREE ? NODES : 1], up[TREE ? NODES : 1];
};

// The few-row way: tiles of TILE rows (16, or 32 where sequences may have more) of one KV head of one
// sequence. q_tile: for its queries, [HD / SUMMED][64], where a lane has no registers left for them.
template <int DT, int HD, int TILE, bool TREE>
__device__ inline void few_rows(const AttendArgs& a, int block, FewLds<HD, TILE>& lds, u32x4* q_tile, TreeLds<TREE>& tree) {
  using R = Rows<DT, HD, TILE>;
  using S = Shape<TILE>;
  constexpr int CH = HD / 8, QK = R::QK, NT = R::NT, NK = R::NK, DV = R::DV, REGS = S::REGS, GROUPS = S::GROUPS;
  constexpr int OWN = FewLds<HD, TILE>::OWN;
  constexpr bool Q_IN_LDS = TILE * HD > 16 * 128;
  auto& others = lds.others;
  auto& stat = lds.stat;
  const Batch& b = a.batch;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = lane / TILE, col = lane % TILE;
  const int h = block % a.kv_heads, rest = block / a.kv_heads;
  const int split = rest % a.small.splits, s = rest / a.small.splits;
  const int mask = (1 << b.page_bits) - 1;
  if (s == b.sequences) {
    if (!a.fill || split != 0) return;
    const int first = clamp_to(b.starts[s], 0, b.tokens);
    const int chunks = a.group * HD / 8;
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(b.tokens - first) * chunks; i += 256)
      *reinterpret_cast<u32x4*>(a.out + (first + i / chunks) * a.out_stride + static_cast<int64_t>(h) * a.group * HD + 8 * (i % chunks)) =
          u32x4{0u, 0u, 0u, 0u};
    return;
  }
  const Sequence q = sequence_of(b, s);
  const int64_t all_rows = static_cast<int64_t>(q.n) * a.group;
  if (q.n == 0 || (all_rows > a.few && !a.every)) return;
  const int rows = static_cast<int>(all_rows);
  const int splits = q.n <= a.few_tokens ? a.small.splits : 1;
  if (split >= splits) return;
  if constexpr (TREE) paths_of(a, q, parent_of(a, q), tree.paths, tree.depth, tree.up);
  const int limit = min(q.length, capacity(b));  // entries that may be there
  const float slack = 8.f / a.scale2;

  for (int r0 = 0; r0 < rows; r0 += TILE) {
    const int i0 = r0 / a.group, i1 = (min(r0 + TILE, rows) - 1) / a.group;
    const Range range = range_of(a, q, i0, i1, splits, FEW_STEP);
    if (split >= range.used) continue;
    const int begin = range.lo + split * range.chunk, end = min(range.hi, begin + range.chunk);
    const int r = min(r0 + col, rows - 1), i = r / a.group, head = h * a.group + r % a.group;
    const Row row = row_of<TREE>(a, q, i, tree.paths, tree.depth);
    // All rows see entries sure_low .. sure_last (of a tree none where a node past the last one is among them).
    const int sure_last = TREE ? (i1 < NODES ? q.base - 1 : -1) : q.base + i0;
    const int sure_low = a.window > 0 ? q.base + (TREE ? q.n - 1 : i1) - a.window + 1 : 0;

    // A step: 32 entries from t, in one page or two. Its keys' registers take the next step's keys as
    // soon as the scores are there, its values' the next step's values after the second product.
    u32x4 kx[NT][QK], vx[NK][DV];
    // Page ids are read two steps ahead and looked at when they are used: a look as they are read would wait
    // for them, and with them for every load before.
    struct Pages {
      int low, high;  // of entries t .. + 15 and t + 16 .. + 31 (past the last entry: the last one's)
    };
    const int32_t* const table = b.tables + static_cast<int64_t>(s) * b.width;
    auto pages_at = [&](int t) __attribute__((always_inline)) -> Pages {
      return Pages{table[min(t, end - 1) >> b.page_bits], table[min(t + 16, end - 1) >> b.page_bits]};
    };
    auto good = [&](int page) __attribute__((always_inline)) -> bool { return page >= 0 && page < b.pages; };
    auto load_k = [&](Pages x, int t) __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int e = entry_of<TILE>(n, col);
        const int page = e >= 16 ? x.high : x.low;
        const int64_t kp = static_cast<int64_t>(good(page) ? page : 0) * a.kv_heads + h;
        const uint16_t* const kr = a.k_cache + (((kp * CH + group) << b.page_bits) + ((t + e) & mask)) * 8;
#pragma unroll
        for (int c = 0; c < QK; ++c) kx[n][c] = *reinterpret_cast<const u32x4*>(kr + (static_cast<int64_t>(GROUPS * c) << b.page_bits) * 8);
      }
    };
    auto load_v = [&](Pages x, int t) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const int e = 8 * (GROUPS * k + group);
        const int page = e >= 16 ? x.high : x.low;
        const int64_t vp = static_cast<int64_t>(good(page) ? page : 0) * a.kv_heads + h;
        const uint16_t* const vr = a.v_cache + (((vp << (b.page_bits - 3)) + (((t + e) & mask) >> 3)) * HD + col) * 8;
#pragma unroll
        for (int d = 0; d < DV; ++d) vx[k][d] = *reinterpret_cast<const u32x4*>(vr + TILE * 8 * d);
      }
    };

    // Steps of 32 entries, wave w's the w-th of each 128.
    int t = begin + 32 * wave;
    Pages page{-1, -1}, next = page;
    if (begin < end) {
      page = pages_at(t);
      next = pages_at(t + FEW_STEP);
    }
    u32x4 qx[Q_IN_LDS ? 1 : QK];
    const uint16_t* const qr = a.q + (q.first + i) * a.q_stride + static_cast<int64_t>(head) * HD;
    if constexpr (Q_IN_LDS) {
#pragma unroll
      for (int c = 0; c < QK / 4; ++c)
        q_tile[(4 * c + wave) * 64 + lane] = *reinterpret_cast<const u32x4*>(qr + 8 * (GROUPS * (4 * c + wave) + group));
      __syncthreads();
    } else {
#pragma unroll
      for (int c = 0; c < QK; ++c) qx[c] = *reinterpret_cast<const u32x4*>(qr + 8 * (GROUPS * c + group));
    }
    R st;
    st.clear();
    if (t < end) {
      load_k(page, t);
      load_v(page, t);
    }
    // (`more`: whether a step follows, known to the compiler, which then counts the loads in flight.)
    auto step = [&](auto more) __attribute__((always_inline)) {
      constexpr bool MORE = decltype(more)::value;
      const Pages after = pages_at(t + 2 * FEW_STEP);
      const int there = min(limit, end) - t;
      uint32_t valid = there >= 32 ? ~0u : (1u << max(there, 0)) - 1u;
      if (!good(page.low)) valid &= 0xffff0000u;
      if (!good(page.high)) valid &= 0xffffu;
      const bool sure = valid == ~0u && t + 31 <= sure_last && t >= sure_low;
      uint32_t seen[1] = {~0u};
      if (!sure) {
        // Values of entries that are not there become 0 (their weight is 0, but they may hold anything).
        seen[0] = seen_of<TREE, TILE>(row, t, valid, q.base, group);
        uint32_t odd = 0;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
          const u32x4 on = masks_of(valid >> (8 * (GROUPS * k + group)));
#pragma unroll
          for (int d = 0; d < DV; ++d) {
            vx[k][d] = and_of(vx[k][d], on);
            odd |= any_odd<DT>(vx[k][d]);
          }
        }
        if (__ballot(odd != 0) != 0) {
          st.template add_odd<1>(seen, [&](int k, int d) __attribute__((always_inline)) { return vx[k][d]; });
#pragma unroll
          for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int d = 0; d < DV; ++d) vx[k][d] = finite_of<DT>(vx[k][d]);
        }
      }
      typename S::acc sc[NT];
      if constexpr (Q_IN_LDS) __asm__ volatile("" ::: "memory");  // (read again for each step)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < REGS; ++e) sc[n][e] = 0.f;
#pragma unroll
        for (int c = 0; c < QK; ++c) sc[n] = mma<DT, TILE>(kx[n][c], Q_IN_LDS ? q_tile[Q_IN_LDS ? c * 64 + lane : 0] : qx[Q_IN_LDS ? 0 : c], sc[n]);
      }
      if constexpr (MORE) load_k(next, t + FEW_STEP);
      if (!sure) R::template hide<1>(sc, seen);
      u32x4 p[NK];
      st.template weigh<1>(sc, p, a.scale2, slack);
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int d = 0; d < DV; ++d) st.o[d] = mma<DT, TILE>(vx[k][d], p[k], st.o[d]);
      if constexpr (MORE) load_v(next, t + FEW_STEP);
      page = next;
      next = after;
    };
    for (; t + FEW_STEP < end; t += FEW_STEP) step(std::true_type{});
    if (t < end) step(std::false_type{});

    // The four waves' rows into one: each scales its outputs to the common maximum, hands each other wave the
    // registers of that one's share, and adds up its own share in the waves' order.
    const float l = sum_across<TILE>(st.l);
    const float mine = stored_max<DT>(st.m, a.scale2);
    if (group == 0) stat[wave][col][0] = mine, stat[wave][col][1] = l;
    __syncthreads();
    float m = stat[0][col][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, stat[w][col][0]);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += stat[w][col][1] * (m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(stat[w][col][0] - m));
    const float by = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mine - m);
    f32x4 own[OWN / 4];
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int g = 0; g < OWN / 4; ++g) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = st.o[(w * OWN + 4 * g + e) / REGS][(w * OWN + 4 * g + e) % REGS] * by;
        if (w == wave) own[g] = v;
        else others[w][wave - (wave > w ? 1 : 0)][g][lane] = v;
      }
    __syncthreads();
    f32x4 total[OWN / 4];
#pragma unroll
    for (int g = 0; g < OWN / 4; ++g)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const f32x4 v = w == wave ? own[g] : others[wave][max(w - (w > wave ? 1 : 0), 0)][g][lane];
        total[g] = w == 0 ? v : f32x4{total[g][0] + v[0], total[g][1] + v[1], total[g][2] + v[2], total[g][3] + v[3]};
      }
    if (r0 + col < rows) {
      // Group g of this wave's registers: four dimensions from `dim`.
      auto dim_of = [&](int g) { const int reg = wave * OWN + 4 * g; return reg / REGS * TILE + reg % REGS * GROUPS + 4 * group; };
      if (range.used == 1) {
        const float n = norm_of(m, sum, a.sinks, head);
        uint16_t* const to = a.out + (q.first + i) * a.out_stride + static_cast<int64_t>(head) * HD;
#pragma unroll
        for (int g = 0; g < OWN / 4; ++g)
          *reinterpret_cast<u32x2*>(to + dim_of(g)) = u32x2{pack2<DT>(total[g][0] * n, total[g][1] * n), pack2<DT>(total[g][2] * n, total[g][3] * n)};
      } else {
        const int64_t at = split * a.small.rows + part_row(a, true, s, q, i, head);
#pragma unroll
        for (int g = 0; g < OWN / 4; ++g) *reinterpret_cast<f32x4*>(a.small.sums + at * HD + dim_of(g)) = total[g];
        if (wave == 0 && group == 0) a.small.stats[2 * at] = m, a.small.stats[2 * at + 1] = sum;
      }
    }
    __syncthreads();  // `stat`, `others` and the queries are the next tile's
  }
}

template <int DT, int HD, int TILE, bool TREE>
__global__ __launch_bounds__(256, 2) void paged_few_kernel(AttendArgs a) {
  __shared__ FewLds<HD, TILE> lds;
  __shared__ u32x4 q_tile[HD * TILE * 2 / 16];
  __shared__ TreeLds<TREE> tree;
  few_rows<DT, HD, TILE, TREE>(a, blockIdx.x, lds, q_tile, tree);
}

__device__ inline int many_slot(const AttendArgs& a, int s) {
  return static_cast<int>(static_cast<int64_t>(clamp_to(a.batch.starts[s], 0, a.batch.tokens)) * a.group / MANY) + s;
}

// The many-row way, for the tiles of `slots` slots; past their workgroups, the sequences of few rows. WIDE:
// pages of 64 entries and more, a tile of entries in one of them, its addresses scalar ones. (A vector
// instruction costs a wave's matrix unit half its own time; those of a step that only find addresses are
// a tenth of it.) Four workgroups a CU at head_dim 64 (for a few registers' spills): 8191 tokens in a window of
// 128, 53.7 us against 60 with three.
template <int DT, int HD, bool TREE, bool WIDE>
__global__ __launch_bounds__(256, HD == 64 && !TREE ? 4 : 2) void paged_many_kernel(AttendArgs a, int slots) {
  using R = Rows<DT, HD, 32>;
  constexpr int CH = HD / 8, QK = R::QK, DV = R::DV;
  constexpr int UNITS = HD * MANY_STEP / 8;  // 16-byte units of K's tile, and of V's
  // Two tiles, K: [CH][64 entries] and V: [8 eights of entries][HD]. (Two arrays: of one, the compiler
  // has every read wait for the loads in flight into the other half.)
  __shared__ u32x4 tile0[2 * UNITS], tile1[2 * UNITS];
  __shared__ TreeLds<TREE> tree;
  __shared__ uint32_t odd_waves[4];
  const int tiles = slots * a.kv_heads * a.large.splits;
  if (static_cast<int>(blockIdx.x) >= tiles) {
    static_assert(sizeof(FewLds<HD, 16>) <= sizeof(tile0), "the few-row way's LDS");
    few_rows<DT, HD, 16, TREE>(a, blockIdx.x - tiles, *reinterpret_cast<FewLds<HD, 16>*>(tile0), tile1, tree);
    return;
  }
  const Batch& b = a.batch;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int h = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
  // The last tiles first: of a prompt they see the most.
  const int split = rest % a.large.splits, slot = slots - 1 - rest / a.large.splits;
  const int s = find_sequence(b.sequences, slot, [&](int i) { return many_slot(a, i); });
  const Sequence q = sequence_of(b, s);
  const int rows = static_cast<int>(static_cast<int64_t>(q.n) * a.group);
  const int local = slot - many_slot(a, s);
  if (rows <= a.few || local < 0 || local >= (rows + MANY - 1) / MANY) return;
  const int r0 = local * MANY;
  const int i0 = r0 / a.group, i1 = (min(r0 + MANY, rows) - 1) / a.group;
  const Range range = range_of(a, q, i0, i1, a.large.splits, MANY_STEP);
  if (split >= range.used) return;
  const int begin = range.lo + split * range.chunk, end = min(range.hi, begin + range.chunk);
  const int limit = min(min(q.length, capacity(b)), end);
  const int mask = (1 << b.page_bits) - 1;
  const float slack = 8.f / a.scale2;

  // This wave's rows, and what all of them and what any of them see (of the workgroup's rows, too); nodes of a tree
  // past the last one see nothing.
  const int w0 = r0 + 32 * wave;
  const bool busy = w0 < rows;
  const int r = min(w0 + col, rows - 1), i = r / a.group, head = h * a.group + r % a.group;
  const int wa = min(w0, rows - 1) / a.group, wz = min(w0 + 31, rows - 1) / a.group;
  const int sure_last = TREE ? (wz < NODES ? q.base - 1 : -1) : q.base + wa, sure_low = a.window > 0 ? q.base + (TREE ? q.n - 1 : wz) - a.window + 1 : 0;
  const int any_last = TREE ? q.length - 1 : q.base + wz, any_low = a.window > 0 ? q.base + (TREE ? 0 : wa) - a.window + 1 : 0;
  const int all_last = TREE ? (i1 < NODES ? q.base - 1 : -1) : q.base + i0, all_low = a.window > 0 ? q.base + (TREE ? q.n - 1 : i1) - a.window + 1 : 0;

  R st;
  st.clear();
  u32x4 qx[QK];
  const uint16_t* const qr = a.q + (q.first + i) * a.q_stride + static_cast<int64_t>(head) * HD;
#pragma unroll
  for (int c = 0; c < QK; ++c) qx[c] = *reinterpret_cast<const u32x4*>(qr + 16 * c + 8 * half);

  // A tile's loads: lane l has the page id of entry t + l, read two tiles ahead and looked at when it is
  // used. K goes eight dimensions of 64 entries an instruction, V 64 dimensions of eight entries.
  const int32_t* const table = b.tables + static_cast<int64_t>(s) * b.width;
  auto page_at = [&](int t) __attribute__((always_inline)) -> int { return table[min(t + lane, end - 1) >> b.page_bits]; };
  auto good = [&](int page) __attribute__((always_inline)) -> bool { return page >= 0 && page < b.pages; };
  struct Source {
    const uint16_t* k;  // dimensions 0 .. 7 of the tile's first entry, or with !WIDE of this lane's
    int page;           // of the tile, or of this lane's entry
    int t;
  };
  auto source_of = [&](int id, int t) __attribute__((always_inline)) -> Source {
    if constexpr (WIDE) id = __builtin_amdgcn_readfirstlane(id);
    const int page = good(id) ? id : 0;
    const int64_t kp = static_cast<int64_t>(page) * a.kv_heads + h;
    return Source{a.k_cache + ((kp * CH << b.page_bits) + ((WIDE ? t : t + lane) & mask)) * 8, page, t};
  };
  auto to_lds = [&](const uint16_t* from, int at, u32x4* to) __attribute__((always_inline)) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(reinterpret_cast<const char*>(from) + static_cast<uint32_t>(at)),
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  // Load i of this wave's LOADS of a tile.
  constexpr int K_LOADS = CH / 4, LOADS = 2 * K_LOADS;
  auto load_one = [&](const Source& x, u32x4* to, int i) __attribute__((always_inline)) {
    if (i < K_LOADS) {
      const int c = wave * K_LOADS + i;
      to_lds(x.k + (static_cast<int64_t>(c) << b.page_bits) * 8, WIDE ? lane * 16 : 0, to + c * 64);
    } else {
      const int part = wave * K_LOADS + i - K_LOADS;
      const int e8 = part / (HD / 64), d = part % (HD / 64);  // the eight entries 8 e8 .., 64 dimensions
      const int64_t vp = static_cast<int64_t>(WIDE ? x.page : __builtin_amdgcn_readlane(x.page, 8 * e8)) * a.kv_heads + h;
      to_lds(a.v_cache + (((vp << (b.page_bits - 3)) + (((x.t + 8 * e8) & mask) >> 3)) * HD + 64 * d) * 8, lane * 16,
             to + UNITS + e8 * HD + 64 * d);
    }
  };
  // The entries of the tile at t that are there.
  auto there_of = [&](int id, int t) __attribute__((always_inline)) -> uint64_t {
    if constexpr (!WIDE) return __ballot(t + lane < limit && good(id));
    const int many = limit - t;
    return !good(__builtin_amdgcn_readfirstlane(id)) || many <= 0 ? 0 : many >= 64 ? ~0ull : (1ull << many) - 1;
  };

  const int entry = entry_of<32>(0, col);
  int id = -1, next = -1, parent = -1;
  // (Without a window, a part that ends before the draft needs no paths.)
  const bool nodes = TREE && (a.window > 0 || end > q.base);
  if (nodes) parent = parent_of(a, q);
  if (begin < end) {
    id = page_at(begin);
    next = page_at(begin + MANY_STEP);
    const Source first = source_of(id, begin);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load_one(first, tile0, i);
  }
  if constexpr (TREE) {
    if (nodes) paths_of(a, q, parent, tree.paths, tree.depth, tree.up);
  }
  const Row row = row_of<TREE>(a, q, i, tree.paths, tree.depth);
  loads_done();
  lds_barrier();
  auto step = [&](int t, u32x4* cur, u32x4* other) __attribute__((always_inline)) {
    const uint64_t valid = there_of(id, t);
    id = next;
    next = page_at(t + 2 * MANY_STEP);
    const Source source = source_of(id, t + MANY_STEP);
    u32x4* const kt = cur;
    u32x4* const vt = cur + UNITS;
    // Where some row does not see all of the tile, V's entries that are not there become 0 (their
    // weight is 0, but they may hold anything), and its infinities and NaNs are looked for. (All there: looked for only.
    // A window of 128 over 8191 tokens at head_dim 64, 56.5 us against 57.8.)
    uint32_t odd = 0;
    if (valid != ~0ull || t + 63 > all_last || t < all_low) {
      uint32_t found = 0;
      if (valid == ~0ull) {
#pragma unroll
        for (int n = 0; n < UNITS / 256; ++n) found |= any_odd<DT>(vt[n * 256 + tid]);
      } else {
#pragma unroll
        for (int n = 0; n < UNITS / 256; ++n) {
          const int u = n * 256 + tid;
          const uint32_t there = static_cast<uint32_t>(valid >> (8 * (u / HD))) & 0xffu;
          const u32x4 v = and_of(vt[u], masks_of(there));
          found |= any_odd<DT>(v);
          if (there != 0xffu) vt[u] = v;
        }
      }
      const uint64_t lanes = __ballot(found != 0);
      if (lane == 0) odd_waves[wave] = lanes != 0 ? 1u : 0u;
      lds_barrier();
      odd = odd_waves[0] | odd_waves[1] | odd_waves[2] | odd_waves[3];
    }
    const bool takes = busy && t <= any_last && t + 63 >= any_low && valid != 0;
    const bool sure = valid == ~0ull && t + 63 <= sure_last && t >= sure_low;
    uint32_t seen[2];
    auto look = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int n = 0; n < 2; ++n) seen[n] = seen_of<TREE, 32>(row, t + 32 * n, static_cast<uint32_t>(valid >> (32 * n)), q.base, half);
    };
    auto v_of = [&](int k, int d) __attribute__((always_inline)) -> u32x4 { return vt[(2 * k + half) * HD + 32 * d + col]; };
    if (odd != 0) {
      if (takes) {
        look();
        st.template add_odd<2>(seen, v_of);
      }
      lds_barrier();
#pragma unroll
      for (int n = 0; n < UNITS / 256; ++n) vt[n * 256 + tid] = finite_of<DT>(vt[n * 256 + tid]);
      lds_barrier();
    }
    if (takes) {
      f32x16 sc[2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[n][e] = 0.f;
      // The next tile's loads go out between these products (past the last tile the last one's again, into
      // the buffer that is not read): the CU takes 64 bytes of them a cycle, and a wave waits to issue the next.
#pragma unroll
      for (int c = 0; c < QK; ++c) {
#pragma unroll
        for (int n = 0; n < 2; ++n) sc[n] = mma<DT, 32>(kt[(2 * c + half) * 64 + 32 * n + entry], qx[c], sc[n]);
        load_one(source, other, c);
      }
      if (!sure) {
        look();
        R::template hide<2>(sc, seen);
      }
      u32x4 p[4];
      st.template weigh<2>(sc, p, a.scale2, slack);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int d = 0; d < DV; ++d) st.o[d] = mma<DT, 32>(v_of(k, d), p[k], st.o[d]);
    }
    if (!takes) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) load_one(source, other, i);
    }
    loads_done();
    lds_barrier();
  };
  for (int t = begin; t < end; t += 2 * MANY_STEP) {
    step(t, tile0, tile1);
    if (t + MANY_STEP < end) step(t + MANY_STEP, tile1, tile0);
  }

  if (w0 + col >= rows) return;
  const float l = sum_across<32>(st.l);
  const float m = stored_max<DT>(st.m, a.scale2);
  if (range.used == 1) {
    const float n = norm_of(m, l, a.sinks, head);
    uint16_t* const to = a.out + (q.first + i) * a.out_stride + static_cast<int64_t>(head) * HD;
#pragma unroll
    for (int d = 0; d < DV; ++d)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        // Register group g of both halves: the halves trade, so that each stores eight dimensions together.
        uint32_t x[2], y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[e] = pack2<DT>(st.o[d][4 * g + 2 * e] * n, st.o[d][4 * g + 2 * e + 1] * n);
          y[e] = pack2<DT>(st.o[d][4 * g + 4 + 2 * e] * n, st.o[d][4 * g + 5 + 2 * e] * n);
          const auto t = __builtin_amdgcn_permlane32_swap(x[e], y[e], false, false);
          x[e] = t[0], y[e] = t[1];
        }
        *reinterpret_cast<u32x4*>(to + 32 * d + 8 * (g + half)) = u32x4{x[0], x[1], y[0], y[1]};
      }
  } else {
    const int64_t at = split * a.large.rows + part_row(a, false, s, q, i, head);
#pragma unroll
    for (int d = 0; d < DV; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(a.large.sums + at * HD + 32 * d + 8 * g + 4 * half) =
            f32x4{st.o[d][4 * g], st.o[d][4 * g + 1], st.o[d][4 * g + 2], st.o[d][4 * g + 3]};
    if (half == 0) a.large.stats[2 * at] = m, a.large.stats[2 * at + 1] = l;
  }
}

// A token whose rows may be in parts: of `small` the i-th new one of a few-row sequence, else one of the batch;
// n == 0 where it is none.
struct Joined {
  Sequence q;
  int s, i;
};

__device__ inline Joined joined_of(const AttendArgs& a, bool small, int at) {
  const Batch& b = a.batch;
  Joined j;
  j.s = small ? at / a.few_tokens : find_sequence(b.sequences, at, [&](int n) { return clamp_to(b.starts[n], 0, b.tokens); });
  j.q = sequence_of(b, j.s);
  j.i = small ? at % a.few_tokens : at - j.q.first;
  const bool few = static_cast<int64_t>(j.q.n) * a.group <= a.few || a.every;
  if (j.i < 0 || j.i >= j.q.n || few != small || (small && j.q.n > a.few_tokens)) j.q.n = 0;
  return j;
}

// The parts of head `head` of it, as its tile was computed.
__device__ inline Range parts_of(const AttendArgs& a, bool small, const Joined& j, int head) {
  const int per = small ? a.few_tile : MANY;
  const int64_t rows = static_cast<int64_t>(j.q.n) * a.group;
  const int64_t r0 = (static_cast<int64_t>(j.i) * a.group + head % a.group) / per * per;
  return range_of(a, j.q, static_cast<int>(r0 / a.group), static_cast<int>((min(r0 + per, rows) - 1) / a.group),
                  small ? a.small.splits : a.large.splits, small ? FEW_STEP : MANY_STEP);
}

// The parts of rows added in order: HEADS (1 or 4) heads of a token to a wave, up to 64 / HEADS parts of each. Lane
// PARTS r + c has part c of head r's maximum and sum; then every lane adds its dimensions of all.
template <int DT, int HD, int HEADS>
__global__ __launch_bounds__(256) void paged_join_kernel(AttendArgs a, int64_t small_tokens, int64_t tokens) {
  constexpr int PARTS = 64 / HEADS;
  constexpr int D = HD / 64;         // dimensions a lane
  constexpr int AHEAD = 16 / HEADS;  // parts of a head loaded together
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int blocks = (a.heads + HEADS - 1) / HEADS;
  const int64_t at_block = blockIdx.x * int64_t{4} + wave;
  if (at_block >= tokens * blocks) return;
  const int64_t token = at_block / blocks;
  const bool small = token < small_tokens;
  const Parts& part = small ? a.small : a.large;
  const int head0 = static_cast<int>(at_block % blocks) * HEADS;
  const int head = head0 + lane / PARTS, c = lane % PARTS;
  const int64_t at0 = (small ? token : token - small_tokens) * a.heads + head0;  // (part_row)
  // Read before the batch says which of the parts are there: a wave waits once, not twice.
  const float* const st = part.stats + 2 * (min(c, part.splits - 1) * part.rows + min(at0 + lane / PARTS, part.rows - 1));
  const float m_read = st[0], l_read = st[1];
  const Joined j = joined_of(a, small, static_cast<int>(small ? token : token - small_tokens));
  if (j.q.n == 0) return;
  const int used = head < a.heads ? parts_of(a, small, j, head).used : 1;
  const int most = static_cast<int>(wave_max(static_cast<float>(used)));
  if (most == 1) return;
  float m = -INFINITY, l = 0.f;
  if (head < a.heads && c < used && used > 1) m = m_read, l = l_read;
  float top = m;
#pragma unroll
  for (int off = 1; off < PARTS; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  const float w = c >= used ? 0.f : m == -INFINITY ? (top == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(m - top);
  l *= w;
#pragma unroll
  for (int off = 1; off < PARTS; off <<= 1) l += __shfl_xor(l, off, 64);
  const float n = norm_of(top, l, a.sinks, min(head, a.heads - 1));
  float o[HEADS][D] = {};
  for (int c0 = 0; c0 < most; c0 += AHEAD) {
    float x[HEADS][AHEAD][D];
#pragma unroll
    for (int r = 0; r < HEADS; ++r)
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        // (Past the last part or head: read again, and not used.)
        const int64_t at = at0 + min(r, a.heads - 1 - head0) + min(c0 + e, most - 1) * part.rows;
#pragma unroll
        for (int d = 0; d < D; ++d) x[r][e][d] = part.sums[at * HD + lane * D + d];
      }
#pragma unroll
    for (int r = 0; r < HEADS; ++r)
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const int lane_of = PARTS * r + min(c0 + e, PARTS - 1);
        const float by = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), lane_of));
        // (A part whose weight is 0 is added too: a row that sees an infinity or a NaN in it is no number.)
        const bool there = c0 + e < __builtin_amdgcn_readlane(used, PARTS * r);
#pragma unroll
        for (int d = 0; d < D; ++d) o[r][d] += there ? by * x[r][e][d] : 0.f;
      }
  }
#pragma unroll
  for (int r = 0; r < HEADS; ++r) {
    if (head0 + r >= a.heads || __builtin_amdgcn_readlane(used, PARTS * r) == 1) continue;
    const float by = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, n), PARTS * r));
    uint16_t* const to = a.out + (j.q.first + j.i) * a.out_stride + static_cast<int64_t>(head0 + r) * HD + lane * D;
    if constexpr (D == 2) *reinterpret_cast<uint32_t*>(to) = pack2<DT>(o[r][0] * by, o[r][D - 1] * by);
    else *to = static_cast<uint16_t>(pack2<DT>(o[r][0] * by, 0.f));
  }
}

// The same of any number of parts: a row to a workgroup, whose waves take the parts in turn.
template <int DT, int HD>
__global__ __launch_bounds__(256) void paged_join_wide_kernel(AttendArgs a, int64_t small_tokens, int64_t tokens) {
  constexpr int D = HD / 64, AHEAD = 8;
  __shared__ float weights[MAX_SPLITS];
  __shared__ float sums[3][HD];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = blockIdx.x / a.heads;
  const int head = blockIdx.x % a.heads;
  if (token >= tokens) return;
  const bool small = token < small_tokens;
  const Parts& part = small ? a.small : a.large;
  const int64_t at = (small ? token : token - small_tokens) * a.heads + head;  // (part_row)
  // Statistics and, of few rows (of many it could be traffic for nothing), the first parts are read before the batch
  // says which of them are there: a wave waits once, not three times.
  constexpr int STATS = MAX_SPLITS / 64;
  float ms[STATS], ls[STATS];
#pragma unroll
  for (int n = 0; n < STATS; ++n) {
    const float* const st = part.stats + 2 * (min(lane + 64 * n, part.splits - 1) * part.rows + at);
    ms[n] = st[0], ls[n] = st[1];
  }
  const float* const from = part.sums + at * HD + lane * D;
  float x[AHEAD][D];
  auto load = [&](int c0, int last) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      const int c = min(c0 + 4 * n, last);  // (past the last: read again, and not used)
#pragma unroll
      for (int d = 0; d < D; ++d) x[n][d] = from[c * part.rows * HD + d];
    }
  };
  const bool early = gridDim.x <= 256;
  if (early) load(wave, part.splits - 1);
  const Joined j = joined_of(a, small, static_cast<int>(small ? token : token - small_tokens));
  if (j.q.n == 0) return;
  const int used = parts_of(a, small, j, head).used;
  if (used == 1) return;
  if (!early) load(wave, used - 1);
  float m = -INFINITY;
#pragma unroll
  for (int n = 0; n < STATS; ++n) m = fmaxf(m, lane + 64 * n < used ? ms[n] : -INFINITY);
  m = wave_max(m);
  float l = 0.f;
#pragma unroll
  for (int n = 0; n < STATS; ++n) {
    const int c = lane + 64 * n;
    const float w = ms[n] == -INFINITY ? (m == -INFINITY ? 1.f : 0.f) : __builtin_amdgcn_exp2f(ms[n] - m);
    if (c < used) l = fmaf(ls[n], w, l);
    if (wave == 0 && c < used) weights[c] = w;
  }
  l = wave_sum(l);
  __syncthreads();
  float o[D] = {};
  for (int c0 = wave; c0 < used; c0 += 4 * AHEAD) {
    if (c0 != wave) load(c0, used - 1);
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      const int c = c0 + 4 * n;
      const float w = weights[min(c, used - 1)];
#pragma unroll
      for (int d = 0; d < D; ++d) o[d] += c < used ? w * x[n][d] : 0.f;  // (parts of weight 0 too, as above)
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int d = 0; d < D; ++d) sums[wave - 1][lane * D + d] = o[d];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int n = 0; n < 3; ++n)
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] += sums[n][lane * D + d];
  const float n = norm_of(m, l, a.sinks, head);
  uint16_t* const to = a.out + (j.q.first + j.i) * a.out_stride + static_cast<int64_t>(head) * HD + lane * D;
  if constexpr (D == 2) *reinterpret_cast<uint32_t*>(to) = pack2<DT>(o[0] * n, o[D - 1] * n);
  else *to = static_cast<uint16_t>(pack2<DT>(o[0] * n, 0.f));
}

// ------------------------------------------------------------------ the host's side

// What a call launches: `few` alone where no sequence has more rows, else both; the splits of either,
// and where their parts lie in the workspace (f32).
struct Plan {
  bool many;
  int few, few_tile;
  int64_t few_tokens, few_splits, many_splits, slots, few_rows, many_rows;
  int64_t few_floats, floats;
};

inline int64_t up_to(int64_t v, int64_t by) { return (v + by - 1) / by; }

static Plan plan_of(int64_t sequences, int64_t width, int64_t page, int64_t tokens, int64_t heads, int64_t kv_heads,
                    int64_t head_dim, int64_t most, int64_t window) {
  Plan p{};
  const int64_t group = heads / kv_heads;
  most = most > tokens ? tokens : most;
  most = most < 1 ? 1 : most;
  // (Without sequences there are no rows but those of no sequence, which the few-row kernel clears.)
  p.many = sequences > 0 && most * group > FEW;
  p.few = p.many ? 16 : FEW;
  p.few_tokens = p.few / group < 1 ? 1 : p.few / group;
  if (!p.many && most < p.few_tokens) p.few_tokens = most;
  p.few_tile = p.many || p.few_tokens * group <= 16 ? 16 : 32;
  // Entries that a tile of `queries` tokens may see, at most.
  auto seen_by = [&](int64_t queries) {
    const int64_t all = width * page, near = window + queries + FEW_STEP;
    return window > 0 && near < all ? near : all;
  };
  auto bounded = [](int64_t v, int64_t hi) {
    v = v > hi ? hi : v;
    return v < 1 ? int64_t{1} : v;
  };
  {
    // As many workgroups as the chip holds at once (3 a CU at head_dim 64, 2 at 128), and none of much over 1024
    // entries where lengths differ. One row of 131000 entries at head_dim 64: 57.0 us with 768 workgroups, 59.9 with
    // 512 or 1024, 62.3 with 2048; 64 rows of 230000 at 128: 180.6 with parts of 1024, 183.4 of 2048, 184.5 of 512.
    // (By what the tables can hold. Under tables much wider than the lengths parts are shorter, at least FEW_STEP: 64 sequences of
    // 1800 to 5400 entries under 131072 each 291 to 303 us, under 5440 each 172.)
    const int64_t base = sequences * kv_heads, seen = seen_by(p.few_tokens);
    int64_t want = up_to(head_dim == 64 ? 768 : 512, base > 0 ? base : 1);
    if (want < up_to(seen, 1024)) want = up_to(seen, 1024);
    // Parts cost a second kernel, of the GPU's time and of the host's. In a graph, 8 KV heads of 250 entries take 5.9 us whole
    // and 9.2 in parts, of 500 7.4 and 9.3, of 1000 10.0 and 9.1 (launched one by one 10.1 and 12.8); 64 of 375 to 750
    // 10.4 and 11.6; 512 of 1000 47.6 and 55.8.
    if (seen <= (base < 64 ? 1024 : 1280)) want = 1;
    const int64_t top = up_to(seen, FEW_STEP);
    p.few_splits = bounded(want, top < MAX_SPLITS ? top : MAX_SPLITS);
  }
  if (sequences == 0 || (p.many && group > p.few)) p.few_splits = 1;  // (no sequence has so few rows)
  p.many_splits = 1;
  if (p.many) {
    p.slots = tokens * group / MANY + sequences;
    const int64_t base = p.slots * kv_heads;
    // Twice what the chip holds at once, as the tiles differ: 16 trees of 900 nodes 131 us with 1024 (or 768), 149 with 512;
    // one of 24 over 1000 entries 14.5 with parts of 64 entries, 17.0 of 256.
    const int64_t top = up_to(seen_by(most), MANY_STEP);
    p.many_splits = bounded(up_to(1024, base > 0 ? base : 1), top < 64 ? top : 64);
  }
  p.many_rows = p.many_splits > 1 ? tokens * heads : 0;
  const int64_t many_floats = p.many_rows * p.many_splits * (head_dim + 2);  // (below 2^26: rows that are few for the chip)
  const int64_t one_part = sequences * p.few_tokens * heads * (head_dim + 2);
  if (p.few_splits * one_part > MOST_FLOATS - 4 - many_floats) p.few_splits = bounded((MOST_FLOATS - 4 - many_floats) / one_part, MAX_SPLITS);
  p.few_rows = p.few_splits > 1 ? sequences * p.few_tokens * heads : 0;
  p.few_floats = (p.few_rows * p.few_splits * (head_dim + 2) + 3) / 4 * 4;
  p.floats = p.few_floats + many_floats;
  return p;
}

template <int DT, int HD, bool TREE>
static LnqStatus attend(AttendArgs a, const Plan& p, float* work, hipStream_t st) {
  const int64_t sequences = a.batch.sequences;
  const dim3 block(256);
  a.small = {work, work + p.few_rows * p.few_splits * HD, p.few_rows, static_cast<int>(p.few_splits)};
  float* const more = work + p.few_floats;
  a.large = {more, more + p.many_rows * p.many_splits * HD, p.many_rows, static_cast<int>(p.many_splits)};
  a.every = !p.many;
  a.few = p.few, a.few_tile = p.few_tile;
  a.few_tokens = static_cast<int>(p.few_tokens);
  const int64_t few = (sequences + (a.fill ? 1 : 0)) * a.kv_heads * p.few_splits;
  if (p.many) {
    const int64_t tiles = p.slots * a.kv_heads * p.many_splits;
    const dim3 grid(static_cast<unsigned>(tiles + few));
    if (tiles + few > 0 && a.batch.page_bits >= 6)
      hipLaunchKernelGGL((paged_many_kernel<DT, HD, TREE, true>), grid, block, 0, st, a, static_cast<int>(p.slots));
    else if (tiles + few > 0)
      hipLaunchKernelGGL((paged_many_kernel<DT, HD, TREE, false>), grid, block, 0, st, a, static_cast<int>(p.slots));
  } else if (few > 0) {
    const dim3 grid(static_cast<unsigned>(few));
    if (p.few_tile == 16) hipLaunchKernelGGL((paged_few_kernel<DT, HD, 16, TREE>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_few_kernel<DT, HD, 32, TREE>), grid, block, 0, st, a);
  }
  const int64_t small = p.few_splits > 1 ? sequences * p.few_tokens : 0, joined = small + (p.many_splits > 1 ? a.batch.tokens : 0);
  if (joined > 0) {
    const int64_t parts = p.few_splits > p.many_splits ? p.few_splits : p.many_splits, rows = joined * a.heads;
    // 28800 rows of 3 parts: 13 us at four heads a wave, 30 at a row a wave, 75 at a row a workgroup; 768 of 16: 6.9, 4.2 and
    // 7.2; 32 of 8: 4.6, 4.9 at a row a wave, 4.6.
    if (rows > 2048 && parts <= 16)
      hipLaunchKernelGGL((paged_join_kernel<DT, HD, 4>), dim3(static_cast<unsigned>(up_to(joined * up_to(a.heads, 4), 4))), block, 0, st, a, small, joined);
    else if (rows > 256 && parts <= 64)
      hipLaunchKernelGGL((paged_join_kernel<DT, HD, 1>), dim3(static_cast<unsigned>(up_to(rows, 4))), block, 0, st, a, small, joined);
    else
      hipLaunchKernelGGL((paged_join_wide_kernel<DT, HD>), dim3(static_cast<unsigned>(rows)), block, 0, st, a, small, joined);
  }
  return launched("paged_attention");
}

}  // namespace paged
}  // namespace lnq

using namespace lnq;

// The sizes that both entry points take; an empty message if they go.
static const char* sizes_refused(int64_t sequences, int64_t width, int64_t pages, int64_t page, int64_t tokens, int64_t heads,
                                 int64_t kv_heads, int64_t head_dim, int64_t most, int64_t window) {
  const char* const no = paged::refused({sequences, width, pages, page, tokens});
  if (no != nullptr) return no;
  if (head_dim != 64 && head_dim != 128) return "head_dim is 64 or 128";
  if (kv_heads < 1 || kv_heads > 65536 || heads < 1 || heads > 65536 || heads % kv_heads != 0) return "heads are a multiple of kv_heads (at most 65536)";
  if (most < 0) return "a negative number of queries";
  if (window < 0 || window > (1 << 30)) return "a window is 0 (none) to 2^30 entries";
  if (tokens * heads > INT32_MAX || sequences * heads * 32 > INT32_MAX) return "too many tokens, sequences or heads";
  const paged::Plan p = paged::plan_of(sequences, width, page, tokens, heads, kv_heads, head_dim, most, window);
  // (A join takes a workgroup a row where there are more than 64 parts, and one for four rows otherwise.)
  const int64_t parts = p.few_splits > p.many_splits ? p.few_splits : p.many_splits;
  if ((sequences + 1) * kv_heads * p.few_splits + p.slots * kv_heads * p.many_splits > paged::MOST_WORKGROUPS ||
      (p.few_rows + p.many_rows) / (parts > 64 ? 1 : 4) >= paged::MOST_WORKGROUPS)
    return "too many tokens, sequences or heads";
  return nullptr;
}

extern "C" {

LNQ_API LnqStatus lnq_paged_attention_workspace(int64_t sequences, int64_t width, int64_t page, int64_t tokens, int64_t heads,
                                                int64_t kv_heads, int64_t head_dim, int64_t max_queries, int64_t window,
                                                int64_t* floats) {
  const char* const no = sizes_refused(sequences, width, 0, page, tokens, heads, kv_heads, head_dim, max_queries, window);
  LNQ_REQUIRE(no == nullptr, "lnq_paged_attention_workspace: %s", no);
  LNQ_REQUIRE(floats != nullptr, "lnq_paged_attention_workspace: null pointer");
  *floats = paged::plan_of(sequences, width, page, tokens, heads, kv_heads, head_dim, max_queries, window).floats;
  clear_error();
  return LNQ_OK;
}

LNQ_API LnqStatus lnq_paged_attention(const void* q, int64_t q_stride, const void* k_cache, const void* v_cache, void* out,
                                      int64_t out_stride, int32_t fill, const int32_t* tables, const int32_t* lengths,
                                      const int32_t* starts, const int32_t* parents, const float* sinks, float* workspace,
                                      int64_t workspace_floats, int64_t sequences, int64_t width, int64_t pages, int64_t page,
                                      int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_queries,
                                      int64_t window, float scale, int32_t dtype, void* stream) {
  const char* const no = sizes_refused(sequences, width, pages, page, tokens, heads, kv_heads, head_dim, max_queries, window);
  LNQ_REQUIRE(no == nullptr, "lnq_paged_attention: %s", no);
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16, "lnq_paged_attention: dtype %d is not bf16 or f16", dtype);
  LNQ_REQUIRE(scale >= 1e-9f && scale <= 1e9f, "lnq_paged_attention: the scale is a positive number, not %g", static_cast<double>(scale));
  if (tokens == 0) {
    clear_error();
    return LNQ_OK;
  }
  const paged::Plan p = paged::plan_of(sequences, width, page, tokens, heads, kv_heads, head_dim, max_queries, window);
  LNQ_REQUIRE(workspace_floats >= p.floats && (workspace != nullptr || p.floats == 0),
              "lnq_paged_attention: a workspace of %lld floats, %lld needed", (long long)workspace_floats, (long long)p.floats);
  LNQ_REQUIRE(q && out && starts && (lengths || sequences == 0) && (tables || width == 0 || sequences == 0) && ((k_cache && v_cache) || pages == 0),
              "lnq_paged_attention: null pointer");
  LNQ_REQUIRE(aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16) && aligned(workspace, 16) &&
                  q_stride % 8 == 0 && out_stride % 8 == 0,
              "lnq_paged_attention: operands must be 16-byte aligned, strides whole 16 bytes");
  LNQ_REQUIRE(tokens == 1 || (q_stride >= heads * head_dim && out_stride >= heads * head_dim),
              "lnq_paged_attention: a row stride is shorter than a row");
  paged::AttendArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k_cache = static_cast<const uint16_t*>(k_cache);
  a.v_cache = static_cast<const uint16_t*>(v_cache);
  a.out = static_cast<uint16_t*>(out);
  a.q_stride = q_stride, a.out_stride = out_stride;
  a.sinks = sinks;
  a.parents = parents;
  a.batch = {tables, lengths, starts, static_cast<int>(sequences), static_cast<int>(width), static_cast<int>(pages),
             paged::bits_of(page), static_cast<int>(tokens)};
  a.heads = static_cast<int>(heads), a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(heads / kv_heads);
  a.window = static_cast<int>(window);
  a.scale2 = scale * 1.44269504088896341f;
  a.fill = fill != 0;
  const auto st = static_cast<hipStream_t>(stream);
#define LNQ_ATTEND(DT_, HD_) \
  (parents != nullptr ? paged::attend<DT_, HD_, true>(a, p, workspace, st) : paged::attend<DT_, HD_, false>(a, p, workspace, st))
  if (dtype == LNQ_BF16) return head_dim == 128 ? LNQ_ATTEND(LNQ_BF16, 128) : LNQ_ATTEND(LNQ_BF16, 64);
  return head_dim == 128 ? LNQ_ATTEND(LNQ_F16, 128) : LNQ_ATTEND(LNQ_F16, 64);
#undef LNQ_ATTEND
}

}  // extern "C"
