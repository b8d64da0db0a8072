// New tokens into a KV cache in pages, and an accepted path of drafted ones to its place.
//
// append: per token and head of q and k, y = x * rsqrt(mean(x^2) + eps) * w (where there are
// norms), then the pairs (i, i + r) of the first 2 r dimensions by the angle of the token's
// position, y'_i = y_i cos_i - y_(i+r) sin_i, y'_(i+r) = y_(i+r) cos_i + y_i sin_i, in f32 and
// rounded once; k and v into the cache, q out. Bound by memory: each value is read once and
// written once.
//
// Eight entries at an aligned place of a sequence are the unit, as V's layout keeps eight entries
// of a dimension together: one wave takes one head of one unit. Of q and k a lane holds one or two times 8
// dimensions of a token (16 bytes; the other of a pair is its own or comes from the lane that holds it), of v a
// lane holds two dimensions of all eight tokens, so that V's 16-byte pieces come out of registers by
// v_perm. A whole unit is written in whole lines, a partial one (a single token of a decode step)
// by its entries alone. 8191 tokens of 32 + 8 + 8 heads of 128 (202 MB): 41 us, 4.9 TB/s (58 with 16 lanes a token of K,
// which writes half lines); one token 3.1 in a graph, a launch and four dependent loads.
#include "paged.hpp"

namespace lnq {
namespace paged {

struct AppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const float *cos, *sin;     // [positions, half]
  const int32_t* positions;   // [tokens], or nullptr: the entries
  const float *q_norm, *k_norm;
  uint16_t *q_out, *k_cache, *v_cache;
  int64_t q_out_stride;
  Batch batch;
  int heads, kv_heads, half, table, groups;
  float eps;
  bool fill;                  // q_out's rows past the last sequence become zeros
};

constexpr int UNIT = 8;
constexpr int WAVES = 4;

__device__ inline int append_slot(const Batch& b, int s) { return clamp_to(b.starts[s], 0, b.tokens) / UNIT + 2 * s; }

template <int DT, int HD, int HEADS>
__global__ __launch_bounds__(64 * WAVES) void paged_append_kernel(AppendArgs a) {
  using E = Elem<DT>;
  constexpr int CH = HD / 8;  // 16-byte chunks a head
  const Batch& b = a.batch;
  const int slot = blockIdx.x / a.groups;
  // The wave's work: HEADS heads of q's and k's, one after the other, or past those one of v's.
  const int task = (blockIdx.x % a.groups) * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int turned_heads = a.heads + a.kv_heads, turned_tasks = (turned_heads + HEADS - 1) / HEADS;
  const int lane = threadIdx.x & 63;
  // The sequences, and after them the tokens that belong to none.
  const int s = find_sequence(b.sequences + 1, slot, [&](int i) { return append_slot(b, i); });
  if (task >= turned_tasks + a.kv_heads) return;
  const int local = slot - append_slot(b, s);
  if (local < 0) return;
  if (s == b.sequences) {
    const int first = clamp_to(b.starts[s], 0, b.tokens) + local * UNIT;
    if (!a.fill || first + lane / 8 >= b.tokens) return;
    for (int head = task * HEADS; head < min((task + 1) * HEADS, a.heads); ++head)
#pragma unroll
      for (int r = 0; r < CH / 8; ++r)
        *reinterpret_cast<u32x4*>(a.q_out + (first + lane / 8) * a.q_out_stride + head * HD + 8 * (8 * r + lane % 8)) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  const Sequence q = sequence_of(b, s);
  const int e0 = ((q.base >> 3) + local) * UNIT;  // the unit's first entry (base may be negative)
  if (e0 >= q.length || q.n == 0) return;
  // The page of the whole unit (pages hold whole units): its id is read here and looked at where it is used,
  // so that the loads below need not wait for it.
  const bool listed = e0 >= 0 && e0 < capacity(b);
  int id = -1;
  if (listed) id = b.tables[static_cast<int64_t>(s) * b.width + (e0 >> b.page_bits)];
  const int place = e0 & ((1 << b.page_bits) - 1);
  // The token of entry e0 + j (the nearest one where that is none), and its position if it has a row of the tables.
  auto token = [&](int j) { return q.first + clamp_to(e0 + j - q.base, 0, q.n - 1); };
  auto is_new = [&](int j) { return e0 + j >= q.base && e0 + j < q.length; };
  auto position = [&](int j) -> int {
    if (!is_new(j)) return -1;
    const int p = a.positions != nullptr ? a.positions[token(j)] : e0 + j;
    return a.half == 0 ? max(p, 0) : p < a.table ? p : -1;
  };

  if (task >= turned_tasks) {
    const int h = task - turned_tasks;
    if (2 * lane >= HD) return;
    uint32_t x[UNIT];
    uint32_t there = 0;
#pragma unroll
    for (int j = 0; j < UNIT; ++j) x[j] = *reinterpret_cast<const uint32_t*>(a.v + token(j) * a.v_stride + h * HD + 2 * lane);
#pragma unroll
    for (int j = 0; j < UNIT; ++j) there |= position(j) >= 0 ? 1u << j : 0u;
    if (id < 0 || id >= b.pages) return;
    uint16_t* const to = a.v_cache + ((static_cast<int64_t>(id) * a.kv_heads + h) << b.page_bits) * HD + static_cast<int64_t>(place) * HD +
                         16 * lane;
    if (there == 0xffu) {
      u32x4 lo, hi;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        lo[d] = __builtin_amdgcn_perm(x[2 * d + 1], x[2 * d], 0x05040100u);
        hi[d] = __builtin_amdgcn_perm(x[2 * d + 1], x[2 * d], 0x07060302u);
      }
      *reinterpret_cast<u32x4*>(to) = lo;
      *reinterpret_cast<u32x4*>(to + 8) = hi;
    } else {
#pragma unroll
      for (int j = 0; j < UNIT; ++j)
        if (there >> j & 1) {
          to[j] = static_cast<uint16_t>(x[j]);
          to[8 + j] = static_cast<uint16_t>(x[j] >> 16);
        }
    }
    return;
  }

  // Lane 8 j + i takes chunks i, i + 8 of token j: K's lines (eight tokens of a chunk) are written whole, and at
  // a head of 128 rotated dimensions a pair's two are the lane's own.
  constexpr int ROUNDS = CH / 8;
  const int j = lane >> 3, i = lane & 7;
  const int turn = a.half / 8;  // chunks from a pair's first dimension to its second
  const int at = position(j);
  // Every load before any of them is used (a row or head that is not there: one that is, and not used).
  u32x4 raw[HEADS][ROUNDS];
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    const int head = min(task * HEADS + n, turned_heads - 1);
    const uint16_t* const src = head < a.heads ? a.q + token(j) * a.q_stride + head * HD : a.k + token(j) * a.k_stride + (head - a.heads) * HD;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) raw[n][r] = *reinterpret_cast<const u32x4*>(src + 8 * (8 * r + i));
  }
  f32x4 cs[ROUNDS][2], sn[ROUNDS][2];
  if (a.half > 0 && a.table > 0) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      if (r > 0 && turn == 8) {  // the same angles
#pragma unroll
        for (int d = 0; d < 2; ++d) cs[r][d] = cs[0][d], sn[r][d] = sn[0][d];
        continue;
      }
      const int c = 8 * r + i;
      const int64_t row = static_cast<int64_t>(max(at, 0)) * a.half + (c < turn ? 8 * c : c < 2 * turn ? 8 * (c - turn) : 0);
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        cs[r][d] = *reinterpret_cast<const f32x4*>(a.cos + row + 4 * d);
        sn[r][d] = *reinterpret_cast<const f32x4*>(a.sin + row + 4 * d);
      }
    }
  }
  const bool stored = at >= 0 && id >= 0 && id < b.pages;
#pragma unroll
  for (int n = 0; n < HEADS; ++n) {
    const int head = task * HEADS + n;
    if (head >= turned_heads) break;
    const bool is_q = head < a.heads;
    const float* const norm = is_q ? a.q_norm : a.k_norm;
    float x[ROUNDS][8];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        x[r][2 * d] = E::to_f32(static_cast<uint16_t>(raw[n][r][d] & 0xffffu));
        x[r][2 * d + 1] = E::to_f32(static_cast<uint16_t>(raw[n][r][d] >> 16));
      }
    if (norm != nullptr) {
      float sum = chunk_squares(x[0]);
      if constexpr (ROUNDS == 2) sum += chunk_squares(x[ROUNDS - 1]);
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor(sum, off, 64);
      const float by = rsqrtf(sum / static_cast<float>(HD) + a.eps);
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(norm + 8 * (8 * r + i) + 4 * d);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[r][4 * d + e] = x[r][4 * d + e] * by * w[e];
        }
    }
    if (a.half > 0) {
      float y[ROUNDS][8];  // the pairs' other dimensions
      if (ROUNDS == 2 && turn == 8) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
          for (int d = 0; d < 8; ++d) y[r][d] = x[ROUNDS - 1 - r][d];
      } else {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
          const int c = 8 * r + i, other = c < turn ? c + turn : c < 2 * turn ? c - turn : c;
          const int lane_of = (lane & ~7) | (other & 7);
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            y[r][d] = __shfl(x[0][d], lane_of, 64);
            if constexpr (ROUNDS == 2) {
              const float high = __shfl(x[ROUNDS - 1][d], lane_of, 64);
              if (other >= 8) y[r][d] = high;
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int c = 8 * r + i;
        if (c < 2 * turn) {
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const float cv = cs[r][d / 4][d % 4], sv = sn[r][d / 4][d % 4];
            x[r][d] = c < turn ? fmaf(x[r][d], cv, -(y[r][d] * sv)) : fmaf(x[r][d], cv, y[r][d] * sv);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      u32x4 out;
#pragma unroll
      for (int d = 0; d < 4; ++d)
        out[d] = static_cast<uint32_t>(E::from_f32(x[r][2 * d])) | (static_cast<uint32_t>(E::from_f32(x[r][2 * d + 1])) << 16);
      const int c = 8 * r + i;
      if (is_q) {
        // (A token whose position has no row of the tables: zeros.)
        if (is_new(j)) *reinterpret_cast<u32x4*>(a.q_out + token(j) * a.q_out_stride + head * HD + 8 * c) = at >= 0 ? out : u32x4{0u, 0u, 0u, 0u};
      } else if (stored) {
        const int64_t to = (static_cast<int64_t>(id) * a.kv_heads + head - a.heads) * CH + c;
        *reinterpret_cast<u32x4*>(a.k_cache + ((to << b.page_bits) + place + j) * 8) = out;
      }
    }
  }
}

// keep: entry base + path[j] of each sequence to base + j, in every layer's cache, for the nodes
// path[0] < path[1] < .. of an accepted path (to the first entry that is no later node), and the
// sequence's new length base + their number. A wave takes one KV head of one layer of one sequence, eight
// nodes at a time, all of them read before any is written; as path[j] >= j and ascends, none is written before
// it has been read. Bound by lines: eight entries of a dimension share 16 bytes, so an entry's V is read
// and written in all lines of its eight. 48 sequences' paths out of 2700 nodes, 32 layers of 8 KV heads of 128: 62 us (70 to 80
// with a node at a time, its V sixteen dimensions a lane); one sequence's 4.0.
struct KeepArgs {
  uint16_t *k_cache, *v_cache;
  const int32_t* kept;  // [sequences, path]
  int32_t* lengths_out;
  Batch batch;
  int64_t layer_step;   // values from a layer's cache to the next one's
  int path, layers, kv_heads;
};

template <int HD>
__global__ __launch_bounds__(64 * WAVES) void paged_keep_kernel(KeepArgs a) {
  constexpr int CH = HD / 8, TOKENS = 64 / CH;
  const Batch& b = a.batch;
  const int per = a.layers * a.kv_heads;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * WAVES + (threadIdx.x >> 6);
  if (at >= static_cast<int64_t>(per) * b.sequences) return;
  const int s = static_cast<int>(at / per), head = static_cast<int>(at % per);
  const int lane = threadIdx.x & 63;
  const Sequence q = sequence_of(b, s);
  const int32_t* const path = a.kept + static_cast<int64_t>(s) * a.path;
  int number = 0;
  for (int j0 = 0; j0 < a.path; j0 += 64) {
    const int j = j0 + lane;
    bool good = false;
    if (j < a.path) {
      const int node = path[j];
      good = node >= 0 && node < q.n && (j == 0 || node > path[j - 1]);
    }
    const uint64_t run = __ballot(good);
    number += run == ~0ull ? 64 : __builtin_ctzll(~run);
    if (run != ~0ull) break;
  }
  if (head == 0 && lane == 0) a.lengths_out[s] = max(q.base + number, 0);
  const int layer = head / a.kv_heads, h = head % a.kv_heads;
  uint16_t* const kc = a.k_cache + layer * a.layer_step;
  uint16_t* const vc = a.v_cache + layer * a.layer_step;
  const int c = lane % CH;
  const int mask = (1 << b.page_bits) - 1;
  constexpr int BATCH = 8, ROUNDS = BATCH / TOKENS;
  for (int j0 = 0; j0 < number; j0 += BATCH) {
    // Lane k (of each 8) has node j0 + k: its entry and place to go, in K's pages (in 16-byte pieces from dimension
    // 0) and V's (in values), or -1 where it stays.
    const int j = j0 + lane % BATCH;
    int64_t from_v = -1, to_v = -1, from_k = -1, to_k = -1;
    if (j < number) {
      const int node = path[j];
      const int from = q.base + node, to = q.base + j;
      const int from_page = node != j ? page_of(b, s, from) : -1, to_page = node != j ? page_of(b, s, to) : -1;
      if (from_page >= 0 && to_page >= 0) {
        const int64_t fp = static_cast<int64_t>(from_page) * a.kv_heads + h, tp = static_cast<int64_t>(to_page) * a.kv_heads + h;
        from_k = (fp * CH << b.page_bits) + (from & mask);
        to_k = (tp * CH << b.page_bits) + (to & mask);
        from_v = ((fp << (b.page_bits - 3)) + ((from & mask) >> 3)) * HD * 8 + (from & 7);
        to_v = ((tp << (b.page_bits - 3)) + ((to & mask) >> 3)) * HD * 8 + (to & 7);
      }
    }
    u32x4 kv[ROUNDS];
    int64_t k_to[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int lane_of = r * TOKENS + lane / CH;
      const int64_t at = __shfl(from_k, lane_of, 64);
      k_to[r] = __shfl(to_k, lane_of, 64);
      kv[r] = u32x4{0u, 0u, 0u, 0u};
      if (at >= 0) kv[r] = *reinterpret_cast<const u32x4*>(kc + (at + (static_cast<int64_t>(c) << b.page_bits)) * 8);
    }
    // V: a lane a dimension, so that an instruction reads eight neighbouring lines of one entry.
    uint16_t v[BATCH][HD / 64];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int64_t at = __shfl(from_v, k, 64);
#pragma unroll
      for (int d = 0; d < HD / 64; ++d) v[k][d] = at >= 0 ? vc[at + (64 * d + lane) * 8] : uint16_t{0};
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
      if (k_to[r] >= 0) *reinterpret_cast<u32x4*>(kc + (k_to[r] + (static_cast<int64_t>(c) << b.page_bits)) * 8) = kv[r];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int64_t at = __shfl(to_v, k, 64);
#pragma unroll
      for (int d = 0; d < HD / 64; ++d)
        if (at >= 0) vc[at + (64 * d + lane) * 8] = v[k][d];
    }
  }
}

}  // namespace paged
}  // namespace lnq

using namespace lnq;

extern "C" {

LNQ_API LnqStatus lnq_paged_append(const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                                   int64_t v_stride, const float* cos, const float* sin, int64_t table, int64_t half,
                                   const int32_t* positions, const float* q_norm, const float* k_norm, float eps,
                                   void* q_out, int64_t q_out_stride, int32_t fill, void* k_cache, void* v_cache,
                                   const int32_t* tables, const int32_t* lengths, const int32_t* starts,
                                   int64_t sequences, int64_t width, int64_t pages, int64_t page, int64_t tokens,
                                   int64_t heads, int64_t kv_heads, int64_t head_dim, int32_t dtype, void* stream) {
  const char* const no = paged::refused({sequences, width, pages, page, tokens});
  LNQ_REQUIRE(no == nullptr, "lnq_paged_append: %s", no);
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16, "lnq_paged_append: dtype %d is not bf16 or f16", dtype);
  LNQ_REQUIRE(head_dim == 64 || head_dim == 128, "lnq_paged_append: head_dim is 64 or 128, not %lld", (long long)head_dim);
  LNQ_REQUIRE(heads >= 0 && kv_heads >= 1 && heads <= 65536 && kv_heads <= 65536, "lnq_paged_append: bad heads %lld / %lld",
              (long long)heads, (long long)kv_heads);
  LNQ_REQUIRE(half >= 0 && half % 8 == 0 && 2 * half <= head_dim,
              "lnq_paged_append: tables of half=%lld angles (a multiple of 8, at most head_dim / 2)", (long long)half);
  LNQ_REQUIRE(table >= 0 && table <= INT32_MAX, "lnq_paged_append: bad tables");
  const int64_t units = tokens / paged::UNIT + 2 * sequences + 2;
  // Two heads of q's and k's a wave once there are more waves than the chip holds: 8191 tokens of 40 heads 41.0 us against 44.9
  // at one and 42.1 at four; one token 4.1 and 4.9 against 3.5.
  const int64_t turned = heads + kv_heads, each = units * (turned + kv_heads) > 8192 ? 2 : 1;
  const int64_t groups = ((turned + each - 1) / each + kv_heads + paged::WAVES - 1) / paged::WAVES;
  LNQ_REQUIRE(units * groups <= paged::MOST_WORKGROUPS, "lnq_paged_append: too large (fewer tokens a call)");
  if (tokens == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(k && v && ((k_cache && v_cache) || pages == 0) && starts && (lengths || sequences == 0) &&
                  (tables || width == 0 || sequences == 0) &&
                  (heads == 0 || (q && q_out)) && (half == 0 || (cos && sin)),
              "lnq_paged_append: null pointer");
  LNQ_REQUIRE(aligned(q, 16) && aligned(k, 16) && aligned(v, 4) && aligned(q_out, 16) && aligned(k_cache, 16) &&
                  aligned(v_cache, 16) && aligned(cos, 16) && aligned(sin, 16) && aligned(q_norm, 16) && aligned(k_norm, 16) &&
                  q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 2 == 0 && q_out_stride % 8 == 0,
              "lnq_paged_append: operands must be 16-byte aligned, strides whole 16 bytes");
  LNQ_REQUIRE(tokens == 1 || (q_stride >= heads * head_dim && k_stride >= kv_heads * head_dim &&
                              v_stride >= kv_heads * head_dim && q_out_stride >= heads * head_dim),
              "lnq_paged_append: a row stride is shorter than a row");
  paged::AppendArgs a{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
                      q_stride, k_stride, v_stride, cos, sin, positions, q_norm, k_norm, static_cast<uint16_t*>(q_out),
                      static_cast<uint16_t*>(k_cache), static_cast<uint16_t*>(v_cache), q_out_stride,
                      {tables, lengths, starts, static_cast<int>(sequences), static_cast<int>(width),
                       static_cast<int>(pages), paged::bits_of(page), static_cast<int>(tokens)},
                      static_cast<int>(heads), static_cast<int>(kv_heads), static_cast<int>(half),
                      static_cast<int>(table), static_cast<int>(groups), eps, fill != 0};
  const dim3 grid(static_cast<unsigned>(units * groups)), block(64 * paged::WAVES);
  const auto st = static_cast<hipStream_t>(stream);
#define LNQ_APPEND(DT_, HD_)                                                                                            \
  if (each == 2) hipLaunchKernelGGL((paged::paged_append_kernel<DT_, HD_, 2>), grid, block, 0, st, a);                \
  else hipLaunchKernelGGL((paged::paged_append_kernel<DT_, HD_, 1>), grid, block, 0, st, a)
  if (dtype == LNQ_BF16 && head_dim == 128) { LNQ_APPEND(LNQ_BF16, 128); }
  else if (dtype == LNQ_BF16) { LNQ_APPEND(LNQ_BF16, 64); }
  else if (head_dim == 128) { LNQ_APPEND(LNQ_F16, 128); }
  else { LNQ_APPEND(LNQ_F16, 64); }
#undef LNQ_APPEND
  return launched("paged_append");
}

LNQ_API LnqStatus lnq_paged_keep(void* k_cache, void* v_cache, int64_t layers, int64_t layer_step, const int32_t* tables,
                                 const int32_t* lengths, const int32_t* starts, const int32_t* kept, int64_t path,
                                 int32_t* lengths_out, int64_t sequences, int64_t width, int64_t pages, int64_t page,
                                 int64_t tokens, int64_t kv_heads, int64_t head_dim, void* stream) {
  const char* const no = paged::refused({sequences, width, pages, page, tokens});
  LNQ_REQUIRE(no == nullptr, "lnq_paged_keep: %s", no);
  LNQ_REQUIRE(head_dim == 64 || head_dim == 128, "lnq_paged_keep: head_dim is 64 or 128, not %lld", (long long)head_dim);
  LNQ_REQUIRE(kv_heads >= 1 && kv_heads <= 65536 && layers >= 1 && layers <= 65536 && path >= 0 && path <= INT32_MAX,
              "lnq_paged_keep: bad shape layers=%lld kv_heads=%lld path=%lld", (long long)layers, (long long)kv_heads, (long long)path);
  const int64_t one = pages * kv_heads * page * head_dim;
  LNQ_REQUIRE(layers == 1 || (layer_step >= one && layer_step % 8 == 0), "lnq_paged_keep: layers overlap");
  const int64_t waves = sequences * layers * kv_heads, blocks = (waves + paged::WAVES - 1) / paged::WAVES;
  LNQ_REQUIRE(layers * kv_heads <= INT32_MAX && blocks <= paged::MOST_WORKGROUPS, "lnq_paged_keep: too large (fewer layers a call)");
  if (sequences == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(((k_cache && v_cache) || pages == 0) && lengths && starts && lengths_out && (tables || width == 0) && (kept || path == 0),
              "lnq_paged_keep: null pointer");
  LNQ_REQUIRE(aligned(k_cache, 16) && aligned(v_cache, 16), "lnq_paged_keep: caches must be 16-byte aligned");
  paged::KeepArgs a{static_cast<uint16_t*>(k_cache), static_cast<uint16_t*>(v_cache), kept, lengths_out,
                    {tables, lengths, starts, static_cast<int>(sequences), static_cast<int>(width),
                     static_cast<int>(pages), paged::bits_of(page), static_cast<int>(tokens)},
                    layer_step, static_cast<int>(path), static_cast<int>(layers), static_cast<int>(kv_heads)};
  const dim3 grid(static_cast<unsigned>(blocks)), block(64 * paged::WAVES);
  const auto st = static_cast<hipStream_t>(stream);
  if (head_dim == 128) hipLaunchKernelGGL(paged::paged_keep_kernel<128>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(paged::paged_keep_kernel<64>, grid, block, 0, st, a);
  return launched("paged_keep");
}

}  // extern "C"
