// New tokens into a KV cache in pages, and an accepted path of drafted ones to its place.
//
// append: per token and head of q and k, y = x * rsqrt(mean(x^2) + eps) * w (where there are
// norms), then the pairs (i, i + r) of the first 2 r dimensions by the angle of the token's
// position, y'_i = y_i cos_i - y_(i+r) sin_i, y'_(i+r) = y_(i+r) cos_i + y_i sin_i, in f32 and
// rounded once; k and v into the cache, q out. Bound by memory: each value is read once and
// written once.
//
// Eight entries at an aligned place of a sequence are the unit, as V's layout keeps eight entries
// of a dimension together: one wave takes one head of one unit. Of q and k a lane holds 8
// dimensions of a token (16 bytes; the other of a pair comes from the lane that holds it), of v a
// lane holds two dimensions of all eight tokens, so that V's 16-byte pieces come out of registers by
// v_perm. A whole unit is written in whole lines, a partial one (a single token of a decode step)
// by its entries alone.
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

template <int DT, int HD>
__global__ __launch_bounds__(64 * WAVES) void paged_append_kernel(AppendArgs a) {
  using E = Elem<DT>;
  constexpr int CH = HD / 8;         // 16-byte chunks a head
  constexpr int TOKENS = 64 / CH;    // tokens a wave's load covers
  const Batch& b = a.batch;
  const int slot = blockIdx.x / a.groups;
  const int head = (blockIdx.x % a.groups) * WAVES + (threadIdx.x >> 6);  // q's heads, k's, v's
  const int lane = threadIdx.x & 63;
  // The sequences, and after them the tokens that belong to none.
  const int s = find_sequence(b.sequences + 1, slot, [&](int i) { return append_slot(b, i); });
  if (head >= a.heads + 2 * a.kv_heads) return;
  const int local = slot - append_slot(b, s);
  if (local < 0) return;
  if (s == b.sequences) {
    const int first = clamp_to(b.starts[s], 0, b.tokens) + local * UNIT;
    if (!a.fill || head >= a.heads) return;
#pragma unroll
    for (int it = 0; it < UNIT / TOKENS; ++it) {
      const int t = first + it * TOKENS + lane / CH;
      if (t < b.tokens)
        *reinterpret_cast<u32x4*>(a.q_out + t * a.q_out_stride + head * HD + 8 * (lane % CH)) = u32x4{0u, 0u, 0u, 0u};
    }
    return;
  }
  const Sequence q = sequence_of(b, s);
  const int e0 = ((q.base >> 3) + local) * UNIT;  // the unit's first entry (base may be negative)
  if (e0 >= q.length || q.n == 0) return;
  const int page = page_of(b, s, e0);  // of the whole unit: pages hold whole units
  const int place = e0 & ((1 << b.page_bits) - 1);

  // Whether entry e0 + j is a new token whose position has a row of the tables.
  auto position = [&](int j) -> int {
    const int i = e0 + j - q.base;
    if (i < 0 || i >= q.n) return -1;
    const int p = a.positions != nullptr ? a.positions[q.first + i] : e0 + j;
    return a.half == 0 ? max(p, 0) : p < a.table ? p : -1;
  };

  if (head >= a.heads + a.kv_heads) {
    if (page < 0) return;
    const int h = head - a.heads - a.kv_heads;
    if (2 * lane >= HD) return;
    uint32_t x[UNIT];
    uint32_t there = 0;
#pragma unroll
    for (int j = 0; j < UNIT; ++j) {
      x[j] = 0;
      if (position(j) >= 0) {
        there |= 1u << j;
        x[j] = *reinterpret_cast<const uint32_t*>(a.v + (q.first + e0 + j - q.base) * a.v_stride + h * HD + 2 * lane);
      }
    }
    uint16_t* const to = a.v_cache + ((static_cast<int64_t>(page) * a.kv_heads + h) << b.page_bits) * HD + static_cast<int64_t>(place) * HD +
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

  const bool is_q = head < a.heads;
  const int h = is_q ? head : head - a.heads;
  const uint16_t* const src = is_q ? a.q : a.k;
  const int64_t stride = is_q ? a.q_stride : a.k_stride;
  const float* const norm = is_q ? a.q_norm : a.k_norm;
  const int c = lane % CH;
  f32x4 w0 = {1.f, 1.f, 1.f, 1.f}, w1 = w0;
  if (norm != nullptr) {
    w0 = *reinterpret_cast<const f32x4*>(norm + 8 * c);
    w1 = *reinterpret_cast<const f32x4*>(norm + 8 * c + 4);
  }
  // The lane with the other dimension of this one's pairs, and the pairs' first angle.
  const int turn = a.half / 8;
  const bool first_half = c < turn, turned = c < 2 * turn;
  const int other = (lane & ~(CH - 1)) | (first_half ? c + turn : turned ? c - turn : c);
  const int angle = 8 * (first_half ? c : c - turn);
#pragma unroll
  for (int it = 0; it < UNIT / TOKENS; ++it) {
    const int j = it * TOKENS + lane / CH;
    const int i = e0 + j - q.base, p = position(j);
    const bool mine = i >= 0 && i < q.n;
    u32x4 raw = {0u, 0u, 0u, 0u};
    if (p >= 0) raw = *reinterpret_cast<const u32x4*>(src + (q.first + i) * stride + h * HD + 8 * c);
    float x[8];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      x[2 * d] = E::to_f32(static_cast<uint16_t>(raw[d] & 0xffffu));
      x[2 * d + 1] = E::to_f32(static_cast<uint16_t>(raw[d] >> 16));
    }
    if (norm != nullptr) {
      float sum = chunk_squares(x);
#pragma unroll
      for (int off = 1; off < CH; off <<= 1) sum += __shfl_xor(sum, off, 64);
      const float by = rsqrtf(sum / static_cast<float>(HD) + a.eps);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        x[d] = x[d] * by * w0[d];
        x[4 + d] = x[4 + d] * by * w1[d];
      }
    }
    if (a.half > 0) {
      float y[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) y[d] = __shfl(x[d], other, 64);
      if (turned && p >= 0) {
        const float* const cp = a.cos + static_cast<int64_t>(p) * a.half + angle;
        const float* const sp = a.sin + static_cast<int64_t>(p) * a.half + angle;
        const f32x4 c0 = *reinterpret_cast<const f32x4*>(cp), c1 = *reinterpret_cast<const f32x4*>(cp + 4);
        const f32x4 s0 = *reinterpret_cast<const f32x4*>(sp), s1 = *reinterpret_cast<const f32x4*>(sp + 4);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const float cv = d < 4 ? c0[d & 3] : c1[d & 3], sv = d < 4 ? s0[d & 3] : s1[d & 3];
          x[d] = first_half ? fmaf(x[d], cv, -(y[d] * sv)) : fmaf(x[d], cv, y[d] * sv);
        }
      }
    }
    u32x4 out;
#pragma unroll
    for (int d = 0; d < 4; ++d)
      out[d] = static_cast<uint32_t>(E::from_f32(x[2 * d])) | (static_cast<uint32_t>(E::from_f32(x[2 * d + 1])) << 16);
    if (is_q) {
      // (A token whose position has no row of the tables: zeros.)
      if (mine) *reinterpret_cast<u32x4*>(a.q_out + (q.first + i) * a.q_out_stride + h * HD + 8 * c) = p >= 0 ? out : u32x4{0u, 0u, 0u, 0u};
    } else if (p >= 0 && page >= 0) {
      const int64_t at = (static_cast<int64_t>(page) * a.kv_heads + h) * CH + c;
      *reinterpret_cast<u32x4*>(a.k_cache + ((at << b.page_bits) + place + j) * 8) = out;
    }
  }
}

// keep: entry base + path[j] of each sequence to base + j, in every layer's cache, for the nodes
// path[0] < path[1] < .. of an accepted path (to the first entry that is no later node), and the
// sequence's new length base + their number. A wave takes one KV head of one layer of one sequence, 64 chunks
// of 16 bytes at a time; as path[j] >= j and ascends, no entry is written before it has been read.
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
  for (int j0 = 0; j0 < number; j0 += TOKENS) {
    const int j = j0 + lane / CH;
    bool move = j < number;
    int from = 0, to = 0, from_page = -1, to_page = -1;
    if (move) {
      const int node = path[j];
      from = q.base + node;
      to = q.base + j;
      if (node != j) {
        from_page = page_of(b, s, from);
        to_page = page_of(b, s, to);
      }
    }
    move = move && from_page >= 0 && to_page >= 0;
    if (!move) continue;
    const int64_t from_k = (((static_cast<int64_t>(from_page) * a.kv_heads + h) * CH + c) << b.page_bits) + (from & mask);
    const int64_t to_k = (((static_cast<int64_t>(to_page) * a.kv_heads + h) * CH + c) << b.page_bits) + (to & mask);
    auto v_at = [&](int page, int e) {
      const int64_t eight = ((static_cast<int64_t>(page) * a.kv_heads + h) << (b.page_bits - 3)) + ((e & mask) >> 3);
      return (eight * HD + 8 * c) * 8 + (e & 7);
    };
    const uint16_t* const from_v = vc + v_at(from_page, from);
    uint16_t* const to_v = vc + v_at(to_page, to);
    const u32x4 kv = *reinterpret_cast<const u32x4*>(kc + from_k * 8);
    uint16_t v[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) v[d] = from_v[8 * d];
    *reinterpret_cast<u32x4*>(kc + to_k * 8) = kv;
#pragma unroll
    for (int d = 0; d < 8; ++d) to_v[8 * d] = v[d];
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
  const int64_t groups = (heads + 2 * kv_heads + paged::WAVES - 1) / paged::WAVES;
  LNQ_REQUIRE(units * groups <= INT32_MAX, "lnq_paged_append: too large");
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
  if (dtype == LNQ_BF16 && head_dim == 128) hipLaunchKernelGGL((paged::paged_append_kernel<LNQ_BF16, 128>), grid, block, 0, st, a);
  else if (dtype == LNQ_BF16) hipLaunchKernelGGL((paged::paged_append_kernel<LNQ_BF16, 64>), grid, block, 0, st, a);
  else if (head_dim == 128) hipLaunchKernelGGL((paged::paged_append_kernel<LNQ_F16, 128>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged::paged_append_kernel<LNQ_F16, 64>), grid, block, 0, st, a);
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
  LNQ_REQUIRE(layers * kv_heads <= INT32_MAX && blocks <= INT32_MAX, "lnq_paged_keep: too large");
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
