// The KV cache in pages, as its append, attention and keep kernels see it: a batch of sequences
// over one pool of pages.
//
// Layouts (16-bit values). K [pages, kv_heads, head_dim / 8, page, 8], V [pages, kv_heads,
// page / 8, head_dim, 8]: K's product with a query sums over dimensions and V's with the weights
// over entries, and an MFMA operand is 8 values of the summed index a lane. So a lane's operand is 16
// contiguous bytes of the pool and a wave's operand of 32 rows two runs of 512 bytes, from memory as
// from LDS, with no shuffle on the way.
//
// Everything on the device (tables, lengths, starts) is the caller's and is read with its bounds
// checked: an entry past its sequence's table, or in a page that is not in the pool, is not there.
#pragma once

#include "common.hpp"

namespace lnq {
namespace paged {

struct Batch {
  const int32_t* tables;   // [sequences, width]: page ids
  const int32_t* lengths;  // [sequences]: entries, the new tokens among them
  const int32_t* starts;   // [sequences + 1]: each sequence's first new token
  int sequences, width, pages, page_bits, tokens;
};

// One sequence of a batch: its new tokens [first, first + n) are its entries base .. base + n - 1.
struct Sequence {
  int first, n, length, base;
};

__device__ inline int clamp_to(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

__device__ inline Sequence sequence_of(const Batch& b, int s) {
  Sequence q;
  q.first = clamp_to(b.starts[s], 0, b.tokens);
  q.n = clamp_to(b.starts[s + 1], q.first, b.tokens) - q.first;
  q.length = clamp_to(b.lengths[s], 0, 0x7f000000);  // (sums with it stay in 32 bits)
  q.base = q.length - q.n;
  return q;
}

// Entries a table can hold (the host keeps it below 2^30).
__device__ inline int capacity(const Batch& b) { return b.width << b.page_bits; }

// The page of entry e (any int) of sequence s, -1 where it has none.
__device__ inline int page_of(const Batch& b, int s, int e) {
  if (e < 0 || e >= capacity(b)) return -1;
  const int p = b.tables[static_cast<int64_t>(s) * b.width + (e >> b.page_bits)];
  return p >= 0 && p < b.pages ? p : -1;
}

// Work is laid out in slots: a sequence of n tokens has at most n / per + more blocks (of `per`
// aligned entries, or of rows), and slot_of(start, s) = start / per + more * s leaves that many
// slots between a sequence's first token and the next one's, so that the grid's size needs the
// number of tokens alone. The last sequence in [0, count) whose first slot is not past `slot`, of one
// sequence at least (nothing that looks for one is launched without any); the whole wave takes part (64
// sequences a look, or 64 samples of them first).
template <class SlotOf>
__device__ inline int find_sequence(int count, int slot, SlotOf slot_of) {
  if (count <= 1) return 0;
  const int lane = threadIdx.x & 63;
  int from = 0, to = count;
  if (count > 64) {
    const int step = (count + 63) / 64;
    const int s = lane * step;
    const uint64_t before = __ballot(s < count && slot_of(s) <= slot);
    from = max(static_cast<int>(__popcll(before)) - 1, 0) * step;
    to = min(from + step, count);
  }
  int last = from;
  for (int s0 = from; s0 < to; s0 += 64) {
    const int s = s0 + lane;
    const int many = static_cast<int>(__popcll(__ballot(s < to && slot_of(s) <= slot)));
    if (many > 0) last = s0 + many - 1;
    if (many < 64) break;
  }
  return __builtin_amdgcn_readfirstlane(last);
}

// The host's checks of a batch; an empty message if it is one.
struct BatchCheck {
  int64_t sequences, width, pages, page, tokens;
};

inline const char* refused(const BatchCheck& c) {
  if (c.page != 16 && c.page != 32 && c.page != 64 && c.page != 128) return "a page holds 16, 32, 64 or 128 entries";
  if (c.sequences < 0 || c.sequences > (1 << 20)) return "at most 2^20 sequences";
  if (c.tokens < 0 || c.tokens > (1 << 24)) return "at most 2^24 new tokens";
  if (c.pages < 0 || c.pages > INT32_MAX) return "at most 2^31 - 1 pages";
  if (c.width < 0 || c.width * c.page > (1 << 30)) return "tables of at most 2^30 entries a sequence";
  return nullptr;
}

// Workgroups of 256 a launch takes at most (its threads are counted in 32 bits).
constexpr int64_t MOST_WORKGROUPS = (int64_t{1} << 24) - 1;

inline int bits_of(int64_t page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

}  // namespace paged
}  // namespace lnq
