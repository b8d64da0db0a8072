// The router of a mixture of experts: for each token the experts its row of logits chooses,
// and their weights.
//
//   s_e = exp(l_e) / sum_j exp(l_j)  or  1 / (1 + exp(-l_e))      the scores
//   c_e = s_e + b_e                                               what the choice goes by
//   a group's score: the sum of its best one or two c_e (of a group of one expert, its c_e);
//   the best groups are kept
//   the `top` kept experts of largest c, equal ones by the lower index
//   w_e = s_e (over the sum of the chosen s), times a factor
//
// Scores and choices are held in 64 bits: two choices next to each other then go by what the
// scores are and not by the rounding of an exponential. Without a bias the choice goes by the
// logits themselves, which order as the scores do. An expert whose logit is -inf, or whose
// choice is -inf or NaN, is never chosen; a place that no expert is left for holds -1 with a
// weight of 0 (the experts' products give zeros for it). A row with a NaN logit (or +inf under
// softmax) has no scores: its experts are -1, its weights NaN.
//
// A wave takes a row: with G groups rounded up to a power of two, 64 / G lanes hold a group, S
// experts a lane, so that experts rise with the lane and its slot. Bound by VALU issue, not by
// the row's bytes: so
// * an exponential is 2^n times a polynomial and a quotient a reciprocal with two Newton steps, a
//   third of the instructions that the library's functions take for every case;
// * a group's two best are a butterfly over its lanes, and its rank among the groups a count;
// * a choice is the wave's largest key, the choice rounded once to f32 (order survives rounding)
//   with its bits in integer order: six DPP maxima. Only where several experts hold that key,
//   which differ in 64 bits, are those compared.
// 8192 rows of 256 experts in 8 groups, top 8: 13.9 us, 730 vector instructions a row (54 us with a
// lane a group in turn, 18.7 with the library's exponential and choices by floats).
#include <algorithm>

#include "common.hpp"

namespace lnq {

namespace route {
constexpr int THREADS = 256;
constexpr int MAX_TOP = 64;    // a lane holds a choice
constexpr int MAX_COUNT = 1024;
constexpr int MAX_SLOTS = 32;  // experts of a lane: 1024 in 33 groups leave a lane a group of 31
}  // namespace route

struct RouteArgs {
  const float* bias;
  int64_t* experts;
  float* weights;
  int64_t stride;  // logits from row to row
  int rows, count, top, groups, group_top, group_best;
  int size, lanes;  // experts and lanes of a group
  int softmax, renormalize;
  double scale;
};

// `v` of another lane by a DPP control (lanes without a partner: `old`).
template <int CTRL>
__device__ inline float dpp(float old, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, v), CTRL,
                                                               0xf, 0xf, false));
}

template <int CTRL>
__device__ inline double dpp(double old, double v) {
  const uint64_t o = __builtin_bit_cast(uint64_t, old), b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(o), static_cast<int>(b), CTRL, 0xf, 0xf, false));
  const uint32_t hi =
      static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(o >> 32), static_cast<int>(b >> 32), CTRL, 0xf, 0xf, false));
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

__device__ inline float lane_of(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

__device__ inline double lane_of(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane));
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

// The wave's largest value: within rows of 16 lanes (row_shr 1, 2, 4, 8), then over the rows
// (row_bcast 15, 31); lane 63 ends with it.
__device__ inline double wave_top(double v) {
  v = fmax(v, dpp<0x111>(v, v));
  v = fmax(v, dpp<0x112>(v, v));
  v = fmax(v, dpp<0x114>(v, v));
  v = fmax(v, dpp<0x118>(v, v));
  v = fmax(v, dpp<0x142>(v, v));
  v = fmax(v, dpp<0x143>(v, v));
  return lane_of(v, 63);
}

template <int CTRL>
__device__ inline uint32_t larger(uint32_t v) {  // 0: what lanes without a partner compare with
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false)));
}

__device__ inline uint32_t wave_top(uint32_t v) {
  v = larger<0x111>(v);
  v = larger<0x112>(v);
  v = larger<0x114>(v);
  v = larger<0x118>(v);
  v = larger<0x142>(v);
  v = larger<0x143>(v);
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

// A float's bits in the order of integers, above 0 (the place of no choice); both zeros alike.
__device__ inline uint32_t key_of(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

__device__ inline float value_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// e^x for |x| <= 800 (past a double's range: infinity, 0): x = n ln 2 + r, |r| <= ln 2 / 2, and e^r's
// series up to r^13 / 13! (the next term is below 2^-57 of it).
__device__ inline double exp_of(double x) {
  const double n = rint(x * 0x1.71547652b82fep+0);
  const double r = fma(n, -0x1.abc9e3b39803fp-56, fma(n, -0x1.62e42fefa39efp-1, x));
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, static_cast<int>(n));
}

// The wave's sum: that of each row of 16 lanes in its last lane, the four added.
__device__ inline double wave_total(double v) {
  v += dpp<0x111>(0.0, v);
  v += dpp<0x112>(0.0, v);
  v += dpp<0x114>(0.0, v);
  v += dpp<0x118>(0.0, v);
  return (lane_of(v, 15) + lane_of(v, 31)) + (lane_of(v, 47) + lane_of(v, 63));
}

// The partner's value in the butterfly step over `d` lanes, where every lane of a run of d
// holds the same (quad_perm, then mirrors of 8 and 16 lanes).
__device__ inline double across(double v, int d) {
  if (d == 1) return dpp<0xb1>(v, v);
  if (d == 2) return dpp<0x4e>(v, v);
  if (d == 4) return dpp<0x141>(v, v);
  if (d == 8) return dpp<0x140>(v, v);
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(__shfl_xor(static_cast<int>(b), d, 64));
  const uint32_t hi = static_cast<uint32_t>(__shfl_xor(static_cast<int>(b >> 32), d, 64));
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

template <int DT, int S>
__global__ __launch_bounds__(route::THREADS) void expert_route_kernel(const typename Elem<DT>::storage* __restrict__ logits,
                                                                      RouteArgs a) {
  using E = Elem<DT>;
  const int lane = threadIdx.x & 63;
  const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * (route::THREADS / 64) + (threadIdx.x >> 6));
  if (row >= a.rows) return;  // the whole wave
  const double none = -__builtin_huge_val();
  const float nothing = -__builtin_huge_valf();
  const typename E::storage* from = logits + row * a.stride;
  const int group = lane / a.lanes, place = (lane - group * a.lanes) * S;
  const int e0 = group * a.size + place;  // this lane's first expert
  const int held = group < a.groups ? min(S, a.size - place) : 0;
  const bool biased = a.bias != nullptr;
  float l[S], b[S], most = nothing;
  bool bad = false;
  // All loads before the first use; slots past the held ones read the last expert, for nothing.
  typename E::storage raw[S];
#pragma unroll
  for (int i = 0; i < S; ++i) raw[i] = from[min(e0 + i, a.count - 1)];
  if (biased) {
#pragma unroll
    for (int i = 0; i < S; ++i) b[i] = a.bias[min(e0 + i, a.count - 1)];
  }
#pragma unroll
  for (int i = 0; i < S; ++i) {
    l[i] = i < held ? E::to_f32(raw[i]) : nothing;
    bad = bad || l[i] != l[i] || (a.softmax && l[i] == __builtin_huge_valf());
    most = fmaxf(most, l[i]);
  }
  int64_t* const experts = a.experts + static_cast<int64_t>(row) * a.top;
  float* const weights = a.weights + static_cast<int64_t>(row) * a.top;
  if (__ballot(bad)) {
    if (lane < a.top) experts[lane] = -1, weights[lane] = __builtin_nanf("");
    return;
  }

  double s[S];
  if (a.softmax) {
    const float high = value_of(wave_top(key_of(most)));
    const double top = high == nothing ? 0 : high;
    double sum = 0;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      s[i] = l[i] == nothing ? 0 : exp_of(fmax(l[i] - top, -800.0));
      sum += s[i];
    }
    sum = wave_total(sum);
    const double part = sum > 0 ? 1 / sum : 0;
#pragma unroll
    for (int i = 0; i < S; ++i) s[i] *= part;
  } else {
    bool far = false;
    double d[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      d[i] = 1 + exp_of(-static_cast<double>(fminf(fmaxf(l[i], -800.0f), 800.0f)));
      far = far || d[i] > 0x1p1000;
      double y = __builtin_amdgcn_rcp(d[i]);
      y = fma(fma(-d[i], y, 1.0), y, y);
      s[i] = fma(fma(-d[i], y, 1.0), y, y);
    }
    if (__ballot(far)) {  // where the steps' products leave a double's range
#pragma unroll
      for (int i = 0; i < S; ++i) s[i] = d[i] > 0x1p1000 ? 1 / d[i] : s[i];
    }
#pragma unroll
    for (int i = 0; i < S; ++i) s[i] = l[i] == nothing ? 0 : s[i];
  }
  // The choices and their keys.
  double c[S];
  uint32_t key[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    if (biased) {
      c[i] = s[i] + static_cast<double>(b[i]);
      c[i] = l[i] != nothing && c[i] > none ? c[i] : none;
    } else {
      c[i] = l[i];
    }
    key[i] = c[i] == none ? 0 : key_of(static_cast<float>(c[i]));
  }

  if (a.groups > 1) {
    // The two best of the group; without a bias their scores, which rise with the logits.
    double v = none, w = none;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const double q = c[i] == none || biased || a.group_best == 1 ? c[i] : s[i];
      w = fmax(w, fmin(v, q));
      v = fmax(v, q);
    }
    for (int d = 1; d < a.lanes; d *= 2) {
      const double v2 = across(v, d), w2 = across(w, d);
      w = fmax(fmax(w, w2), fmin(v, v2));
      v = fmax(v, v2);
    }
    if (a.group_best == 2) v = w == none ? none : v + w;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double other = lane_of(v, g * a.lanes);
      rank += other > v || (other == v && g < group);
    }
    if (rank >= a.group_top) {
#pragma unroll
      for (int i = 0; i < S; ++i) key[i] = 0;
    }
  }

  int mine = -1;
  double weight = 0, total = 0;
  for (int i = 0; i < a.top; ++i) {
    uint32_t best = key[0];
#pragma unroll
    for (int j = 1; j < S; ++j) best = max(best, key[j]);
    const uint32_t top = wave_top(best);
    if (top == 0) break;
    // The lanes that hold it in each slot. One place, mostly: taken by selects, without a branch.
    uint64_t with[S], any = 0;
    int places = 0;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      with[j] = __ballot(key[j] == top);
      places += __popcll(with[j]);
      any |= with[j];
    }
    // Of several the first expert, by the choices themselves where those are more than the key shows.
    if (places > 1) {
      if (biased) {
        double most_c = none;
#pragma unroll
        for (int j = 0; j < S; ++j) most_c = fmax(most_c, key[j] == top ? c[j] : none);
        most_c = wave_top(most_c);
        any = 0;
#pragma unroll
        for (int j = 0; j < S; ++j) {
          with[j] = __ballot(key[j] == top && c[j] == most_c);
          any |= with[j];
        }
      }
      uint64_t bit = any & (~any + 1);
#pragma unroll
      for (int j = 0; j < S; ++j) {
        with[j] &= bit;
        bit &= ~with[j];
      }
    }
    const int owner = __builtin_ctzll(any);
    int e = e0;
    double v = s[0];
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const bool here = __builtin_amdgcn_inverse_ballot_w64(with[j]);
      if (j > 0) e = here ? e0 + j : e, v = here ? s[j] : v;
      key[j] = here ? 0 : key[j];
    }
    const int at = __builtin_amdgcn_readlane(e, owner);
    v = lane_of(v, owner);
    total += v;
    if (lane == i) mine = at, weight = v;
  }
  if (a.renormalize) weight = total > 0 ? weight / total : 0;
  if (lane < a.top) experts[lane] = mine, weights[lane] = static_cast<float>(weight * a.scale);
}

}  // namespace lnq

using namespace lnq;

extern "C" {

LNQ_API LnqStatus lnq_expert_route(const void* logits, int64_t stride, const float* bias, int64_t* experts, float* weights,
                                   int64_t rows, int64_t num_experts, int64_t top, int64_t groups, int64_t group_top,
                                   int64_t group_best, int32_t softmax, int32_t renormalize, double scale, int32_t dtype,
                                   void* stream) {
  LNQ_REQUIRE(dtype == LNQ_BF16 || dtype == LNQ_F16 || dtype == LNQ_F32, "lnq_expert_route: dtype %d is not bf16, f16 or f32",
              dtype);
  LNQ_REQUIRE(rows >= 0 && rows <= INT32_MAX && num_experts > 0 && num_experts <= route::MAX_COUNT,
              "lnq_expert_route: %lld rows of %lld experts (1 to %d)", static_cast<long long>(rows),
              static_cast<long long>(num_experts), route::MAX_COUNT);
  LNQ_REQUIRE(groups > 0 && groups <= 64 && num_experts % groups == 0 && group_top > 0 && group_top <= groups &&
                  (group_best == 1 || group_best == 2),
              "lnq_expert_route: %lld experts in %lld groups (1 to 64, of equal size), %lld kept by their best %lld (1 or 2)",
              static_cast<long long>(num_experts), static_cast<long long>(groups), static_cast<long long>(group_top),
              static_cast<long long>(group_best));
  LNQ_REQUIRE(top > 0 && top <= route::MAX_TOP && top <= group_top * (num_experts / groups),
              "lnq_expert_route: %lld choices a row (1 to %d, from %lld groups of %lld)", static_cast<long long>(top),
              route::MAX_TOP, static_cast<long long>(group_top), static_cast<long long>(num_experts / groups));
  if (rows == 0) {
    clear_error();
    return LNQ_OK;
  }
  LNQ_REQUIRE(logits && experts && weights, "lnq_expert_route: null pointer");
  LNQ_REQUIRE(stride >= 0, "lnq_expert_route: a negative row stride");
  RouteArgs a{};
  a.bias = bias;
  a.experts = experts;
  a.weights = weights;
  a.stride = stride;
  a.rows = static_cast<int>(rows);
  a.count = static_cast<int>(num_experts);
  a.top = static_cast<int>(top);
  a.groups = static_cast<int>(groups);
  a.group_top = static_cast<int>(group_top);
  a.size = a.count / a.groups;
  a.group_best = static_cast<int>(std::min<int64_t>(group_best, a.size));
  int wide = 1;
  while (wide < a.groups) wide *= 2;
  a.lanes = 64 / wide;
  a.softmax = softmax != 0;
  a.renormalize = renormalize != 0;
  a.scale = scale;
  const dim3 grid((a.rows + route::THREADS / 64 - 1) / (route::THREADS / 64));
  const int slots = (a.size + a.lanes - 1) / a.lanes;  // at most 31: 1024 / 33 with a lane a group
#define LNQ_ROUTE(DT, S)                                                                                \
  hipLaunchKernelGGL((expert_route_kernel<DT, S>), grid, dim3(route::THREADS), 0,                       \
                     static_cast<hipStream_t>(stream), static_cast<const typename Elem<DT>::storage*>(logits), a)
#define LNQ_ROUTE_S(DT)                        \
  do {                                         \
    if (slots <= 1) LNQ_ROUTE(DT, 1);          \
    else if (slots <= 2) LNQ_ROUTE(DT, 2);     \
    else if (slots <= 4) LNQ_ROUTE(DT, 4);     \
    else if (slots <= 8) LNQ_ROUTE(DT, 8);     \
    else if (slots <= 16) LNQ_ROUTE(DT, 16);   \
    else LNQ_ROUTE(DT, 32);                    \
  } while (0)
  if (dtype == LNQ_BF16) LNQ_ROUTE_S(LNQ_BF16);
  else if (dtype == LNQ_F16) LNQ_ROUTE_S(LNQ_F16);
  else LNQ_ROUTE_S(LNQ_F32);
#undef LNQ_ROUTE_S
#undef LNQ_ROUTE
  return launched("expert_route");
}

}  // extern "C"
