// The router of a mixture of experts: for each token the experts its row of logits chooses,
// and their weights.
//
//   s_e = exp(l_e) / sum_j exp(l_j)  or  1 / (1 + exp(-l_e))      the scores
//   c_e = s_e + b_e                                               what the choice goes by
//   a group's score: the sum of its best one or two c_e; the best groups are kept
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
// A wave takes a row, lane l the experts l S .. l S + S - 1.
#include "common.hpp"

namespace lnq {

namespace route {
constexpr int THREADS = 256;
constexpr int MAX_TOP = 64;      // a lane holds a choice
constexpr int MAX_SLOTS = 16;    // experts of a lane
}  // namespace route

struct RouteArgs {
  const float* bias;
  int64_t* experts;
  float* weights;
  int64_t stride;  // logits from row to row
  int rows, count, top, groups, group_top, group_best;
  int softmax, renormalize;
  double scale;
};

__device__ inline double shfl_double(double v, int from) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(__shfl(static_cast<int>(b & 0xffffffffu), from, 64));
  const uint32_t hi = static_cast<uint32_t>(__shfl(static_cast<int>(b >> 32), from, 64));
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}

__device__ inline double shfl_xor_double(double v, int mask) { return shfl_double(v, (threadIdx.x & 63) ^ mask); }

// The largest v of the wave and the lowest index that has it, in every lane.
__device__ inline void wave_best(double& v, int& at) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double w = shfl_xor_double(v, off);
    const int o = __shfl_xor(at, off, 64);
    if (w > v || (w == v && o < at)) v = w, at = o;
  }
}

__device__ inline double wave_sum_double(double v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v += shfl_xor_double(v, off);
  return v;
}

template <int DT, int S>
__global__ __launch_bounds__(route::THREADS) void expert_route_kernel(const typename Elem<DT>::storage* __restrict__ logits,
                                                                      RouteArgs a) {
  using E = Elem<DT>;
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * (route::THREADS / 64) + (threadIdx.x >> 6);
  if (row >= a.rows) return;  // the whole wave
  const double none = -__builtin_huge_val();
  const typename E::storage* from = logits + row * a.stride;
  float l[S];
  double top = none;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int e = lane * S + i;
    l[i] = e < a.count ? E::to_f32(from[e]) : -__builtin_huge_valf();
    bad = bad || l[i] != l[i] || (a.softmax && l[i] == __builtin_huge_valf());
    top = fmax(top, static_cast<double>(l[i]));
  }
  int64_t* const experts = a.experts + static_cast<int64_t>(row) * a.top;
  float* const weights = a.weights + static_cast<int64_t>(row) * a.top;
  if (__ballot(bad)) {
    if (lane < a.top) experts[lane] = -1, weights[lane] = __builtin_nanf("");
    return;
  }
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) top = fmax(top, shfl_xor_double(top, off));

  double s[S], c[S], sum = 0;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const double v = l[i];
    if (v == none) s[i] = 0;
    else if (a.softmax) s[i] = exp(v - top);
    else s[i] = 1 / (1 + exp(-v));
    sum += s[i];
  }
  if (a.softmax) {
    sum = wave_sum_double(sum);
#pragma unroll
    for (int i = 0; i < S; ++i) s[i] = sum > 0 ? s[i] / sum : 0;
  }
#pragma unroll
  for (int i = 0; i < S; ++i) {
    c[i] = l[i];
    if (a.bias != nullptr && c[i] != none) {
      c[i] = s[i] + static_cast<double>(a.bias[min(lane * S + i, a.count - 1)]);
      if (c[i] != c[i]) c[i] = none;
    }
  }

  // The value of slot i of the lane that holds expert `at`, in every lane.
  auto pick = [&](const double (&v)[S], int at) -> double {
    double mine = 0;
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (at % S == i) mine = v[i];
    return shfl_double(mine, at / S);
  };
  // The best expert that `in` lets through: its choice and index (none: `none`).
  auto best = [&](auto in, int& at) -> double {
    double v = none;
    at = INT32_MAX;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int e = lane * S + i;
      if (in(e) && c[i] > v) v = c[i], at = e;
    }
    wave_best(v, at);
    return v;
  };

  if (a.groups > 1) {
    const int size = a.count / a.groups;
    double score = none;  // lane g: group g's
    for (int g = 0; g < a.groups; ++g) {
      int at, second;
      double v = best([&](int e) { return e / size == g; }, at);
      if (a.group_best == 2 && v != none) {
        const double w = best([&](int e) { return e / size == g && e != at; }, second);
        if (w == none) v = none;
        else v = a.bias != nullptr ? v + w : pick(s, at) + pick(s, second);
      }
      if (lane == g) score = v;
    }
    uint64_t kept = 0;
    for (int i = 0; i < a.group_top; ++i) {
      double v = (kept >> lane) & 1 || lane >= a.groups ? none : score;
      int at = (kept >> lane) & 1 || lane >= a.groups ? INT32_MAX : lane;
      wave_best(v, at);
      kept |= uint64_t{1} << at;
    }
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (!((kept >> ((lane * S + i) / size & 63)) & 1)) c[i] = none;
  }

  int mine = -1;
  double weight = 0, total = 0;
  for (int i = 0; i < a.top; ++i) {
    int at;
    if (best([](int) { return true; }, at) == none) break;
    const double v = pick(s, at);
    total += v;
    if (lane == i) mine = at, weight = v;
#pragma unroll
    for (int j = 0; j < S; ++j)
      if (lane * S + j == at) c[j] = none;
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
  LNQ_REQUIRE(rows >= 0 && rows <= INT32_MAX && num_experts > 0 && num_experts <= 64 * route::MAX_SLOTS,
              "lnq_expert_route: %lld rows of %lld experts (1 to %d)", static_cast<long long>(rows),
              static_cast<long long>(num_experts), 64 * route::MAX_SLOTS);
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
  a.group_best = static_cast<int>(group_best);
  a.softmax = softmax != 0;
  a.renormalize = renormalize != 0;
  a.scale = scale;
  const dim3 grid((a.rows + route::THREADS / 64 - 1) / (route::THREADS / 64));
  const int slots = (a.count + 63) / 64;
#define LNQ_ROUTE(DT, S)                                                                                \
  hipLaunchKernelGGL((expert_route_kernel<DT, S>), grid, dim3(route::THREADS), 0,                       \
                     static_cast<hipStream_t>(stream), static_cast<const typename Elem<DT>::storage*>(logits), a)
#define LNQ_ROUTE_S(DT)                        \
  do {                                         \
    if (slots <= 1) LNQ_ROUTE(DT, 1);          \
    else if (slots <= 2) LNQ_ROUTE(DT, 2);     \
    else if (slots <= 4) LNQ_ROUTE(DT, 4);     \
    else if (slots <= 8) LNQ_ROUTE(DT, 8);     \
    else LNQ_ROUTE(DT, 16);                    \
  } while (0)
  if (dtype == LNQ_BF16) LNQ_ROUTE_S(LNQ_BF16);
  else if (dtype == LNQ_F16) LNQ_ROUTE_S(LNQ_F16);
  else LNQ_ROUTE_S(LNQ_F32);
#undef LNQ_ROUTE_S
#undef LNQ_ROUTE
  return launched("expert_route");
}

}  // extern "C"
