// Pieces of token scoring shared by the kernels that have logits in memory
// (score.hip) and those that have them in accumulators (fp8.hip).
//
// With a reference logit r, the statistics of a set of logits x are
//   s = sum 2^d,   t = sum 2^d d,   d = log2(e) (x - r),
// so that an exponential is one v_exp_f32. r is the set's largest logit, so no
// term overflows and the largest is 1. The difference is taken before the factor:
// a row of the type's lowest values (a mask) has differences of 0, and their
// products with log2(e) would overflow. Two sets join by moving both to the larger
// reference R, D = log2(e) (r - R):
//   s' = s 2^D,   t' = 2^D (t + s D).
// At the end, with R, S, T of the whole row,
//   log p(i) = x_i - R - ln 2 log2 S,   H = ln 2 (log2 S - T / S).
// All of it is f32: the terms are positive (t's of one sign), so a sum in a tree is
// off by a few half steps.
#pragma once

#include "common.hpp"
#include "fp8.hpp"

namespace uocr {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kErrShape = 4;

struct ScorePart {
  float r, s, t, unused;
};

// The statistics of no logit, or of banned ones (-inf) only: no reference.
__device__ __forceinline__ ScorePart empty_part() { return {-INFINITY, 0.0f, 0.0f, 0.0f}; }

__device__ __forceinline__ ScorePart join(const ScorePart& a, const ScorePart& b) {
  // A part without a logit has s = 0; a part with a NaN has s = NaN and keeps it.
  if (b.s == 0.0f) return a;
  if (a.s == 0.0f) return b;
  const float r = fmaxf(a.r, b.r);
  const float da = (a.r - r) * kLog2e, db = (b.r - r) * kLog2e;
  const float ea = __builtin_amdgcn_exp2f(da), eb = __builtin_amdgcn_exp2f(db);
  ScorePart o;
  o.r = r;
  o.s = a.s * ea + b.s * eb;
  // A factor that vanished takes its (possibly infinite) distance with it.
  const float ta = ea == 0.0f ? 0.0f : ea * fmaf(a.s, da, a.t);
  const float tb = eb == 0.0f ? 0.0f : eb * fmaf(b.s, db, b.t);
  o.t = ta + tb;
  o.unused = 0.0f;
  return o;
}

__device__ __forceinline__ ScorePart shfl_xor(const ScorePart& p, int o) {
  return {__shfl_xor(p.r, o), __shfl_xor(p.s, o), __shfl_xor(p.t, o), 0.0f};
}

// op over the lanes of equal lane % R (a power of two), in each of them: rotations
// within rows of 16 lanes, then across the rows.
template <int R, class Op>
__device__ __forceinline__ float lanes_reduce(float v, const Op& op) {
  if (R <= 1) v = op(v, dpp_move<0x121>(v));
  if (R <= 2) v = op(v, dpp_move<0x122>(v));
  if (R <= 4) v = op(v, dpp_move<0x124>(v));
  if (R <= 8) v = op(v, dpp_move<0x128>(v));
  if (R <= 16) v = op(v, __shfl_xor(v, 16));
  if (R <= 32) v = op(v, __shfl_xor(v, 32));
  return v;
}
// The join of those lanes' parts, all moved to their largest reference at once: one
// exponential instead of two for each pair.
template <int R>
__device__ __forceinline__ ScorePart lanes_join(const ScorePart& p) {
  const bool some = p.s != 0.0f;  // a NaN counts
  auto add = [](float a, float b) { return a + b; };
  ScorePart o;
  o.r = lanes_reduce<R>(some ? p.r : -INFINITY, [](float a, float b) { return fmaxf(a, b); });
  const float d = (p.r - o.r) * kLog2e, e = __builtin_amdgcn_exp2f(d);
  o.s = lanes_reduce<R>(some ? p.s * e : 0.0f, add);
  o.t = lanes_reduce<R>(some && e != 0.0f ? e * fmaf(p.s, d, p.t) : 0.0f, add);
  o.unused = 0.0f;
  return o;
}

// A key that orders logits by value descending, then by index ascending, as
// unsigned numbers; -0 equals 0.
__device__ __forceinline__ unsigned long long order_key(float v, uint32_t index) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)o << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long key) {
  return 0xffffffffu - (uint32_t)key;
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

// Whether a row has a distribution: some finite logit, no NaN and no +inf.
__device__ __forceinline__ bool has_distribution(const ScorePart& p) {
  return p.s > 0.0f && p.s < INFINITY && fabsf(p.r) < INFINITY && p.t == p.t;
}

// Writes row `row`'s log probability and entropy from its statistics and the
// given token's logit.
__device__ __forceinline__ void write_scores(const TokenScores& out, size_t row, int token,
                                             int vocab, const ScorePart& p, float given,
                                             int* err) {
  const bool good = has_distribution(p);
  if (!good) raise_error(err, kErrNumerical);
  const float l = log2f(p.s);
  const float bad = __uint_as_float(0x7fc00000u);
  if (out.logprobs) {
    float lp = bad;
    if (token >= vocab)
      raise_error(err, kErrShape);
    else if (good)
      lp = given - p.r - kLn2 * l;
    out.logprobs[row] = lp;
  }
  if (out.entropy) out.entropy[row] = good ? kLn2 * (l - p.t / p.s) : bad;
}

}  // namespace uocr
