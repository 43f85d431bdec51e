// Scores of logits in memory: the log probability of each row's given token,
// the entropy of its distribution, and its most probable tokens.
//
// One pass over the logits (scores.hpp has the mathematics) leaves, per chunk
// of a row, its statistics and, where alternatives are asked for, the largest
// logit of every group of adjacent columns. The n largest logits of a row lie
// in the n groups with the largest maxima (of equal ones, the leftmost): each
// group in front of another holds an element that comes before all of the
// other's. So the second launch, one workgroup per row, joins the statistics,
// picks n groups from the maxima (1/64 or 1/128 of the row) and reads only
// those again.
#include <algorithm>

#include "fp8.hpp"
#include "scores.hpp"

namespace uocr {

constexpr int kScoreThreads = 256;

template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float widen(float v) { return v; }
};
struct Bf16 {
  uint16_t bits;
};
template <>
struct Logits<Bf16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float widen(Bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
};
template <>
struct Logits<_Float16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float widen(_Float16 v) { return (float)v; }
};

static int vec_of(int type) { return type == kTypeF32 ? 4 : 8; }
static int group_of(int type) { return 16 * vec_of(type); }

// Vectors per thread of a chunk: large chunks where there are many rows, small
// ones where a few rows have to fill the card.
static int chunk_vectors(size_t rows, int vocab, int type) {
  int v = 8;
  while (v > 1 && rows * (((size_t)vocab + kScoreThreads * vec_of(type) * v - 1) /
                          (kScoreThreads * vec_of(type) * v)) < 2048)
    v /= 2;
  return v;
}

struct ScorePlan {
  int vectors, chunk, chunks, groups;
  size_t maxima_at, bytes;
};
static ScorePlan plan_scores(size_t rows, int vocab, int type, int top) {
  ScorePlan p;
  p.vectors = chunk_vectors(rows, vocab, type);
  p.chunk = kScoreThreads * vec_of(type) * p.vectors;
  p.chunks = (int)(((size_t)vocab + p.chunk - 1) / p.chunk);
  p.groups = (int)(((size_t)vocab + group_of(type) - 1) / group_of(type));
  // Room for `rows` rows or fewer: fewer rows may take smaller chunks (at most
  // 2 * 2047 of them in all, or one vector per thread each).
  const size_t unit = (size_t)kScoreThreads * vec_of(type);
  const size_t most = std::max(rows * (((size_t)vocab + 8 * unit - 1) / (8 * unit)),
                               std::min<size_t>(4096, rows * (((size_t)vocab + unit - 1) / unit)));
  p.maxima_at = most * sizeof(ScorePart);
  p.bytes = p.maxima_at + (top ? rows * p.groups * sizeof(float) : 0);
  return p;
}

size_t token_score_bytes(size_t rows, int vocab, int type, int top) {
  return plan_scores(rows, vocab, type, top).bytes;
}

size_t token_score_rows(int vocab, int type) {
  // Many rows take chunks of eight vectors per thread.
  const size_t chunk = (size_t)kScoreThreads * vec_of(type) * 8;
  const size_t chunks = ((size_t)vocab + chunk - 1) / chunk;
  const size_t rows = (((size_t)1 << 24) - 1) / chunks;
  return rows < ((size_t)1 << 22) ? (rows ? rows : 1) : (size_t)1 << 22;
}

// One vector of a row as f32, -inf behind the row's end. Rows may start at any
// element.
template <typename T>
__device__ __forceinline__ void load_logits(const T* row, int c, int vocab, float (&v)[Logits<T>::kVec]) {
  constexpr int kVec = Logits<T>::kVec;
  if (c + kVec <= vocab) {
    T raw[kVec];
    __builtin_memcpy(raw, row + c, sizeof raw);
#pragma unroll
    for (int j = 0; j < kVec; j++) v[j] = Logits<T>::widen(raw[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; j++) v[j] = c + j < vocab ? Logits<T>::widen(row[c + j]) : -INFINITY;
  }
}

template <typename T>
__global__ __launch_bounds__(kScoreThreads) void score_chunks_kernel(
    const T* __restrict__ logits, int vocab, size_t ld, const int32_t* __restrict__ tokens,
    int vectors, int chunks, ScorePart* __restrict__ parts, float* __restrict__ maxima, int groups) {
  constexpr int kVec = Logits<T>::kVec;
  __shared__ ScorePart held[kScoreThreads / 64];
  const size_t row = blockIdx.x / (unsigned)chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)chunks);
  if (tokens && tokens[row] < 0) return;  // a padding row is not read
  const T* x = logits + row * ld;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  ScorePart p = empty_part();
  for (int i = 0; i < vectors; i++) {
    const int c = ((chunk * vectors + i) * kScoreThreads + tid) * kVec;
    float v[kVec];
    load_logits<T>(x, c, vocab, v);
    float most = v[0];
#pragma unroll
    for (int j = 1; j < kVec; j++) most = fmaxf(most, v[j]);
    ScorePart q = empty_part();
    bool nan = false;
#pragma unroll
    for (int j = 0; j < kVec; j++) nan |= v[j] != v[j];
    if (most > -INFINITY || nan) {
      q.r = most;
#pragma unroll
      for (int j = 0; j < kVec; j++) {
        const float d = (v[j] - q.r) * kLog2e;
        const float e = __builtin_amdgcn_exp2f(d);
        q.s += e;
        q.t = fmaf(e, fmaxf(d, -1000.0f), q.t);  // a banned word: 0 times -inf is 0 here
      }
    }
    p = join(p, q);
    if (maxima) {
      float g = most;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor(g, o));
      if ((lane & 15) == 0 && c < vocab) maxima[row * groups + c / (16 * kVec)] = g;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) p = join(p, shfl_xor(p, o));
  if (lane == 0) held[wave] = p;
  __syncthreads();
  if (tid == 0) parts[blockIdx.x] = join(join(held[0], held[1]), join(held[2], held[3]));
}

// The workgroup's largest key.
__device__ __forceinline__ unsigned long long block_max(unsigned long long key,
                                                        unsigned long long* held) {
  key = wave_max_u64(key);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) held[threadIdx.x >> 6] = key;
  __syncthreads();
  unsigned long long best = held[0];
#pragma unroll
  for (int w = 1; w < kScoreThreads / 64; w++) best = held[w] > best ? held[w] : best;
  return best;
}

template <typename T>
__global__ __launch_bounds__(kScoreThreads) void score_rows_kernel(
    const T* __restrict__ logits, int vocab, size_t ld, int chunks,
    const ScorePart* __restrict__ parts, const float* __restrict__ maxima, int groups,
    TokenScores out, int* err) {
  constexpr int kGroup = 16 * Logits<T>::kVec;
  __shared__ ScorePart held[kScoreThreads / 64];
  __shared__ unsigned long long keys[kScoreThreads / 64];
  __shared__ int picked[kMaxTop];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int token = out.tokens ? out.tokens[row] : 0;
  const int top = out.top;
  if (token < 0) {  // a padding row
    if (tid == 0 && out.logprobs) out.logprobs[row] = 0.0f;
    if (tid == 0 && out.entropy) out.entropy[row] = 0.0f;
    for (int i = tid; i < top; i += kScoreThreads) {
      out.top_ids[row * top + i] = -1;
      out.top_logprobs[row * top + i] = -INFINITY;
    }
    return;
  }
  ScorePart p = empty_part();
  for (int c = tid; c < chunks; c += kScoreThreads) p = join(p, parts[row * chunks + c]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) p = join(p, shfl_xor(p, o));
  if (lane == 0) held[wave] = p;
  __syncthreads();
  p = join(join(held[0], held[1]), join(held[2], held[3]));
  const T* x = logits + row * ld;
  if (tid == 0)
    write_scores(out, row, token, vocab, p,
                 out.logprobs && token < vocab ? Logits<T>::widen(x[token]) : 0.0f, err);
  if (top == 0) return;
  if (!has_distribution(p)) {
    for (int i = tid; i < top; i += kScoreThreads) {
      out.top_ids[row * top + i] = -1;
      out.top_logprobs[row * top + i] = __uint_as_float(0x7fc00000u);
    }
    return;
  }
  // The groups, in order; keys are distinct, so each is the largest below the
  // one before it.
  const int some = min(top, groups);
  unsigned long long last = ~0ull;
  for (int i = 0; i < some; i++) {
    unsigned long long best = 0;
    for (int g = tid; g < groups; g += kScoreThreads) {
      const unsigned long long key = order_key(maxima[row * groups + g], (uint32_t)g);
      if (key < last && key > best) best = key;
    }
    last = block_max(best, keys);
    if (tid == 0) picked[i] = (int)key_index(last);
  }
  __syncthreads();
  const float l = log2f(p.s);
  last = ~0ull;
  for (int i = 0; i < top; i++) {
    unsigned long long best = 0;
    for (int c = tid; c < some * kGroup; c += kScoreThreads) {
      const int col = picked[c / kGroup] * kGroup + c % kGroup;
      if (col >= vocab) continue;
      const unsigned long long key = order_key(Logits<T>::widen(x[col]), (uint32_t)col);
      if (key < last && key > best) best = key;
    }
    last = block_max(best, keys);
    if (tid == 0) {
      out.top_ids[row * top + i] = (int32_t)key_index(last);
      out.top_logprobs[row * top + i] = key_value(last) - p.r - kLn2 * l;
    }
  }
}

template <typename T>
static void launch(const T* logits, size_t rows, int vocab, size_t ld, const ScorePlan& plan,
                   const TokenScores& out, void* work, int* err, hipStream_t s) {
  auto* parts = static_cast<ScorePart*>(work);
  float* maxima = out.top ? reinterpret_cast<float*>(static_cast<char*>(work) + plan.maxima_at) : nullptr;
  score_chunks_kernel<T><<<(unsigned)(rows * plan.chunks), kScoreThreads, 0, s>>>(
      logits, vocab, ld, out.tokens, plan.vectors, plan.chunks, parts, maxima, plan.groups);
  score_rows_kernel<T><<<(unsigned)rows, kScoreThreads, 0, s>>>(logits, vocab, ld, plan.chunks, parts,
                                                                maxima, plan.groups, out, err);
}

void launch_token_scores(const void* logits, int type, size_t rows, int vocab, size_t ld,
                         const TokenScores& out, void* work, int* err, hipStream_t s) {
  const ScorePlan plan = plan_scores(rows, vocab, type, out.top);
  if (type == kTypeF32)
    launch((const float*)logits, rows, vocab, ld, plan, out, work, err, s);
  else if (type == kTypeBf16)
    launch((const Bf16*)logits, rows, vocab, ld, plan, out, work, err, s);
  else
    launch((const _Float16*)logits, rows, vocab, ld, plan, out, work, err, s);
}

}  // namespace uocr
